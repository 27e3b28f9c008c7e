"""How many bits the attention over the 8-bit cache keeps, by the rms of its
error: bounds on single elements add worst cases up, and would not see a lost
digit of q or half of a probability."""
import numpy as np
import pytest

from tests import kv_reference as ref
from tests.gpu_util import dev, host
from tests.test_gpu_kvcache import Both, check, fill, note

pytestmark = pytest.mark.gpu

# A rounding to f16 is uniform over 2^-10 of the number's power of two: its rms is
# 2^-11 / sqrt(3) of that, and over mantissas m spread evenly in their logarithm,
# E[m^2] = 3 / (2 ln 2), 2^-11 / sqrt(3) sqrt(2 ln 2 / 3) of the numbers' rms.
F16 = 2.0 ** -11 / np.sqrt(3) * np.sqrt(2 * np.log(2) / 3)

# f32: exponents below 32 are rounded in the reference taken off (at most twice 2^-20
# between two tiles), in the tile's offset (2^-20) and in the difference (2^-21):
# 3.5 * 2^-20 ln 2 = 2.3e-6. A score below 18 in base 2 has its factors and itself
# rounded, 4 * 2^-24 * 18 ln 2 = 3.0e-6, q and p in 22 bits 2 * 2^-22 * 4. The sums of
# products are random in sign.
F32 = 8e-6


def quiet_cache(both, rms, seed):
    """Codes of K with this rms in pages whose scores are nevertheless the same:
    what a page holds whose scale a loud token set."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    e4m3 = both.gpu.format == "e4m3"
    for t, size in ((both.k, rms), (both.v, 42.0)):
        x = torch.randn(t.shape, generator=g, device="cuda").mul(size)
        t.copy_(x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8) if e4m3
                else x.round().clamp(-127, 127).to(torch.int8).view(torch.uint8))
    both.ks.copy_((torch.rand(both.ks.shape, generator=g, device="cuda") * 0.5 + 0.75) / rms)
    both.vs.copy_(torch.rand(both.vs.shape, generator=g, device="cuda") * 0.01 + 0.01)
    return g


@pytest.mark.parametrize("rms", [42.0, 5.0, 1.0])
@pytest.mark.parametrize("new", [1, 32])
@pytest.mark.parametrize("fmt,dim", [("i8", 64), ("i8", 96), ("i8", 128), ("i8", 256), ("e4m3", 64), ("e4m3", 128),
                                     ("e4m3", 256)])
def test_rms_of_the_error(fmt, dim, new, rms):
    """32 tokens of 4 heads take the kernel for many query rows, 1 token the other."""
    import torch
    note(f"rms of the error {fmt} dim={dim} new={new} rms={rms}")
    n, group, page = 2000, 4, 64
    both = Both(np.random.default_rng(dim), 1, -(-n // page), 1, dim, page, fmt)
    g = quiet_cache(both, rms, dim)
    both.call([n], [new], new == 1)
    scale = dim ** -0.5
    q = 2 * torch.randn(new, group, dim, generator=g, device="cuda")
    grid = torch.from_numpy(ref.grid(fmt)).cuda()
    ids = torch.from_numpy(both.ref.table[0]).cuda().long()
    k = (grid[both.k[ids].long()] * both.ks[ids].double()[..., None, None]).permute(1, 0, 2, 3).reshape(-1, dim)[:n]
    v = (grid[both.v[ids].long()] * both.vs[ids].double()[..., None, None]).permute(1, 0, 3, 2).reshape(-1, dim)[:n]
    x = q.double().view(-1, dim)
    s = scale * (x @ k.t().contiguous())
    hide = torch.arange(n, device="cuda") > (n - new + torch.arange(new, device="cuda")).repeat_interleave(group)[:, None]
    s = s.masked_fill(hide, -torch.inf)
    p = torch.softmax(s, -1)
    want = p @ v
    size = want.pow(2).mean()
    assert float(s.amax() / np.log(2)) < 18
    err = {}
    for f16 in (False, True):
        out = torch.full((new, group, dim), 7.0, device="cuda", dtype=torch.float16 if f16 else torch.float32)
        both.gpu.attend(q.data_ptr(), group * dim, group, out.data_ptr(), group * dim, new, new, scale=scale, out_f16=f16)
        err[f16] = float(((out.double().view(-1, dim) - want).pow(2).mean() / size).sqrt())
    assert err[False] <= F32, err
    # f16 results: their own rounding, and for many query rows probabilities of 11
    # bits and (int8 codes in products of 64 dims) queries of 16 bits of the row's
    # largest, whose steps are uniform: each is off by 1/sqrt(12) of a step.
    var = (want.half().double() - want).pow(2).mean()
    if new > 1:
        var = var + (F16 ** 2 * (p * p) @ (v * v)).mean()
        if fmt == "i8" and dim % 64 == 0:
            step = x.abs().amax(1, keepdim=True) / 32639
            w = p * p * (scale * step) ** 2 / 12 * (k * k).sum(1)
            var = var + (w @ (v * v) - 2 * want * (w @ v) + want * want * w.sum(1, keepdim=True)).mean()
    # a few hundred weights count, so that the rms of their roundings is its
    # expectation to about 4 %: five times that
    assert err[True] <= 1.2 * float((var / size).sqrt()) + F32, (err, float((var / size).sqrt()))


@pytest.mark.parametrize("peak", [False, True])
@pytest.mark.parametrize("fmt,dim", [("i8", 64), ("i8", 96), ("i8", 128), ("i8", 256), ("e4m3", 128), ("e4m3", 256)])
def test_scores_at_the_bounds_of_their_sums(fmt, dim, peak):
    """q constant and K at its largest code, so that the sums of products reach
    their bounds, over scales that take the scores from 1e3 to 1e9: every token
    counts alike, or one alone."""
    import torch
    note(f"scores at the bounds {fmt} dim={dim} peak={peak}")
    n, new, page = 330, 60, 32
    both = Both(np.random.default_rng(dim), 1, -(-n // page), 1, dim, page, fmt)
    most, less = (127, 100) if fmt == "i8" else (0x7E, 0x7C)  # 448, 384
    both.k.fill_(less if peak else most)
    both.k[int(both.ref.table[0, 0]), 0, 10] = most
    g = torch.Generator(device="cuda")
    g.manual_seed(dim)
    v = torch.randn(both.v.shape, generator=g, device="cuda").mul(40).clamp(-127, 127)
    both.v.copy_((v.to(torch.int8) if fmt == "i8" else v.to(torch.float8_e4m3fn)).view(torch.uint8))
    both.ks.fill_(2.0 ** -6)
    both.vs.fill_(2.0 ** -7)
    grid = torch.from_numpy(ref.grid(fmt)).cuda()
    ids = torch.from_numpy(both.ref.table[0]).cuda().long()
    v = (grid[both.v[ids].long()] * 2.0 ** -7).permute(1, 0, 3, 2).reshape(-1, dim)[:n]
    count = (n - new + 1 + torch.arange(new, device="cuda", dtype=torch.float64))[:, None]
    if peak:
        want, size = v[10].expand(new, dim), v[10].abs().expand(new, dim)
    else:
        want, size = (y.cumsum(0)[n - new:] / count for y in (v, v.abs()))
    both.call([n], [new])
    q = torch.ones(new, dim, device="cuda")
    for f16 in (False, True):
        out = torch.empty(new, dim, device="cuda", dtype=torch.float16 if f16 else torch.float32)
        top = grid[most].item() * 2.0 ** -6 * dim  # q . k
        for score in 10.0 ** np.linspace(3, 9, 301):
            out.fill_(7.0)
            both.gpu.attend(q.data_ptr(), dim, 1, out.data_ptr(), dim, new, new, scale=score / top, out_f16=f16)
            off = (out.double() - want).abs()
            # sums of equal weights in f32, weights of 22 bits. Equal scores t in base 2
            # have equal weights where each is rounded to f32 by itself. Below 2^19 a tile
            # that all rows see all of may take t less its reference in one step, and the
            # other tiles round t first (2^-24 t): its largest (2^-24 t) and its offset
            # (2^-24 t) are rounded instead, and its weights are off from theirs by
            # 3 * 2^-24 t ln 2.
            t = score / np.log(2) + 7
            e = (96 + n / 32) * 2.0 ** -24 + 2.0 ** -22 + (3 * 2.0 ** -24 * t * np.log(2) if t < 2 ** 19 else 0.0)
            # f16: weights of 11 bits, all rounded alike, and the result's own rounding
            most_off = e * (size + want.abs()) + (2.0 ** -10 * want.abs() + 2.0 ** -24 if f16 else 0)
            assert bool((off <= most_off).all()), (f16, score, float((off / most_off).max()))


def ends(fmt, dim, new, f16, q, scale):
    """Attention over 100 tokens in two pages of 64 for these queries, against the reference."""
    import torch
    both = Both(np.random.default_rng(3), 1, 2, 1, dim, 64, fmt)
    fill(both, np.random.default_rng(4), [100])
    both.call([100], [new], new == 1)
    out = torch.full((new, 4, dim), 7.0, device="cuda", dtype=torch.float16 if f16 else torch.float32)
    both.gpu.attend(dev(q).data_ptr(), 4 * dim, 4, out.data_ptr(), 4 * dim, new, new, scale=scale, out_f16=f16)
    want, tol = both.ref.attend(q, [100], [new], scale)
    check(host(out).astype(np.float64), want, tol, f16)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("fmt,dim", [("i8", 64), ("i8", 96), ("i8", 128), ("e4m3", 64), ("e4m3", 256)])
def test_queries_up_to_the_largest_f32(fmt, dim, new, f16):
    """Rows whose largest value is 3.4e38 to 3.4028e38, finite as all others."""
    note(f"queries up to the largest f32 {fmt} dim={dim} new={new} f16={f16}")
    rng = np.random.default_rng(dim + new)
    q = (rng.uniform(-1, 1, (new, 4, dim)) * 1e38).astype(np.float32)
    q[:, 0, 3], q[:, 1, 7], q[:, 2, 0] = 3.401e38, -np.finfo(np.float32).max, 3.3999e38
    q[:, 1, 8:] *= np.float32(0.01)
    ends(fmt, dim, new, f16, q, 3e-38 / np.sqrt(dim))


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("size", [1e-36, 1e-38, 1e-40])
@pytest.mark.parametrize("fmt,dim", [("i8", 64), ("i8", 96), ("i8", 128), ("e4m3", 64), ("e4m3", 256)])
def test_queries_down_to_the_smallest_f32(fmt, dim, size, new, f16):
    """Rows near and below the smallest normal number, under scales that bring the
    scores back."""
    note(f"queries of {size} {fmt} dim={dim} new={new} f16={f16}")
    rng = np.random.default_rng(dim + new)
    q = (rng.uniform(-1, 1, (new, 4, dim)) * size).astype(np.float32)
    ends(fmt, dim, new, f16, q, min(3.0 / size, 2e38) / np.sqrt(dim))
