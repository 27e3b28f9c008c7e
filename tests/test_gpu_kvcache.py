"""Rotary positions and the paged 8-bit cache on the GPU, through the C ABI and
modgrad_amd.kvcache, against the 64-bit reference of tests/kv_reference.py."""
import ctypes

import numpy as np
import pytest

from modgrad_amd import _lib
from tests import kv_reference as ref
from tests.gpu_util import dev, host

pytestmark = pytest.mark.gpu


def note(msg):
    print(f"[case] {msg}", flush=True)


def rope_table_ref(n_pos, rot, first=0, base=10000.0):
    a = np.outer(np.arange(first, first + n_pos, dtype=np.float64), base ** (-2.0 * np.arange(rot // 2) / rot))
    return np.stack([np.cos(a), np.sin(a)], 2)


# ------------------------------------------------------------------- table --

@pytest.mark.parametrize("n_pos,first,rot,kw", [
    (1, 0, 2, {}), (7, 3, 64, {}), (1000, 0, 96, {}), (513, 130000, 128, {"freq_scale": 0.25}),
    (300, 0, 512, {"base": 5e5}), (129, 100000, 128, {"base": 1e6, "freq_scale": 0.25, "ext_factor": 1.0,
                                                      "orig_ctx": 32768.0}),
    (200, 5000, 80, {"freq_scale": 0.5, "ext_factor": 0.7, "orig_ctx": 4096.0, "attn_factor": 1.3}),
    (65, 131007, 64, {"factors": True}), (70000, 0, 18, {})])
def test_rope_table(n_pos, first, rot, kw):
    import torch
    from modgrad_amd.kvcache import RopeScaling, kern
    note(f"table n_pos={n_pos} first={first} rot={rot} {kw}")
    kw = dict(kw)
    i = np.arange(rot // 2, dtype=np.float64)
    base = kw.get("base", 10000.0)
    theta = base ** (-2.0 * i / rot)
    if kw.get("factors"):
        f = np.linspace(1.0, 8.0, rot // 2).astype(np.float32)
        theta, kw["factors"] = theta / f, dev(f)
    t, size = theta * kw.get("freq_scale", 1.0), kw.get("attn_factor", 1.0)
    if kw.get("ext_factor"):
        dim = lambda n: rot * np.log(kw["orig_ctx"] / (2 * np.pi * n)) / (2 * np.log(base))  # noqa: E731
        lo, hi = max(0.0, np.floor(dim(32.0))), min(rot - 1.0, np.ceil(dim(1.0)))
        m = kw["ext_factor"] * (1 - np.clip((i - lo) / max(hi - lo, 0.001), 0, 1))
        t, size = t * (1 - m) + theta * m, size * (1 + 0.1 * np.log(1 / kw["freq_scale"]))
    a = np.outer(np.arange(first, first + n_pos, dtype=np.float64), t)
    want = size * np.stack([np.cos(a), np.sin(a)], 2)
    out = torch.full((n_pos + 1, rot // 2, 2), 7.0, device="cuda")
    kern.rope_table(out.data_ptr(), n_pos, first, rot, RopeScaling(**kw))
    got = host(out)
    assert np.all(got[n_pos] == 7.0)
    # half a step of f32; the 64-bit angle (relative 2^-50 with the frequency's
    # own rounding) times a position of up to 2^17
    assert np.all(np.abs(got[:n_pos] - want) <= 2.0 ** -24 * np.abs(want) + size * (first + n_pos) * 2.0 ** -50)


def test_rope_table_from_gguf(tmp_path):
    from modgrad_amd.gguf import GgmlType, GgufFile, write_gguf
    from modgrad_amd.kvcache import RopeTable
    note("rope table of a GGUF file")
    f = np.linspace(1.0, 4.0, 32).astype(np.float32)
    path = str(tmp_path / "m.gguf")
    write_gguf(path, [("general.architecture", 8, "llama"), ("llama.rope.dimension_count", 4, 64),
                      ("llama.rope.freq_base", 6, 5e5)], [("rope_freqs.weight", [32], GgmlType.F32, f.tobytes())])
    r = RopeTable.from_gguf(GgufFile.open(path), 100, half=False)
    a = np.outer(np.arange(100.0), 5e5 ** (-np.arange(32) / 32.0) / f)
    want = np.stack([np.cos(a), np.sin(a)], 2)
    assert r.rot_dim == 64 and r.n_pos == 100 and not r.half
    assert np.all(np.abs(host(r.table) - want) <= 2.0 ** -24 * np.abs(want) + 100 * 2.0 ** -50)


# -------------------------------------------------------------------- rope --

@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rot,gap,off", [
    (1, 1, 2, 2, 0, 0), (1, 32, 128, 128, 0, 0), (5, 3, 64, 32, 7, 1), (17, 2, 96, 96, 0, 0), (9, 5, 80, 20, 1, 3),
    (33, 7, 128, 24, 64, 0), (3, 1, 256, 256, 0, 2), (257, 4, 66, 66, 0, 0), (2, 2, 512, 512, 0, 0)])
def test_rope(tokens, heads, dim, rot, gap, off, half):
    import torch
    from modgrad_amd.kvcache import RopeTable
    note(f"rope tokens={tokens} heads={heads} dim={dim} rot={rot} gap={gap} off={off} half={half}")
    rng = np.random.default_rng(tokens * dim + rot)
    table = rope_table_ref(300, rot).astype(np.float32)
    rope = RopeTable.wrap(dev(table), half)
    stride = heads * dim + gap
    x = rng.standard_normal(off + tokens * stride).astype(np.float32)
    pos = rng.integers(0, 300, tokens).astype(np.int32)
    xt, pt = dev(x), dev(pos)
    yt = torch.full((tokens * (stride + 3),), 7.0, device="cuda")
    rope.apply(xt.data_ptr() + 4 * off, yt.data_ptr(), pt.data_ptr(), tokens, heads, dim, stride, stride + 3)
    rows = x[off:].reshape(tokens, stride)[:, :heads * dim].reshape(tokens, heads, dim)
    want = np.stack([ref.rotate(rows[t], table[pos[t]], half) for t in range(tokens)])
    got = host(yt).reshape(tokens, stride + 3)
    assert np.all(got[:, heads * dim:] == 7.0)
    got = got[:, :heads * dim].reshape(tokens, heads, dim)
    # one rounding to f32 (2^-24 relative) of a 64-bit value
    assert np.all(np.abs(got - want) <= 2.0 ** -24 * np.abs(want) + 1e-15)
    assert np.array_equal(got[..., rot:], rows[..., rot:])
    rope.apply(xt.data_ptr() + 4 * off, xt.data_ptr() + 4 * off, pt.data_ptr(), tokens, heads, dim, stride, stride)
    again = host(xt)
    assert np.array_equal(again[off:].reshape(tokens, stride)[:, :heads * dim].reshape(got.shape), got)
    if gap:
        assert np.array_equal(again[off:].reshape(tokens, stride)[:, heads * dim:],
                              x[off:].reshape(tokens, stride)[:, heads * dim:])


def test_rope_position_outside_the_table():
    import torch
    from modgrad_amd.kvcache import RopeTable
    note("rope positions outside the table")
    rope = RopeTable.wrap(dev(rope_table_ref(10, 64).astype(np.float32)), True)
    x = torch.ones(4, 64, device="cuda")
    y = torch.zeros(4, 64, device="cuda")
    rope.apply(x.data_ptr(), y.data_ptr(), dev(np.array([9, 10, -1, 2 ** 31 - 1], np.int32)).data_ptr(), 4, 1, 64)
    got = host(y)
    assert np.all(np.isfinite(got[0])) and np.all(np.isnan(got[1:]))


# ------------------------------------------------------------------- cache --

class Both:
    """A cache on the GPU and its reference; bytes behind the lengths and pages
    that nobody has are 0xFF (a NaN in e4m3) with NaN scales."""

    def __init__(self, rng, seqs, max_pages, heads, dim, page, fmt, spare=3, gap=0, absent=()):
        import torch
        from modgrad_amd.kvcache import KvCache
        n = seqs * max_pages + spare
        ids = rng.permutation(n)[:seqs * max_pages].astype(np.int32).reshape(seqs, max_pages)
        for b, slot, what in absent:
            ids[b, slot] = what
        self.ref = ref.Cache(np.full((n, heads, page, dim), 255, np.uint8), np.full((n, heads, dim, page), 255, np.uint8),
                             np.full((n, heads), np.nan, np.float32), np.full((n, heads), np.nan, np.float32), ids, fmt)
        block = heads * page * dim
        kb, vb = (torch.full((n, block + gap), 255, dtype=torch.uint8, device="cuda") for _ in range(2))
        self.k = kb[:, :block].view(n, heads, page, dim) if gap == 0 else kb.as_strided(
            (n, heads, page, dim), (block + gap, page * dim, dim, 1))
        self.v = vb[:, :block].view(n, heads, dim, page) if gap == 0 else vb.as_strided(
            (n, heads, dim, page), (block + gap, page * dim, page, 1))
        self.pads = (kb[:, block:], vb[:, block:])
        self.ks, self.vs = (torch.full((n, heads), float("nan"), device="cuda") for _ in range(2))
        self.length = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.gpu = KvCache.wrap(self.k, self.v, self.ks, self.vs, dev(ids), self.length, fmt=fmt)
        self.seqs, self.heads, self.dim = seqs, heads, dim

    def call(self, lens, new, one_each=False):
        import torch
        self.length.copy_(torch.tensor(lens, dtype=torch.int32))
        self.gpu.use_cu_tokens(None if one_each else dev(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)))

    def same(self):
        assert np.array_equal(host(self.k), self.ref.k)
        assert np.array_equal(host(self.v), self.ref.v)
        assert np.array_equal(host(self.ks), self.ref.ks, equal_nan=True)
        assert np.array_equal(host(self.vs), self.ref.vs, equal_nan=True)
        for p in self.pads:
            assert bool((p == 255).all())


def fill(both, rng, lens, loud=1.0):
    """Tokens 0 .. len-1 of every sequence, appended in one call."""
    seqs, h, d = both.seqs, both.heads, both.dim
    both.call(lens, lens)
    t = sum(lens)
    kv = (rng.standard_normal((t, 2, h, d)) * loud).astype(np.float32)
    kt = dev(kv)
    both.gpu.append(kt.data_ptr(), kt.data_ptr() + 4 * h * d, 2 * h * d, t, max(lens))
    at = 0
    for b, n in enumerate(lens):
        both.ref.append(b, 0, kv[at:at + n, 0].astype(np.float64), kv[at:at + n, 1].astype(np.float64))
        at += n


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("heads,qh,dim,rot,page,half,gap", [
    (1, 1, 64, 64, 16, True, 0), (2, 6, 128, 128, 64, False, 64), (3, 3, 96, 24, 32, True, 0),
    (1, 2, 256, 250, 128, True, 16), (2, 2, 128, 60, 16, False, 0), (2, 4, 64, 0, 32, True, 0)])
def test_append_steps(fmt, heads, qh, dim, rot, page, half, gap):
    """Prompts, single tokens and pieces, one call after another: every byte and
    scale as the reference's, what is behind the lengths untouched."""
    import torch
    from modgrad_amd.kvcache import RopeTable
    rng = np.random.default_rng(heads * 1000 + dim + page)
    both = Both(rng, 3, 4, heads, dim, page, fmt, gap=gap)
    cap = 4 * page
    table = rope_table_ref(cap + 5, max(rot, 2)).astype(np.float32)
    rope = RopeTable.wrap(dev(table), half) if rot else None
    lens = [0, 0, 0]
    for step, new in enumerate([[page + 3, 0, 1], [1, 1, 1], [1, 2 * page, 0], [1, 1, 1], [0, 5, 1], [2, 1, page],
                                [1, 1, 1]]):
        note(f"append {fmt} heads={heads} dim={dim} page={page} step={step} new={new} lens={lens}")
        one = new == [1, 1, 1] and step % 2 == 1
        lens = [a + b for a, b in zip(lens, new)]
        both.call(lens, new, one)
        t = sum(new)
        row = (qh + 2 * heads) * dim + 5
        x = rng.standard_normal((t, row)).astype(np.float32) * np.float32(1.0 + step)
        x[:, ::7] *= 3
        xt = dev(x)
        qo = torch.full((t + 1, qh * dim + 1), 7.0, device="cuda")
        both.gpu.append(xt.data_ptr() + 4 * qh * dim, xt.data_ptr() + 4 * (qh + heads) * dim, row, t, max(new),
                        rope=rope, q=xt.data_ptr(), q_stride=row, q_out=qo.data_ptr(), q_out_stride=qh * dim + 1,
                        n_q_heads=qh)
        q = x[:, :qh * dim].reshape(t, qh, dim)
        k = x[:, qh * dim:(qh + heads) * dim].reshape(t, heads, dim).astype(np.float64)
        v = x[:, (qh + heads) * dim:(qh + 2 * heads) * dim].reshape(t, heads, dim).astype(np.float64)
        want, at = q.astype(np.float64), 0
        for b in range(3):
            for i in range(new[b]):
                if rot:
                    cs = table[lens[b] - new[b] + i]
                    want[at + i] = ref.rotate(q[at + i], cs, half)
                    k[at + i] = ref.rotate(k[at + i], cs, half)
            both.ref.append(b, lens[b] - new[b], k[at:at + new[b]], v[at:at + new[b]])
            at += new[b]
        both.same()
        got = host(qo)
        assert np.all(got[t] == 7.0) and np.all(got[:, qh * dim:] == 7.0)
        assert np.all(np.abs(got[:t, :qh * dim].reshape(want.shape) - want) <= 2.0 ** -24 * np.abs(want) + 1e-15)
    # the pages back as f32: bytes times scale, one rounding
    pages = np.array([both.ref.table[0, 0], -1, both.ref.table[1, 1], len(both.ref.k)], np.int32)
    out = torch.full((2, 4, heads, page, dim), 7.0, device="cuda")
    both.gpu.dequant(dev(pages).data_ptr(), 4, out[0].data_ptr(), out[1].data_ptr())
    got = host(out)
    assert np.all(got[:, [1, 3]] == 0)
    k, v, _ = both.ref.read(0, heads - 1, page)
    assert np.array_equal(got[0, 0, heads - 1], k.astype(np.float32))
    assert np.array_equal(got[1, 0, heads - 1], v.astype(np.float32))


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("one", [True, False])
def test_append_odd_values(fmt, one):
    """Zeros, infinities, NaN, the smallest and the largest; zero pages that get
    a value later; idle slots; sequences past their table; pages of no name."""
    from modgrad_amd.kvcache import RopeTable
    rng = np.random.default_rng(5)
    both = Both(rng, 6, 2, 1, 64, 16, fmt, absent=((3, 0, -1), (4, 0, 10 ** 6)))
    rope = RopeTable.wrap(dev(rope_table_ref(32, 64).astype(np.float32)), True)
    lens = [0, 4, 31, 3, 5, 20]
    note(f"append odd values {fmt} one={one}")
    for step in range(5):
        new = [0, 1, 1, 1, 1, 1]
        lens = [a + b for a, b in zip(lens, new)]
        both.call(lens, new, one)
        x = np.zeros((6, 2, 1, 64), np.float32)
        if step == 1:
            x[1, :, 0, 3], x[2, :, 0, 5], x[5, :, 0, :] = np.inf, np.nan, 1e-42
        if step >= 2:
            x[:] = rng.standard_normal(x.shape) * 10.0 ** (3 * step - 9)
            x[5] *= np.float32(1e30)
            x[1, 1, 0, ::9], x[2, 1, 0, ::5] = -np.inf, np.nan
        if one:
            rows = x
        else:  # slot 0 has no row
            rows = x[1:]
        xt = dev(rows)
        q = dev(np.ones((6, 64), np.float32))
        both.gpu.append(xt.data_ptr(), xt.data_ptr() + 256, 128, len(rows), 1, rope=None, q=q.data_ptr(), q_stride=64,
                        n_q_heads=1)
        for b in range(1, 6):
            p = lens[b] - 1
            if p < 32:
                both.ref.append(b, p, x[b:b + 1, 0].astype(np.float64), x[b:b + 1, 1].astype(np.float64))
        both.same()
    # rotated: the idle slot's query row is NaN, the others finite
    both.call(lens, [0, 1, 1, 1, 1, 1], True)
    xt = dev(np.zeros((6, 2, 64), np.float32))
    both.gpu.append(xt.data_ptr(), xt.data_ptr() + 256, 128, 6, 1, rope=rope, q=q.data_ptr(), q_stride=64, n_q_heads=1)
    got = host(q)
    assert np.all(np.isnan(got[0])) and np.all(np.isfinite(got[[1, 3, 4, 5]])) and np.all(np.isnan(got[2]))


def test_append_leaves_out_what_the_call_does_not_cover():
    """max_new below a sequence's new tokens, and cu_tokens past the rows."""
    rng = np.random.default_rng(6)
    both = Both(rng, 2, 3, 1, 64, 16, "i8")
    note("append max_new, n_tokens bounds")
    x = rng.standard_normal((9, 2, 1, 64)).astype(np.float32)
    xt = dev(x)
    both.call([9, 5], [9, 5])
    both.gpu.append(xt.data_ptr(), xt.data_ptr() + 256, 128, 9, 4)  # rows 9.. of sequence 1 do not exist
    both.ref.append(0, 0, x[:4, 0].astype(np.float64), x[:4, 1].astype(np.float64))
    both.same()


# --------------------------------------------------------------- attention --

def check(got, want, tol, f16, rows_left=None):
    if f16:
        # the result's own rounding, and probabilities of 11 bits: each moves
        # the mean by at most 2^-11 of its share of |v|, which tol's share of
        # 2^-24 (at least 96 of them) scales to
        tol = tol * 2.0 ** 7 + 2.0 ** -11 * np.abs(want) + 2.0 ** -24
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (f"{bad.sum()} of {bad.size} off; first {np.argwhere(bad)[:3].tolist()}: "
                           f"{got[bad][:3]} for {want[bad][:3]}, bound {tol[bad][:3]}")


CASES = [
    # seqs' lengths, new tokens, kv heads, group, dim, page, softcap, window
    ([1], [1], 1, 1, 64, 16, 0, 0),
    ([64], [1], 2, 7, 128, 64, 0, 0),
    ([65], [1], 1, 4, 128, 16, 0, 0),
    ([0, 1, 63, 64, 65, 130, 0], [1, 1, 1, 1, 1, 1, 1], 2, 3, 64, 32, 0, 0),
    ([500, 3, 1200], [1, 1, 1], 2, 5, 96, 32, 0, 0),
    ([777, 90], [1, 1], 1, 16, 256, 128, 30.0, 100),
    ([400], [1], 1, 40, 64, 16, 0, 0),
    ([5], [5], 1, 1, 64, 16, 0, 0),
    ([70, 33, 0, 200], [3, 2, 0, 1], 2, 4, 128, 16, 0, 0),
    ([100], [100], 2, 3, 128, 64, 0, 0),
    ([300, 1, 150], [37, 1, 150], 1, 7, 64, 32, 0, 40),
    ([260], [200], 2, 2, 256, 32, 50.0, 0),
    ([129, 310], [129, 11], 3, 1, 96, 16, 0, 64),
    ([2100], [2], 1, 6, 128, 128, 0, 0),
]


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("k", range(len(CASES)))
def test_attention(k, fmt, f16):
    import torch
    lens, new, heads, group, dim, page, cap, window = CASES[k]
    note(f"attention {CASES[k]} {fmt} f16={f16}")
    rng = np.random.default_rng(50 + k)
    both = Both(rng, len(lens), max(1, -(-max(lens) // page)), heads, dim, page, fmt)
    if sum(lens):
        fill(both, rng, lens)
    rows = sum(new)
    one = all(n == 1 for n in new)
    hq, scale = heads * group, 1.3 / np.sqrt(dim)
    q = rng.standard_normal((rows, hq * dim + 3)).astype(np.float32) * 2
    qt = dev(q)
    out = torch.full((rows + 2, hq * dim + 2), 7.0, device="cuda", dtype=torch.float16 if f16 else torch.float32)
    q3 = q[:, :hq * dim].reshape(rows, hq, dim)
    want, tol = both.ref.attend(q3, lens, new, scale, cap, window)
    for one_each in ([True, False] if one else [False]):
        both.call(lens, new, one_each)
        out.fill_(7.0)
        both.gpu.attend(qt.data_ptr(), hq * dim + 3, hq, out.data_ptr(), hq * dim + 2, rows, max(new), scale=scale,
                        softcap=cap, window=window, out_f16=f16)
        got = host(out).astype(np.float64)
        assert np.all(got[rows:] == 7.0) and np.all(got[:, hq * dim:] == 7.0)
        check(got[:rows, :hq * dim].reshape(want.shape), want, tol, f16)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("new", [1, 30])
def test_attention_absent_and_shared_pages(fmt, new):
    """Tokens in no page are not seen (a row may see nothing); two sequences
    read the same pages; idle slots' NaN queries stay theirs."""
    import torch
    note(f"attention absent pages {fmt} new={new}")
    rng = np.random.default_rng(8)
    both = Both(rng, 5, 6, 2, 64, 16, fmt)
    fill(both, rng, [90, 90, 90, 90, 90])
    t = both.ref.table
    t[1] = t[0]
    t[2, :4] = -1
    t[3] = -1
    t[4, 2], t[4, 4] = 10 ** 6, len(both.ref.k)
    t[4, 1] = t[4, 0]  # the same page twice
    both.gpu.page_table.copy_(torch.from_numpy(t))
    lens, rows = [90, 83, 90, 90, 90], 5 * new
    q = rng.standard_normal((rows, 6, 64)).astype(np.float32)
    for window in (0, 20):
        both.call(lens, [new] * 5, new == 1)
        out = torch.full((rows, 6 * 64), 7.0, device="cuda")
        both.gpu.attend(dev(q).data_ptr(), 384, 6, out.data_ptr(), 384, rows, new, window=window)
        want, tol = both.ref.attend(q, lens, [new] * 5, 0.125, 0, window)
        check(host(out).astype(np.float64).reshape(want.shape), want, tol, False)
        assert np.all(host(out)[3 * new:4 * new] == 0)
    q[0] = np.nan
    lens[0] = 0
    both.call(lens, [new] * 5, new == 1)
    both.gpu.attend(dev(q).data_ptr(), 384, 6, out.data_ptr(), 384, rows, new)
    got = host(out)
    assert np.all(got[0] == 0) and np.all(np.isfinite(got[new:]))


@pytest.mark.parametrize("new", [1, 40])
def test_attention_odd_queries_and_scales(new):
    """Tiny, huge, infinite and NaN queries stay in their rows; pages of very
    different loudness and of zeros."""
    import torch
    note(f"attention odd queries new={new}")
    rng = np.random.default_rng(9)
    both = Both(rng, 4, 5, 1, 64, 16, "i8")
    fill(both, rng, [80, 80, 80, 80])
    for b, f in ((1, 1e-20), (2, 1e15)):
        pid = both.ref.table[b, 1]
        both.ref.vs[pid] *= np.float32(f)
    both.ref.vs[both.ref.table[3, 0]] = 0
    both.ref.v[both.ref.table[3, 0]] = 0
    both.vs.copy_(torch.from_numpy(both.ref.vs))
    both.v.copy_(torch.from_numpy(both.ref.v))
    rows = 4 * new
    q = rng.standard_normal((rows, 3, 64)).astype(np.float32)
    q[:, 1] *= np.float32(1e-38)
    q[0, 0] *= np.float32(1e25)  # a one-hot softmax
    both.call([80] * 4, [new] * 4, new == 1)
    out = torch.full((rows, 192), 7.0, device="cuda")
    both.gpu.attend(dev(q).data_ptr(), 192, 3, out.data_ptr(), 192, rows, new)
    want, tol = both.ref.attend(q, [80] * 4, [new] * 4, 0.125)
    check(host(out).astype(np.float64).reshape(want.shape), want, tol, False)
    clean = host(out).reshape(rows, 3, 64)
    q[0, 2, 5], q[1, 0, 7] = np.nan, np.inf
    both.gpu.attend(dev(q).data_ptr(), 192, 3, out.data_ptr(), 192, rows, new)
    got = host(out).reshape(rows, 3, 64)
    assert np.all(np.isnan(got[0, 2])) and np.all(np.isnan(got[1, 0]))
    got[0, 2], got[1, 0] = clean[0, 2], clean[1, 0]
    assert np.array_equal(got, clean)


def test_attention_one_long_sequence():
    """The split over one sequence's length, its cuts at every place of a tile,
    against torch in 64 bits on the dequantized cache."""
    import torch
    rng = np.random.default_rng(10)
    both = Both(rng, 1, 700, 2, 128, 64, "i8")
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    both.k.copy_(torch.randint(0, 256, both.k.shape, generator=g, device="cuda", dtype=torch.uint8))
    both.v.copy_(torch.randint(0, 256, both.v.shape, generator=g, device="cuda", dtype=torch.uint8))
    for s in (both.ks, both.vs):
        s.copy_(torch.rand(s.shape, generator=g, device="cuda") * 0.02 + 0.005)
    ids = torch.from_numpy(both.ref.table[0]).cuda().long()
    k = both.k[ids].view(torch.int8).double() * both.ks[ids].double()[..., None, None]
    v = both.v[ids].view(torch.int8).double() * both.vs[ids].double()[..., None, None]
    k = k.permute(1, 0, 2, 3).reshape(2, -1, 128)
    v = v.permute(1, 0, 3, 2).reshape(2, -1, 128)
    for n in (44800, 44799, 20001, 4097, 1025, 257, 255):
        note(f"attention long n={n}")
        both.call([n], [1], True)
        q = torch.randn(14, 128, device="cuda", generator=g) * 2
        out = torch.empty(14 * 128, device="cuda")
        both.gpu.attend(q.data_ptr(), 14 * 128, 14, out.data_ptr(), 14 * 128, 1, 1)
        x = q.double().view(2, 7, 128)
        s = x @ k[:, :n].transpose(1, 2) / np.sqrt(128)
        p = torch.softmax(s, -1)
        want = p @ v[:, :n]
        # scores of |s| <= 60 good to (dim + 8) 2^-24 sum|q||k| / sqrt(dim)
        ds = (136 * 2.0 ** -24 / np.sqrt(128)) * (x.abs() @ k[:, :n].abs().transpose(1, 2))
        e = ds + 2.0 ** -23 * (s.abs() + 2 * (s.amax(-1, keepdim=True) - s) + 40) + (96 + n / 32) * 2.0 ** -24
        e = e + ds.amax(-1, keepdim=True)
        tol = (p * e) @ v[:, :n].abs() + (p * e).sum(-1, keepdim=True) * want.abs()
        diff = (out.double().view(2, 7, 128) - want).abs()
        assert bool((diff <= tol).all()), float((diff / tol).max())


@pytest.mark.parametrize("new", [1, 4, 60])
def test_lengths_that_do_not_fit_the_rows(new):
    """Lengths and row starts of any value stay within the call's buffers, with
    the largest window, and sequences beside them keep their results."""
    import torch
    note(f"odd lengths and row starts new={new}")
    rng = np.random.default_rng(21)
    big = 2 ** 31 - 1
    both = Both(rng, 6, 5, 2, 64, 16, "i8")
    random_cache(both, 3)
    kv = torch.randn(2 * new, 128, device="cuda")
    q = torch.randn(2 * new, 4, 64, device="cuda")
    out = torch.zeros(2 * new, 4, 64, device="cuda")
    at = lambda lens, cu: (both.length.copy_(torch.tensor(lens, dtype=torch.int32)),  # noqa: E731
                           both.gpu.use_cu_tokens(torch.tensor(cu, dtype=torch.int32, device="cuda")))
    attend = lambda window: both.gpu.attend(q.data_ptr(), 256, 4, out.data_ptr(), 256, 2 * new, new, window=window)  # noqa: E731
    at([75, 0, 0, 0, 0, 80], [0, new, new, new, new, new, 2 * new])
    attend(0)
    want = host(out).copy()
    for lens, cu in (([75, 3, -5, big, -big, 80], [0, new, new, new, new, new, 2 * new]),
                     ([75, 0, 1, -big, big, 80], [0, new, -big, big, -1, new, 2 * new]),
                     ([75, 0, 2, 5, -1, 80], [0, new, 2 * new + 9, -3, big, new, 2 * new])):
        at(lens, cu)
        for window in (0, big):
            out.fill_(7.0)
            attend(window)
            got = host(out)
            assert np.array_equal(got[:new], want[:new]) and np.array_equal(got[new:], want[new:])
    # more rows than tokens: the rows before the first token see nothing and store nothing
    before = host(both.k).copy()
    at([75, 0, 0, 0, 0, max(new - 1, 0)], [0, new, new, new, new, new, 2 * new])
    for window in (0, 1, big):
        attend(window)
        got = host(out)
        assert np.array_equal(got[:new] if window != 1 else want[:new], want[:new])
        assert np.all(got[new] == 0.0) and np.all(np.isfinite(got))
    both.gpu.append(kv.data_ptr(), kv.data_ptr(), 128, 2 * new, new)
    after = host(both.k)
    held = set(both.ref.table[5, :1 if new < 4 else -(-(new - 1) // 16)]) | set(both.ref.table[0])
    for p in range(len(before)):
        assert p in held or np.array_equal(before[p], after[p])


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("new,dim", [(1, 64), (3, 128), (70, 64), (70, 128), (40, 256)])
def test_attention_of_huge_scores(new, dim, fmt):
    """Scores from 1e4 to 1e12, where the distance of two f32 numbers passes the
    room that f16 weights have: results stay within the values attended to."""
    import torch
    note(f"attention of huge scores new={new} dim={dim} {fmt}")
    rng = np.random.default_rng(dim + new)
    both = Both(rng, 1, 20, 1, dim, 32, fmt)
    random_cache(both, 9)
    both.ref.k[:], both.ref.v[:] = host(both.k), host(both.v)
    both.ref.ks[:], both.ref.vs[:] = host(both.ks), host(both.vs)
    n = 20 * 32 - 5
    both.call([n], [new], new == 1)
    top = max(np.abs(both.ref.read(0, 0, n)[1]).max(), 0.0)
    q = rng.standard_normal((new, 12, dim)).astype(np.float32)
    for f in 10.0 ** np.arange(4, 13, 0.5):
        x = q * np.float32(f)
        xt = dev(x)
        for f16 in (False, True):
            out = torch.full((new, 12, dim), 7.0, device="cuda", dtype=torch.float16 if f16 else torch.float32)
            both.gpu.attend(xt.data_ptr(), 12 * dim, 12, out.data_ptr(), 12 * dim, new, new, scale=1.0, out_f16=f16)
            got = host(out).astype(np.float64)
            assert np.all(np.abs(got) <= top * (1 + 2.0 ** -10)), (f, f16)


@pytest.mark.parametrize("seqs,pages,heads,group,dim,new,fmt", [
    (1, 60, 1, 4, 128, 1, "i8"),      # parts of one row
    (2, 60, 1, 1, 96, 3, "e4m3"),
    (1, 60, 1, 2, 128, 100, "i8"),    # few splits of a block of many rows
    (1, 300, 1, 64, 64, 1, "e4m3"),   # many
])
def test_attention_nan_query_over_split_tokens(seqs, pages, heads, group, dim, new, fmt):
    """A row whose scores are all NaN is NaN however its tokens are split."""
    import torch
    note(f"attention of a NaN query seqs={seqs} pages={pages} heads={heads}x{group} dim={dim} new={new} {fmt}")
    rng = np.random.default_rng(dim + new)
    both = Both(rng, seqs, pages, heads, dim, 64, fmt)
    random_cache(both, pages)
    hq, rows, lens = heads * group, seqs * new, [64 * pages - 3] * seqs
    q = torch.from_numpy(rng.standard_normal((rows, hq, dim)).astype(np.float32)).cuda()
    both.call(lens, [new] * seqs, new == 1)
    outs = []
    for _ in range(2):
        out = torch.full((rows, hq, dim), 7.0, device="cuda")
        both.gpu.attend(q.data_ptr(), hq * dim, hq, out.data_ptr(), hq * dim, rows, new)
        outs.append(host(out))
        q[-1, 0, 1] = float("nan")
    assert np.all(np.isfinite(outs[0])) and np.all(np.isnan(outs[1][-1, 0]))
    outs[1][-1, 0] = outs[0][-1, 0]
    assert np.array_equal(*outs)


def torch_attention(both, q, lens, new, scale, window=0):
    """In 64 bits on the GPU, with the f32 bound of kv_reference.Cache.attend."""
    import torch
    grid = torch.from_numpy(ref.grid(both.gpu.format)).cuda()
    hq, d = q.shape[1], both.dim
    g = hq // both.heads
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    t, eps = 0, 2.0 ** -24
    for b, (n, m) in enumerate(zip(lens, new)):
        if n and m:
            ids = torch.from_numpy(both.ref.table[b, :-(-n // both.gpu.page_tokens)]).cuda().long()
            k = (grid[both.k[ids].long()] * both.ks[ids].double()[..., None, None]).permute(1, 0, 2, 3)
            v = (grid[both.v[ids].long()] * both.vs[ids].double()[..., None, None]).permute(1, 0, 3, 2)
            k, v = (y.reshape(both.heads, -1, d)[:, :n].contiguous() for y in (k, v))
            x = q[t:t + m].double().view(m, both.heads, g, d).permute(1, 2, 0, 3).reshape(both.heads, -1, d)
            s = scale * (x @ k.transpose(1, 2))
            ds = (d + 8) * eps * scale * (x.abs() @ k.abs().transpose(1, 2))
            j = torch.arange(n, device="cuda")
            pos = n - m + torch.arange(m, device="cuda")
            hide = j > pos[:, None]
            if window:
                hide |= j <= pos[:, None] - window
            hide = hide.repeat(g, 1)
            s = s.masked_fill(hide, -torch.inf)
            p = torch.softmax(s, -1)
            top = s.amax(-1, keepdim=True)
            e = ds + ds.amax(-1, keepdim=True) + 2 * eps * (s.abs() + 2 * (top - s) + 34) + 8 * eps + (96 + n / 32) * eps
            e = torch.where(hide, 0.0, e)
            o = p @ v
            w = (p * e) @ v.abs() + (p * e).sum(-1, keepdim=True) * o.abs() + eps * o.abs()
            back = lambda y: y.view(both.heads, g, m, d).permute(2, 0, 1, 3).reshape(m, hq, d)  # noqa: E731
            out[t:t + m], tol[t:t + m] = back(o), back(w)
        t += m
    return out, tol


def random_cache(both, seed):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    for t in (both.k, both.v):
        x = torch.randn(t.shape, generator=g, device="cuda")
        t.copy_(x.mul(40).clamp(-127, 127).to(torch.int8).view(torch.uint8) if both.gpu.format == "i8"
                else x.mul(100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
    for s in (both.ks, both.vs):
        s.copy_(torch.rand(s.shape, generator=g, device="cuda") * 0.02 + 0.005)
    return g


@pytest.mark.parametrize("seqs,most,heads,group,dim,page,new,window,fmt", [
    (300, 300, 2, 4, 64, 16, 1, 0, "i8"),        # more sequences than a work-group has threads
    (300, 1500, 1, 3, 128, 32, 2, 700, "e4m3"),
    (5, 40000, 16, 2, 64, 64, 1, 0, "i8"),       # runs: over 16 tiles for each of the chip's work-groups
    (40, 9000, 8, 7, 128, 128, 1, 0, "e4m3"),
    (90, 400, 2, 2, 64, 16, 40, 0, "i8"),        # more sequences than lanes, many query rows
    (3, 20000, 1, 8, 128, 64, 30, 0, "i8"),      # splits of row blocks, many states
    (2, 6000, 2, 1, 256, 32, 300, 2500, "e4m3"),
    (1, 3000, 4, 7, 128, 64, 2100, 0, "i8"),     # over two work-groups a CU, dealt from both ends
    (500, 512, 8, 1, 64, 64, 1, 0, "i8"),        # rows of at most 8 tiles, far more of them than work-groups
    (300, 512, 8, 1, 256, 64, 1, 0, "e4m3"),
    (600, 9000, 8, 2, 64, 32, 1, 300, "i8"),     # the same by a window
])
def test_attention_large(seqs, most, heads, group, dim, page, new, window, fmt):
    import torch
    note(f"attention large seqs={seqs} most={most} heads={heads}x{group} dim={dim} page={page} new={new} {fmt}")
    rng = np.random.default_rng(seqs + most)
    both = Both(rng, seqs, -(-most // page), heads, dim, page, fmt)
    gen = random_cache(both, most)
    lens = [int(most * rng.random() ** 2) for _ in range(seqs)]
    lens[0] = most
    if seqs > 2:
        lens[-1] = 0
    news = [0 if n == 0 and new > 1 else max(1, min(n, int(new * rng.random()) + 1)) for n in lens]
    news[0] = new
    if new == 1:
        news = [1] * seqs
    rows, hq, scale = sum(news), heads * group, 1.2 / np.sqrt(dim)
    q = torch.randn(rows, hq, dim, generator=gen, device="cuda") * 2
    want, tol = torch_attention(both, q, lens, news, scale, window)
    both.call(lens, news, new == 1)
    ws = both.gpu.attention_workspace(hq, rows, new)
    for f16 in (False, True):
        out = torch.full((rows + 1, hq, dim), 7.0, device="cuda", dtype=torch.float16 if f16 else torch.float32)
        ws.fill_(255)
        both.gpu.attend(q.data_ptr(), hq * dim, hq, out.data_ptr(), hq * dim, rows, new, scale=scale, window=window,
                        out_f16=f16, workspace=ws)
        check(host(out[:rows]).astype(np.float64), host(want), host(tol), f16)
        assert bool((out[rows] == 7.0).all())


@pytest.mark.parametrize("seqs,page,dim", [(300, 16, 64), (70, 128, 256)])
def test_append_many_sequences(seqs, page, dim):
    """One call for hundreds of sequences, single tokens and pieces that pass
    several pages."""
    note(f"append {seqs} sequences page={page} dim={dim}")
    rng = np.random.default_rng(seqs)
    both = Both(rng, seqs, 4, 1, dim, page, "e4m3")
    lens = np.zeros(seqs, int)
    for step in range(3):
        new = rng.integers(0, 2 if step == 1 else page + page // 2, seqs)
        lens = lens + new
        both.call(lens.tolist(), new.tolist())
        x = rng.standard_normal((int(new.sum()), 2, 1, dim)).astype(np.float32) * (1 + step)
        xt = dev(x)
        both.gpu.append(xt.data_ptr(), xt.data_ptr() + 4 * dim, 2 * dim, len(x), int(max(new)))
        t = 0
        for b in range(seqs):
            both.ref.append(b, int(lens[b] - new[b]), x[t:t + new[b], 0].astype(np.float64), x[t:t + new[b], 1].astype(np.float64))
            t += new[b]
        both.same()


def test_append_exact_ties():
    """Quotients that lie on a tie of the code exactly, with scales that have no
    exact reciprocal: largest values 127 s (int8) and 448 s (e4m3), s = 3, 5, 7."""
    note("append exact ties")
    rng = np.random.default_rng(15)
    for fmt in ("i8", "e4m3"):
        for s in (1, 3, 5, 7, 11):
            both = Both(rng, 1, 2, 1, 64, 16, fmt)
            if fmt == "i8":
                x = (rng.integers(-126, 126, (16, 2, 1, 64)) + 0.5) * s
            else:
                g = ref.grid("e4m3")[:126]
                x = (g[:-1] + g[1:])[rng.integers(0, 125, (16, 2, 1, 64))] / 2 * s
            x[0] = ref.MOST[fmt] * s
            x = x.astype(np.float32)
            xt = dev(x)
            both.call([16], [16])
            both.gpu.append(xt.data_ptr(), xt.data_ptr() + 256, 128, 16, 16)
            both.ref.append(0, 0, x[:, 0].astype(np.float64), x[:, 1].astype(np.float64))
            both.same()


def test_prompt_pieces_recorded_once():
    """A recorded call with many query rows (splits and their join), replayed with
    the sequences growing, a dirty workspace and eager work between."""
    import torch
    from modgrad_amd.q4k import Chain
    note("prompt pieces through a chain")
    rng = np.random.default_rng(16)
    both = Both(rng, 3, 12, 2, 256, 128, "e4m3")
    gen = random_cache(both, 5)
    new, hq = [60, 1, 33], 6
    rows = sum(new)
    q = torch.randn(rows, hq, 256, generator=gen, device="cuda")
    out = torch.empty(rows, hq, 256, device="cuda")
    lens = [100, 1, 700]
    both.call(lens, new)
    ws = both.gpu.attention_workspace(hq, rows, 60)
    chain = Chain.from_ops([both.gpu.op_attend(q.data_ptr(), hq * 256, hq, out.data_ptr(), hq * 256, rows, 60, ws)])
    for step in range(5):
        out.fill_(7.0)
        ws.fill_(255)
        both.length.copy_(torch.tensor(lens, dtype=torch.int32))
        chain.launch()
        if step % 2:
            torch.cuda.synchronize()
        want, tol = torch_attention(both, q, lens, new, 1 / 16)
        check(host(out).astype(np.float64), host(want), host(tol), False)
        lens = [n + d for n, d in zip(lens, (177, 64, 130))]


def test_cache_past_4_gib():
    """Offsets that pass 32 bits: pages at both ends of a cache of 5 GiB each."""
    import torch
    from modgrad_amd.kvcache import KvCache
    note("cache past 4 GiB")
    heads, page, dim = 8, 128, 256
    n = 5 * 2 ** 30 // (heads * page * dim)
    k = torch.empty(n, heads, page, dim, dtype=torch.uint8, device="cuda")
    v = torch.empty(n, heads, dim, page, dtype=torch.uint8, device="cuda")
    sc = [torch.zeros(n, heads, device="cuda") for _ in range(2)]
    table = np.array([[n - 1, 0, n // 2]], np.int32)
    c = KvCache.wrap(k, v, *sc, dev(table), torch.zeros(1, dtype=torch.int32, device="cuda"), fmt="i8")
    rng = np.random.default_rng(11)
    x = rng.standard_normal((300, 2, heads, dim)).astype(np.float32)
    c.set_lengths([300], [300])
    xt = dev(x)
    c.append(xt.data_ptr(), xt.data_ptr() + 4 * heads * dim, 2 * heads * dim, 300, 300)
    small = ref.Cache(np.zeros((3, heads, page, dim), np.uint8), np.zeros((3, heads, dim, page), np.uint8),
                      np.zeros((3, heads), np.float32), np.zeros((3, heads), np.float32), np.array([[0, 1, 2]]), "i8")
    small.append(0, 0, x[:, 0].astype(np.float64), x[:, 1].astype(np.float64))
    for i, p in enumerate(table[0]):
        m = min(page, 300 - i * page)
        assert np.array_equal(host(k[int(p)])[:, :m], small.k[i][:, :m])
        assert np.array_equal(host(v[int(p)])[:, :, :m], small.v[i][:, :, :m])
    for new in (1, 20):
        c.set_lengths([300], [new])
        q = rng.standard_normal((new, heads, dim)).astype(np.float32)
        out = torch.empty(new, heads * dim, device="cuda")
        c.attend(dev(q).data_ptr(), heads * dim, heads, out.data_ptr(), heads * dim, new, new)
        want, tol = small.attend(q, [300], [new], 1 / 16)
        check(host(out).astype(np.float64).reshape(want.shape), want, tol, False)


def test_calls_on_two_streams_and_the_default_workspace():
    """Two calls at once, each with its own workspace (one given, one fresh)."""
    import torch
    note("attention on two streams")
    rng = np.random.default_rng(12)
    both = Both(rng, 2, 40, 2, 128, 64, "e4m3")
    fill(both, rng, [2500, 1900])
    both.call([2500, 1900], [1, 1], True)
    q = rng.standard_normal((2, 8, 128)).astype(np.float32)
    want, tol = both.ref.attend(q, [2500, 1900], [1, 1], 1 / np.sqrt(128))
    qt = dev(q)
    ws = both.gpu.attention_workspace(8, 2, 1)
    outs = [torch.zeros(2, 1024, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        both.gpu.attend(qt.data_ptr(), 1024, 8, outs[0].data_ptr(), 1024, 2, 1, workspace=ws, stream=streams[0])
        both.gpu.attend(qt.data_ptr(), 1024, 8, outs[1].data_ptr(), 1024, 2, 1, stream=streams[1])
    torch.cuda.synchronize()
    a, b = host(outs[0]), host(outs[1])
    assert np.array_equal(a, b)
    check(a.astype(np.float64).reshape(want.shape), want, tol, False)


def test_default_workspace_beside_work_on_the_current_stream():
    """The fresh workspace is the launch stream's: what the current stream
    allocates and fills meanwhile does not lie in it."""
    import torch
    note("default workspace, current stream another one")
    rng = np.random.default_rng(22)
    both = Both(rng, 1, 60, 2, 128, 128, "i8")
    random_cache(both, 5)
    q = torch.randn(1, 8, 128, device="cuda")
    both.call([7600], [1], True)
    outs = torch.zeros(32, 1024, device="cuda")
    n = both.gpu.attention_workspace(8, 1, 1).nbytes
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for i in range(32):
            both.gpu.attend(q.data_ptr(), 1024, 8, outs[i].data_ptr(), 1024, 1, 1)  # null stream
            torch.empty(n, dtype=torch.uint8, device="cuda").fill_(255)
    torch.cuda.synchronize()
    got = host(outs)
    assert np.all(np.isfinite(got)) and np.all(got == got[0])


def test_set_lengths_in_place_and_refusals():
    """New lengths reach a chain that was recorded on the old ones, row starts
    included; counts that cannot be are refused and leave the cache as it was."""
    import torch
    from modgrad_amd.kvcache import KvCache
    from modgrad_amd.q4k import BackendError, Chain
    note("set_lengths in place")
    rng = np.random.default_rng(23)
    c = KvCache.new(n_pages=40, page_tokens=16, n_kv_heads=1, head_dim=64, n_seqs=2, max_pages=20)
    sim = None
    kv = torch.empty(8, 2, 64, device="cuda")
    q, out = torch.empty(8, 4, 64, device="cuda"), torch.zeros(8, 4, 64, device="cuda")
    c.set_lengths([5, 3], [5, 3])
    ws = c.attention_workspace(4, 8, 8)
    chain = Chain.from_ops([c.op_append(kv.data_ptr(), kv.data_ptr() + 256, 128, 8, 8),
                            c.op_attend(q.data_ptr(), 256, 4, out.data_ptr(), 256, 8, 8, ws)])
    lens = [0, 0]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for m in ([5, 3], [1, 7], [8, 0], [0, 8], [4, 4]):
        lens = [a + b for a, b in zip(lens, m)]
        with torch.cuda.stream(stream):
            x, y = rng.standard_normal((8, 2, 64)).astype(np.float32), rng.standard_normal((8, 4, 64)).astype(np.float32)
            kv.copy_(torch.from_numpy(x))
            q.copy_(torch.from_numpy(y))
        c.set_lengths(lens, m, stream=stream)
        chain.launch(stream)
        stream.synchronize()
        ids = host(c.page_table)
        if sim is None:
            z = lambda t: np.zeros(tuple(t.shape), host(t).dtype)  # noqa: E731
            sim = ref.Cache(z(c.k), z(c.v), z(c.k_scale), z(c.v_scale), ids.copy(), "i8")
        sim.table, t = ids.copy(), 0
        for b in range(2):
            sim.append(b, lens[b] - m[b], x[t:t + m[b], :1].astype(np.float64), x[t:t + m[b], 1:].astype(np.float64))
            t += m[b]
        want, tol = sim.attend(y, lens, m, 0.125)
        check(host(out).astype(np.float64), want, tol, False)
    was = host(c.seq_len).copy()
    for bad in (dict(lengths=[5]), dict(lengths=[5, -1]), dict(lengths=[5, 3], new=[6, 0]),
                dict(lengths=[5, 3], new=[1, -1]), dict(lengths=[2 ** 30, 3])):
        with pytest.raises(BackendError):
            c.set_lengths(**bad)
    for f in (lambda: c.release(2), lambda: c.release(-1), lambda: c.reserve(2, 1), lambda: c.reserve(0, -1)):
        with pytest.raises(BackendError):
            f()
    assert np.array_equal(host(c.seq_len), was)


def test_tensors_of_the_host_are_refused():
    import torch
    from modgrad_amd.kvcache import KvCache, RopeTable
    from modgrad_amd.q4k import BackendError
    z = lambda *s, dtype=torch.uint8: torch.zeros(*s, dtype=dtype)  # noqa: E731
    c = KvCache.wrap(z(4, 2, 16, 64), z(4, 2, 64, 16), z(4, 2, dtype=torch.float32), z(4, 2, dtype=torch.float32),
                     z(3, 2, dtype=torch.int32), z(3, dtype=torch.int32))
    p = torch.zeros(1024, device="cuda").data_ptr()
    rope = RopeTable.wrap(z(32, 32, 2, dtype=torch.float32), True)
    good = KvCache.new(4, 16, 2, 64, 3, 2)
    for f in (lambda: c.append(p, p, 128, 3, 1), lambda: c.attend(p, 128, 2, p + 2048, 128, 3, 1),
              lambda: c.dequant(p, 1, p, p), lambda: rope.apply(p, p, p, 1, 1, 64),
              lambda: good.append(p, p, 128, 3, 1, rope=rope)):
        with pytest.raises(BackendError):
            f()


@pytest.mark.parametrize("kind", ["chain", "torch graph"])
def test_decode_steps_recorded_once(kind):
    """append + attention recorded once and replayed with growing lengths, eager
    work and synchronizations between the replays."""
    import torch
    from modgrad_amd.kvcache import RopeTable
    from modgrad_amd.q4k import Chain
    note(f"decode steps through a {kind}")
    rng = np.random.default_rng(13)
    both = Both(rng, 3, 6, 2, 64, 16, "i8")
    table = rope_table_ref(96, 64).astype(np.float32)
    rope = RopeTable.wrap(dev(table), False)
    lens = [30, 15, 1]
    fill(both, rng, lens)
    row = (4 + 4) * 64
    x = torch.zeros(3, row, device="cuda")
    qo, out = torch.zeros(3, 256, device="cuda"), torch.zeros(3, 256, device="cuda")
    both.call(lens, [1, 1, 1], True)
    ws = both.gpu.attention_workspace(4, 3, 1)
    at = x.data_ptr()
    app = dict(k=at + 4 * 256, v=at + 4 * 384, kv_stride=row, n_tokens=3, max_new=1, rope=rope, q=at, q_stride=row,
               q_out=qo.data_ptr(), q_out_stride=256, n_q_heads=4)
    att = dict(q=qo.data_ptr(), q_stride=256, n_q_heads=4, out=out.data_ptr(), out_stride=256, n_tokens=3, max_new=1,
               workspace=ws)
    if kind == "chain":
        chain = Chain.from_ops([both.gpu.op_append(**app), both.gpu.op_attend(**att)])
        replay = chain.launch
    else:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s = torch.cuda.current_stream()
            both.gpu.append(**app, stream=s)
            both.gpu.attend(**att, stream=s)
        replay = g.replay
    for step in range(40):
        lens = [n + 1 for n in lens]
        rows = rng.standard_normal((3, row)).astype(np.float32)
        x.copy_(torch.from_numpy(rows))
        both.length.add_(1)
        ws.fill_(255)
        replay()
        if step % 3 == 0:
            torch.cuda.synchronize()
        got = host(out).astype(np.float64).reshape(3, 4, 64)
        q = np.zeros((3, 4, 64))
        for b in range(3):
            cs = table[lens[b] - 1]
            q[b] = ref.rotate(rows[b, :256].reshape(4, 64), cs, False)
            both.ref.append(b, lens[b] - 1, ref.rotate(rows[b, 256:384].reshape(1, 2, 64), cs, False),
                            rows[b, 384:].reshape(1, 2, 64).astype(np.float64))
        assert np.array_equal(host(qo).reshape(q.shape), q.astype(np.float32))
        want, tol = both.ref.attend(q.astype(np.float32), lens, [1, 1, 1], 0.125)
        check(got, want, tol, False)
    both.same()


def test_a_layer_from_prompt_to_tokens():
    """The operators as a decoder layer uses them, with the library's matvecs:
    q, k, v from Q4_K weights, rotation and append, attention, the output
    projection; a prompt through the f16 GEMM, then single tokens."""
    import torch
    from modgrad_amd.kvcache import KvCache, RopeTable
    from modgrad_amd.q4k import Chain, kern, op_matvec
    from oracle import oracle as orc
    note("a layer: prompt, then tokens")
    hid, hq, h, d, t0 = 512, 8, 2, 64, 37
    row = (hq + 2 * h) * d
    wqkv, wo = orc.seeded_weight(1, row, hid, scale=0.05), orc.seeded_weight(2, hid, hq * d, scale=0.05)
    wq, wt = dev(wqkv), dev(wo)
    rng = np.random.default_rng(14)
    cache = KvCache.new(n_pages=8, page_tokens=16, n_kv_heads=h, head_dim=d, n_seqs=1, max_pages=4, fmt="e4m3")
    rope = RopeTable(64, d, half=True)
    table = host(rope.table)
    sim = None
    cache.set_lengths([t0], [t0])
    ids = host(cache.page_table)
    sim = ref.Cache(host(cache.k).copy(), host(cache.v).copy(), host(cache.k_scale).copy(), host(cache.v_scale).copy(),
                    ids.copy(), "e4m3")

    def layer_ref(qkv, lens, new):
        """From the GPU's own q, k, v rows."""
        q = np.zeros((new, hq, d))
        k = np.zeros((new, h, d))
        for i in range(new):
            cs = table[lens - new + i]
            q[i] = ref.rotate(qkv[i, :hq * d].reshape(hq, d), cs, True)
            k[i] = ref.rotate(qkv[i, hq * d:(hq + h) * d].reshape(h, d), cs, True)
        sim.append(0, lens - new, k, qkv[:, (hq + h) * d:].reshape(new, h, d).astype(np.float64))
        return sim.attend(q.astype(np.float32), [lens], [new], d ** -0.5)

    x = torch.from_numpy(rng.standard_normal((t0, hid)).astype(np.float32)).cuda().half()
    qkv = torch.empty(t0, row, device="cuda")
    att = torch.empty(t0, hq * d, device="cuda", dtype=torch.float16)
    y = torch.empty(t0, hid, device="cuda")
    kern.gemm_q4k_f16(wq.data_ptr(), x.data_ptr(), qkv.data_ptr(), row, hid // 256, t0)
    rows = host(qkv).copy()
    at = qkv.data_ptr()
    cache.append(at + 4 * hq * d, at + 4 * (hq + h) * d, row, t0, t0, rope=rope, q=at, q_stride=row, n_q_heads=hq)
    cache.attend(at, row, hq, att.data_ptr(), hq * d, t0, t0, out_f16=True)
    kern.gemm_q4k_f16(wt.data_ptr(), att.data_ptr(), y.data_ptr(), hid, hq * d // 256, t0)
    want, tol = layer_ref(rows, t0, t0)
    check(host(att).astype(np.float64).reshape(want.shape), want, tol, True)
    assert np.all(np.isfinite(host(y)))

    x1, q1 = torch.empty(hid, device="cuda"), torch.empty(row, device="cuda")
    a1, y1 = torch.empty(hq * d, device="cuda"), torch.empty(hid, device="cuda")
    cache.set_lengths([t0 + 1])
    ws = cache.attention_workspace(hq, 1, 1)
    at = q1.data_ptr()
    chain = Chain.from_ops([
        op_matvec(_lib.DTYPE_Q4_K, wq.data_ptr(), x1.data_ptr(), at, row, hid),
        cache.op_append(at + 4 * hq * d, at + 4 * (hq + h) * d, row, 1, 1, rope=rope, q=at, q_stride=row, n_q_heads=hq),
        cache.op_attend(at, row, hq, a1.data_ptr(), hq * d, 1, 1, ws),
        op_matvec(_lib.DTYPE_Q4_K, wt.data_ptr(), a1.data_ptr(), y1.data_ptr(), hid, hq * d)])
    for n in range(t0 + 1, 60):
        cache.set_lengths([n])
        sim.table = host(cache.page_table)
        xs = rng.standard_normal(hid).astype(np.float32)
        x1.copy_(torch.from_numpy(xs))
        kern.matvec_q4k_ex(wq.data_ptr(), x1.data_ptr(), at, row, hid)
        rows = host(q1).copy().reshape(1, row)
        chain.launch()
        want, tol = layer_ref(rows, n, 1)
        got = host(a1)
        check(got.astype(np.float64).reshape(want.shape), want, tol, False)
        yr, absdot = orc.gemv(wo, got, hid, hq * d // 256)
        assert np.all(np.abs(host(y1) - yr) <= 1e-4 * absdot)
    cache.release(0)
    assert host(cache.seq_len)[0] == 0 and len(cache._free) == 8


def test_wrap_refuses():
    import torch
    from modgrad_amd.kvcache import KvCache, RopeScaling, RopeTable
    from modgrad_amd.q4k import BackendError
    z = lambda *s, dtype=torch.uint8: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    good = dict(k=z(4, 2, 16, 64), v=z(4, 2, 64, 16), k_scale=z(4, 2, dtype=torch.float32),
                v_scale=z(4, 2, dtype=torch.float32), page_table=z(3, 2, dtype=torch.int32),
                seq_len=z(3, dtype=torch.int32), cu_tokens=z(4, dtype=torch.int32))
    KvCache.wrap(**good)
    for bad in (dict(k=z(4, 2, 64, 16)), dict(v=z(4, 2, 16, 64)), dict(k=z(4, 2, 16, 64, dtype=torch.int8)),
                dict(k_scale=z(2, 4, dtype=torch.float32)), dict(v_scale=z(4, 2, dtype=torch.float64)),
                dict(page_table=z(3, 2, dtype=torch.int64)), dict(seq_len=z(4, dtype=torch.int32)),
                dict(cu_tokens=z(3, dtype=torch.int32)), dict(v=z(4, 2, 64, 16).cpu()), dict(fmt="e5m2"),
                dict(k=z(4, 16, 2, 64).transpose(1, 2))):
        with pytest.raises(BackendError):
            KvCache.wrap(**{**good, **bad})
    with pytest.raises(BackendError):
        KvCache.wrap(**good).reserve(0, 5)
    with pytest.raises(BackendError):
        RopeTable.wrap(z(4, 32, dtype=torch.float32), True)
    with pytest.raises(BackendError):
        RopeTable(16, 64, True, RopeScaling(factors=z(16, dtype=torch.float32)))
    c = KvCache.new(2, 16, 1, 64, 1, 4)
    with pytest.raises(BackendError):
        c.set_lengths([33])  # 3 pages of 2
    with pytest.raises(BackendError):
        c.set_lengths([65])  # past the table
    with pytest.raises(BackendError):
        c.append(0, 0, 64, 1, 1)
