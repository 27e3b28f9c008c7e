"""Attention behind a shared prefix at sizes where the prefix is gone through once: by few
query rows in blocks of 16 beside the sequences' own tiles, by many in blocks of 128, in
equal parts and in runs that go on into the next block; behind it the sequences' own
tokens, single ones and prompts. Against tests/kv_attend_reference.py."""
import numpy as np
import pytest

from tests import kv_attend_reference as ref
from tests.gpu_util import dev, host
from tests.test_gpu_kv_shared import build, run
from tests.test_gpu_kvcache import check, note

pytestmark = pytest.mark.gpu

# a prefix of less than 1024 tiles (of 64 tokens; 512 for heads of 256), counted for each
# sequence, kv head and 16 query rows, is read by every sequence by itself
CASES = {
    # prefix, sequences, own tokens up to, new tokens up to, kv heads, group, dim, page, softcap
    "few rows": (1024, 20, 60, 1, 4, 3, 64, 16, 0),
    "few rows, one part": (576, 60, 30, 1, 2, 1, 64, 64, 0),
    "few rows, long own": (1088, 9, 1300, 1, 8, 2, 96, 32, 30.0),
    "few rows of several tokens": (960, 12, 90, 4, 8, 4, 128, 64, 0),
    "few rows, heads of 256": (704, 12, 100, 1, 4, 2, 256, 32, 0),
    "16 rows each": (1024, 16, 40, 1, 4, 16, 128, 16, 0),
    "many rows of single tokens": (704, 64, 50, 1, 2, 8, 64, 32, 0),
    "many rows, heads of 128": (832, 70, 90, 1, 2, 7, 128, 64, 50.0),
    "many rows of several tokens": (640, 40, 60, 6, 4, 4, 96, 16, 0),
    "prompts": (1344, 3, 200, 150, 4, 3, 64, 32, 0),
    "prompts, heads of 128": (1088, 4, 170, 120, 4, 2, 128, 64, 0),
    "prompts, heads of 256": (640, 3, 140, 110, 2, 4, 256, 128, 0),
    "prompts in one piece": (256, 40, 140, 130, 4, 8, 64, 64, 0),  # more row blocks than splits are made for
    "runs over two blocks": (3200, 11, 30, 17, 2, 5, 128, 16, 0),
}


def ragged(rng, n, most, least=1):
    x = [int(v) for v in rng.integers(least, most + 1, n)]
    x[0] = most
    return x


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("name", CASES)
def test_paths(name, fmt, f16):
    prefix, seqs, most, new_most, heads, group, dim, page, cap = CASES[name]
    note(f"shared paths {name} {fmt} f16={f16}")
    rng = np.random.default_rng(sum(map(ord, name)))
    new = ragged(rng, seqs, new_most)
    own = [max(a, b) for a, b in zip(ragged(rng, seqs, most), new)]
    if seqs > 4:
        own[2], new[2] = None, 0  # an idle slot
    if new_most == 1 and seqs > 4:
        own[2], new[2] = 1, 1
    both = build(rng, prefix, own, heads, dim, page, fmt)
    lens = [0 if n is None else prefix + n for n in own]
    hq = heads * group
    q = (2 * rng.standard_normal((sum(new), hq, dim))).astype(np.float32)
    want, tol = ref.attend(both.ref, q, lens, new, dim ** -0.5, cap)
    both.call(lens, new, new_most == 1)
    got = run(both, q, new, hq, dim, f16, prefix, cap)
    check(got, want, tol, f16)
    both.call(lens, new)
    assert np.array_equal(run(both, q, new, hq, dim, f16, prefix, cap), got)  # the same bits, by row starts too
    check(run(both, q, new, hq, dim, f16, prefix - 100, cap), want, tol, f16)


WAYS = {"few": (20, 1, 3), "many": (40, 1, 16), "pieces": (24, 5, 6), "prompts": (20, 60, 1)}


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("way", WAYS)
def test_rows_inside_the_prefix(way, fmt):
    """Sequences at different places of one list: each sees its own and earlier positions."""
    seqs, new, group = WAYS[way]
    note(f"shared paths: rows inside the prefix, {way} {fmt}")
    rng = np.random.default_rng(41)
    both = build(rng, 1024, [5] * seqs, 4, 64, 32, fmt)
    lens = [1024, new, 64 + new - 1, 63 + new - 1, 700, 128 + new, 1000, 512] + [1024 - 7 * i for i in range(seqs - 8)]
    q = (2 * rng.standard_normal((seqs * new, 4 * group, 64))).astype(np.float32)
    want, tol = ref.attend(both.ref, q, lens, [new] * seqs, 0.125)
    for one_each in ([True, False] if new == 1 else [False]):
        both.call(lens, [new] * seqs, one_each)
        for shared in (1024, 2 ** 31 - 1):
            check(run(both, q, [new] * seqs, 4 * group, 64, False, shared), want, tol, False)


@pytest.mark.parametrize("way", WAYS)
def test_holes_and_idle_slots(way):
    """Pages of no name among the common ones; idle slots, whose queries stay theirs."""
    import torch
    seqs, new, group = WAYS[way]
    note(f"shared paths: holes, {way}")
    rng = np.random.default_rng(42)
    own = [new + 3] * seqs
    if new == 1:
        own[0] = own[7] = None
    both = build(rng, 1024, own, 4, 64, 32, "e4m3")
    t = both.ref.table
    t[:, 3], t[:, 9], t[:, 31] = -1, 10 ** 6, len(both.ref.k)
    both.gpu.page_table.copy_(torch.from_numpy(t))
    lens = [0 if n is None else 1024 + n for n in own]
    rows = [0 if n is None else new for n in own]
    q = rng.standard_normal((sum(rows), 4 * group, 64)).astype(np.float32)
    want, tol = ref.attend(both.ref, q, lens, rows, 0.125)
    if new == 1:
        full = np.full((seqs, 4 * group, 64), np.nan, np.float32)
        there = np.array(rows) > 0
        full[there] = q
        both.call(lens, [1] * seqs, True)
        got = run(both, full, [1] * seqs, 4 * group, 64, False, 1024)
        assert np.all(got[~there] == 0)
        check(got[there], want, tol, False)
    both.call(lens, rows)
    check(run(both, q, rows, 4 * group, 64, False, 1024), want, tol, False)


@pytest.mark.parametrize("wild", [2 ** 31 - 1, -2 ** 31, -1, 5])
@pytest.mark.parametrize("way", WAYS)
def test_wild_lengths(way, wild):
    """Lengths and row starts that make no sense; rows of no sequence stay as they are."""
    import torch
    seqs, new, group = WAYS[way]
    note(f"shared paths: wild {wild}, {way}")
    rng = np.random.default_rng(43)
    both = build(rng, 1024, [new + 20] * seqs, 4, 64, 64, "i8")
    lens, hq = [1044 + new] * seqs, 4 * group
    q = rng.standard_normal((seqs * new, hq, 64)).astype(np.float32)
    want, tol = ref.attend(both.ref, q, lens, [new] * seqs, 0.125)
    keep = np.ones(seqs * new, bool)
    keep[new:2 * new] = False
    for one_each in ([True, False] if new == 1 else [False]):
        both.call(lens, [new] * seqs, one_each)
        both.length[1] = wild
        got = run(both, q, [new] * seqs, hq, 64, False, 1024)
        check(got[keep], want[keep], tol[keep], False)
    both.call(lens, [new] * seqs)
    cu = (np.arange(seqs + 1) * new).astype(np.int32)
    cu[5] = wild  # sequences 4 and 5 have no rows, or (5, where it is a row) wrong ones
    both.gpu.use_cu_tokens(dev(cu))
    out = torch.full((seqs * new, hq * 64), 7.0, device="cuda")
    qt = dev(q)
    both.gpu.attend(qt.data_ptr(), hq * 64, hq, out.data_ptr(), hq * 64, seqs * new, new, shared=1024)
    got = host(out).reshape(q.shape)
    if wild != 5:
        assert np.all(got[4 * new:6 * new] == 7)
    keep = np.ones(seqs * new, bool)
    keep[4 * new:6 * new] = False
    if wild == 5:
        keep[:6 * new] = False
    check(got[keep], want[keep], tol[keep], False)


@pytest.mark.parametrize("way", WAYS)
def test_odd_queries_and_scales(way):
    """Tiny, huge, infinite and NaN queries, loud and silent pages on either side of the
    prefix's end."""
    import torch
    seqs, new, group = WAYS[way]
    note(f"shared paths: odd queries, {way}")
    rng = np.random.default_rng(44)
    both = build(rng, 1024, [new + 30] * seqs, 4, 64, 16, "i8")
    for slot, f in ((1, 1e-20), (5, 1e15), (60, 1e10)):
        both.ref.vs[both.ref.table[0, slot]] *= np.float32(f)
    both.ref.vs[both.ref.table[3, 64]] *= np.float32(1e18)
    both.vs.copy_(torch.from_numpy(both.ref.vs))
    rows, lens, hq = seqs * new, [1054 + new] * seqs, 4 * group
    q = rng.standard_normal((rows, hq, 64)).astype(np.float32)
    q[:, 1] *= np.float32(1e-38)
    q[0, 0] *= np.float32(1e25)  # a one-hot softmax
    both.call(lens, [new] * seqs, new == 1)
    want, tol = ref.attend(both.ref, q, lens, [new] * seqs, 0.125)
    check(run(both, q, [new] * seqs, hq, 64, False, 1024), want, tol, False)
    q[0, 2, 5], q[1, 0, 7] = np.nan, np.inf
    got = run(both, q, [new] * seqs, hq, 64, False, 1024)
    assert np.all(np.isnan(got[0, 2])) and np.all(np.isnan(got[1, 0]))
    got[0, 2], got[1, 0] = want[0, 2], want[1, 0]
    check(got, want, tol, False)


@pytest.mark.parametrize("way", WAYS)
def test_stream_graph_and_chain(way):
    """A recorded call and a captured one, with workspaces of their own, replay on new
    lengths, eager work between."""
    import torch
    from modgrad_amd.q4k import Chain
    seqs, new, group = WAYS[way]
    note(f"shared paths: recorded, {way}")
    rng = np.random.default_rng(45)
    hq, dim, rows = 4 * group, 64, seqs * new
    both = build(rng, 1024, [new + 90] * seqs, 4, dim, 16, "e4m3")
    lens = [1114 + new] * seqs
    qt = torch.empty(rows, hq * dim, device="cuda")
    outs = [torch.empty(rows, hq * dim, device="cuda") for _ in range(3)]
    both.call(lens, [new] * seqs)
    ws = [both.gpu.attention_workspace(hq, rows, new, shared=1024) for _ in range(2)]
    s = torch.cuda.Stream()
    chain = Chain.from_ops([both.gpu.op_attend(qt.data_ptr(), hq * dim, hq, outs[0].data_ptr(), hq * dim, rows, new,
                                               ws[0], shared=1024)])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        both.gpu.attend(qt.data_ptr(), hq * dim, hq, outs[1].data_ptr(), hq * dim, rows, new, shared=1024,
                        workspace=ws[1], stream=s)
    for now in (lens, [1024 + new] * seqs, [new + 45 * i for i in range(seqs)][::-1]):
        now = [min(n, 1114 + new) for n in now]
        q = rng.standard_normal((rows, hq, dim)).astype(np.float32)
        qt.copy_(torch.from_numpy(q.reshape(rows, -1)))
        both.length.copy_(torch.tensor(now, dtype=torch.int32))
        for w in ws:
            w.fill_(255)
        torch.cuda.synchronize()
        chain.launch()
        g.replay()
        both.gpu.attend(qt.data_ptr(), hq * dim, hq, outs[2].data_ptr(), hq * dim, rows, new, shared=1024)
        want, tol = ref.attend(both.ref, q, now, [new] * seqs, dim ** -0.5)
        for o in outs:
            check(host(o).reshape(q.shape), want, tol, False)
            assert np.array_equal(host(o), host(outs[0]))
