"""Attention over the cache of sequences that begin with the same pages, against the
64-bit reference of tests/kv_attend_reference.py, which reads every sequence by itself."""
import numpy as np
import pytest

from tests import kv_attend_reference as ref
from tests.gpu_util import dev, host
from tests.test_gpu_kvcache import Both, check, note

pytestmark = pytest.mark.gpu


def build(rng, prefix, own, heads, dim, page, fmt, loud=1.0):
    """A cache whose sequences have `prefix` tokens (whole pages) in the same pages and
    own[b] more each; own None: an idle slot without pages."""
    import torch
    assert prefix % page == 0
    common = prefix // page
    most = common + max(1, max(-(-n // page) for n in own if n is not None))
    both = Both(rng, len(own), most, heads, dim, page, fmt)
    t = both.ref.table
    t[1:, :common] = t[0, :common]
    idle = [b for b, n in enumerate(own) if n is None]
    put = lambda: both.gpu.page_table.copy_(torch.from_numpy(t))  # noqa: E731
    put()

    def add(start, lens):
        """lens[b] new tokens of each sequence b at positions `start` on."""
        both.call([start + n if n else 0 for n in lens], lens)
        rows = sum(lens)
        if not rows:
            return
        x = (rng.standard_normal((rows, 2, heads, dim)) * loud).astype(np.float32)
        xt = dev(x)
        both.gpu.append(xt.data_ptr(), xt.data_ptr() + 4 * heads * dim, 2 * heads * dim, rows, max(lens))
        at = 0
        for b, n in enumerate(lens):
            both.ref.append(b, start, x[at:at + n, 0].astype(np.float64), x[at:at + n, 1].astype(np.float64))
            at += n
    first = next(b for b, n in enumerate(own) if n is not None)
    add(0, [prefix if b == first else 0 for b in range(len(own))])
    add(prefix, [n or 0 for n in own])
    both.same()
    for b in idle:
        t[b] = -1
    put()
    return both


def run(both, q, new, hq, dim, f16, shared, cap=0.0, workspace=None, one_each=False):
    import torch
    rows = len(q)
    out = torch.full((rows + 1, hq * dim + 3), 7.0, device="cuda", dtype=torch.float16 if f16 else torch.float32)
    qt = dev(q)
    both.gpu.attend(qt.data_ptr(), hq * dim, hq, out.data_ptr(), hq * dim + 3, rows, max(new), scale=dim ** -0.5,
                    softcap=cap, shared=shared, out_f16=f16, workspace=workspace)
    got = host(out)
    assert np.all(got[rows] == 7) and np.all(got[:, hq * dim:] == 7)
    return got[:rows, :hq * dim].reshape(rows, hq, dim)


CASES = [
    # prefix, own tokens (the new ones among them), new tokens, kv heads, group, dim, page, softcap
    (64, [1, 1], [1, 1], 1, 1, 64, 16, 0),
    (128, [1, 40, 200], [1, 1, 1], 2, 7, 128, 64, 0),
    (80, [5, 70], [1, 1], 1, 4, 96, 16, 0),            # 16 of its tokens are in no whole tile
    (48, [30, 20], [1, 1], 2, 2, 64, 16, 0),           # no whole tile at all
    (640, [100, None, 3, None, 64], [1, 0, 1, 0, 1], 2, 3, 64, 32, 30.0),
    (256, [17, 300], [1, 1], 4, 1, 256, 128, 0),
    (1024, [700, 10, 1], [1, 1, 1], 1, 16, 64, 16, 0),  # 16 rows of one token
    (320, [9, 4, 60], [5, 2, 6], 2, 4, 128, 16, 0),
    (576, [90, 150], [70, 130], 1, 7, 128, 64, 0),     # prompts behind it
    (512, [200, None, 33], [200, 0, 3], 2, 3, 96, 32, 50.0),
    (384, [140, 60], [100, 60], 1, 2, 256, 128, 0),
    (2560, [30, 31, 32, 33, 34], [1, 1, 1, 1, 1], 1, 5, 64, 32, 0),
    (192, [400], [1], 2, 2, 64, 64, 0),                # one sequence
]


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("k", range(len(CASES)))
def test_shared(k, fmt, f16):
    prefix, own, new, heads, group, dim, page, cap = CASES[k]
    note(f"shared {CASES[k]} {fmt} f16={f16}")
    rng = np.random.default_rng(120 + k)
    both = build(rng, prefix, own, heads, dim, page, fmt)
    lens = [0 if n is None else prefix + n for n in own]
    hq = heads * group
    q = (2 * rng.standard_normal((sum(new), hq, dim))).astype(np.float32)
    want, tol = ref.attend(both.ref, q, lens, new, dim ** -0.5, cap)
    both.call(lens, new, new == [1] * len(new))
    got = run(both, q, new, hq, dim, f16, prefix, cap)
    check(got, want, tol, f16)
    assert np.array_equal(run(both, q, new, hq, dim, f16, prefix, cap), got)  # the same bits again
    if new == [1] * len(new):
        both.call(lens, new)  # the same by row starts
        assert np.array_equal(run(both, q, new, hq, dim, f16, prefix, cap), got)
    # less of what is common, and none
    for less in {prefix - 1, prefix // 2, min(prefix, 64), min(prefix, 63)}:
        check(run(both, q, new, hq, dim, f16, less, cap), want, tol, f16)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("new", [1, 30])
def test_rows_inside_the_prefix(fmt, new):
    """Sequences of one list that are at different places of it: a row sees its own
    and earlier positions, however much is said to be shared."""
    note(f"shared: rows inside the prefix {fmt} new={new}")
    rng = np.random.default_rng(31)
    both = build(rng, 960, [20, 20, 20, 20, 20, 20], 2, 64, 32, fmt)
    lens = [980, 960, 64 + new - 1, 63 + new - 1, new, 700]
    q = (2 * rng.standard_normal((6 * new, 6, 64))).astype(np.float32)
    want, tol = ref.attend(both.ref, q, lens, [new] * 6, 0.125)
    both.call(lens, [new] * 6, new == 1)
    for shared in (960, 10 ** 9, 2 ** 31 - 1):
        if shared > 960:  # what follows is each sequence's own: only the others' lengths end it
            lens2 = [min(n, 960) for n in lens]
            want, tol = ref.attend(both.ref, q, lens2, [new] * 6, 0.125)
            both.call(lens2, [new] * 6, new == 1)
        check(run(both, q, [new] * 6, 6, 64, False, shared), want, tol, False)


def test_pages_of_no_name():
    """A hole in the common pages is seen by nobody; idle slots' queries stay theirs."""
    import torch
    note("shared: pages of no name")
    rng = np.random.default_rng(32)
    both = build(rng, 512, [40, None, 90, 5], 1, 128, 32, "i8")
    t = both.ref.table
    t[:, 3], t[:, 7] = -1, 10 ** 6
    t[2, 17] = -1
    both.gpu.page_table.copy_(torch.from_numpy(t))
    lens, new = [552, 0, 602, 517], [1, 1, 1, 1]
    q = rng.standard_normal((4, 3, 128)).astype(np.float32)
    q[1] = np.nan
    both.call(lens, new, True)
    got = run(both, q, new, 3, 128, False, 512)
    assert np.all(got[1] == 0)
    rows = [0, 2, 3]
    want, tol = ref.attend(both.ref, q[rows], lens, [1, 0, 1, 1], 128 ** -0.5)
    check(got[rows], want, tol, False)
    # nothing of the prefix at all
    t[:, :16] = -1
    both.gpu.page_table.copy_(torch.from_numpy(t))
    want, tol = ref.attend(both.ref, q[rows], lens, [1, 0, 1, 1], 128 ** -0.5)
    check(run(both, q, new, 3, 128, False, 512)[rows], want, tol, False)


@pytest.mark.parametrize("new", [2, 80])
def test_rows_of_no_sequence(new):
    """Rows ahead of the first sequence, between two and behind the last stay."""
    import torch
    note(f"shared: rows of no sequence new={new}")
    rng = np.random.default_rng(33)
    both = build(rng, 256, [100, 90], 1, 64, 16, "e4m3")
    rows = 3 + new + 200 + new + 5
    q = rng.standard_normal((rows, 4, 64)).astype(np.float32)
    both.call([356, 346], [new, new])
    # sequence 0 has rows 3 .., sequence 1 those behind a range that a third would have: falling starts have none
    cu = np.array([3, 3 + new, 3 + 2 * new], np.int32)
    both.gpu.use_cu_tokens(dev(cu))
    out = torch.full((rows, 256), 7.0, device="cuda")
    qt = dev(q)
    both.gpu.attend(qt.data_ptr(), 256, 4, out.data_ptr(), 256, rows, new, shared=256)
    got = host(out)
    assert np.all(got[:3] == 7) and np.all(got[3 + 2 * new:] == 7)
    want, tol = ref.attend(both.ref, q[3:3 + 2 * new], [356, 346], [new, new], 0.125)
    check(got[3:3 + 2 * new].reshape(want.shape), want, tol, False)


@pytest.mark.parametrize("wild", [2 ** 31 - 1, -2 ** 31, -1])
@pytest.mark.parametrize("new", [1, 60])
def test_wild_lengths(wild, new):
    """Lengths and row starts that make no sense index nothing outside; the others'
    rows are right."""
    import torch
    note(f"shared: wild {wild} new={new}")
    rng = np.random.default_rng(34)
    both = build(rng, 256, [100, 90, 80], 1, 64, 16, "i8")
    lens = [356, 346, 336]
    q = rng.standard_normal((3 * new, 4, 64)).astype(np.float32)
    want, tol = ref.attend(both.ref, q, lens, [new] * 3, 0.125)
    both.call(lens, [new] * 3)
    both.length[1] = wild
    got = run(both, q, [new] * 3, 4, 64, False, 256)
    for a in (0, 2 * new):
        check(got[a:a + new], want[a:a + new], tol[a:a + new], False)
    both.call(lens, [new] * 3)
    cu = np.array([0, new, wild, 3 * new], np.int32)
    both.gpu.use_cu_tokens(dev(cu))
    out = torch.full((3 * new, 256), 7.0, device="cuda")
    qt = dev(q)
    both.gpu.attend(qt.data_ptr(), 256, 4, out.data_ptr(), 256, 3 * new, new, shared=256)
    check(host(out)[:new].reshape(new, 4, 64), want[:new], tol[:new], False)


@pytest.mark.parametrize("new", [1, 33])
def test_odd_queries_and_scales(new):
    """Tiny, huge, infinite and NaN queries stay in their rows; loud and silent pages on
    either side of the prefix's end."""
    import torch
    note(f"shared: odd queries new={new}")
    rng = np.random.default_rng(35)
    both = build(rng, 320, [50 + new] * 4, 1, 64, 16, "i8")
    for slot, f in ((1, 1e-20), (5, 1e15), (21, 1e10)):
        both.ref.vs[both.ref.table[0, slot]] *= np.float32(f)
    both.ref.vs[both.ref.table[3, 22]] *= np.float32(1e18)
    both.vs.copy_(torch.from_numpy(both.ref.vs))
    rows, lens = 4 * new, [370 + new] * 4
    q = rng.standard_normal((rows, 3, 64)).astype(np.float32)
    q[:, 1] *= np.float32(1e-38)
    q[0, 0] *= np.float32(1e25)  # a one-hot softmax
    both.call(lens, [new] * 4, new == 1)
    want, tol = ref.attend(both.ref, q, lens, [new] * 4, 0.125)
    clean = run(both, q, [new] * 4, 3, 64, False, 320)
    check(clean, want, tol, False)
    q[0, 2, 5], q[1, 0, 7] = np.nan, np.inf
    got = run(both, q, [new] * 4, 3, 64, False, 320)
    assert np.all(np.isnan(got[0, 2])) and np.all(np.isnan(got[1, 0]))
    # the others: to the bound, not the bit, as the rows of a wavefront take a new running
    # maximum (another rounding of every weight) when one of them outgrows its own
    got[0, 2], got[1, 0] = want[0, 2], want[1, 0]
    check(got, want, tol, False)


@pytest.mark.parametrize("new", [1, 50])
def test_stream_graph_and_chain(new):
    """A recorded call and a captured one, with workspaces of their own, replay on new
    lengths, eager work between."""
    import torch
    from modgrad_amd.q4k import Chain
    note(f"shared: recorded new={new}")
    rng = np.random.default_rng(36)
    heads, hq, dim = 2, 4, 64
    both = build(rng, 448, [120, 150, 90], heads, dim, 16, "e4m3")
    lens, rows = [568, 598, 538], 3 * new
    qt = torch.empty(rows, hq * dim, device="cuda")
    outs = [torch.empty(rows, hq * dim, device="cuda") for _ in range(3)]
    both.call(lens, [new] * 3)
    ws = [both.gpu.attention_workspace(hq, rows, new, shared=448) for _ in range(2)]
    s = torch.cuda.Stream()
    chain = Chain.from_ops([both.gpu.op_attend(qt.data_ptr(), hq * dim, hq, outs[0].data_ptr(), hq * dim, rows, new,
                                               ws[0], shared=448)])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        both.gpu.attend(qt.data_ptr(), hq * dim, hq, outs[1].data_ptr(), hq * dim, rows, new, shared=448,
                        workspace=ws[1], stream=s)
    for now in (lens, [new, 500, 448], [448, 449, 512]):
        q = rng.standard_normal((rows, hq, dim)).astype(np.float32)
        qt.copy_(torch.from_numpy(q.reshape(rows, -1)))
        both.length.copy_(torch.tensor(now, dtype=torch.int32))
        for w in ws:
            w.fill_(255)
        torch.cuda.synchronize()
        chain.launch()
        g.replay()
        both.gpu.attend(qt.data_ptr(), hq * dim, hq, outs[2].data_ptr(), hq * dim, rows, new, shared=448)
        want, tol = ref.attend(both.ref, q, now, [new] * 3, dim ** -0.5)
        for o in outs:
            check(host(o).reshape(q.shape), want, tol, False)
            assert np.array_equal(host(o), host(outs[0]))


def test_many_sequences():
    note("shared: 300 sequences")
    rng = np.random.default_rng(37)
    own = [int(n) for n in rng.integers(1, 90, 300)]
    both = build(rng, 256, own, 1, 64, 16, "i8")
    lens, new = [256 + n for n in own], [1] * 300
    q = rng.standard_normal((300, 2, 64)).astype(np.float32)
    want, tol = ref.attend(both.ref, q, lens, new, 0.125)
    for one_each in (True, False):
        both.call(lens, new, one_each)
        check(run(both, q, new, 2, 64, False, 256), want, tol, False)


def test_refuses_a_window():
    import torch
    from modgrad_amd.q4k import BackendError
    rng = np.random.default_rng(38)
    both = build(rng, 64, [1, 1], 1, 64, 16, "i8")
    both.call([65, 65], [1, 1], True)
    x = torch.zeros(2, 64, device="cuda")
    for bad in (dict(window=5), dict(sinks=5), dict(window=5, sinks=5)):
        with pytest.raises(BackendError):
            both.gpu.attend(x.data_ptr(), 64, 1, x.data_ptr(), 64, 2, 1, shared=64, **bad)
        with pytest.raises(BackendError):
            both.gpu.op_attend(x.data_ptr(), 64, 1, x.data_ptr(), 64, 2, 1, x, shared=64, **bad)
    with pytest.raises(BackendError):  # a workspace of another call
        both.gpu.attend(x.data_ptr(), 64, 1, x.data_ptr(), 64, 2, 1, shared=64, workspace=x.view(torch.uint8))
    with pytest.raises(BackendError):
        both.gpu.attend(x.data_ptr(), 64, 1, x.data_ptr(), 64, 2, 1, shared=-64)
