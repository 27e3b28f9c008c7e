"""Attention over the cache with first tokens that stay visible behind the window,
against the 64-bit reference of tests/kv_attend_reference.py."""
import numpy as np
import pytest

from tests import kv_attend_reference as ref
from tests.gpu_util import dev, host
from tests.test_gpu_kvcache import Both, check, fill, note

pytestmark = pytest.mark.gpu

CASES = [
    # lengths, new tokens, kv heads, group, dim, page, softcap, window, sinks
    ([1], [1], 1, 1, 64, 16, 0, 1, 1),
    ([300], [1], 2, 7, 128, 64, 0, 50, 4),
    ([700, 65, 64, 3, 0, 1], [1, 1, 1, 1, 1, 1], 2, 3, 64, 32, 0, 64, 64),
    ([1500, 900], [1, 1], 1, 4, 96, 32, 30.0, 200, 65),
    ([2200], [1], 2, 4, 256, 128, 0, 1, 100),          # only its own and the first
    ([640], [1], 1, 8, 128, 16, 0, 320, 300),          # the two meet in a tile
    ([640], [1], 1, 8, 128, 16, 0, 320, 320),          # they touch
    ([640], [1], 1, 8, 128, 16, 0, 320, 5000),         # more first tokens than there are
    ([4000, 77], [1, 1], 1, 2, 64, 16, 0, 700, 129),   # long lists, split
    ([500], [5], 2, 2, 128, 64, 0, 33, 7),
    ([900, 40, 0, 333], [3, 2, 0, 1], 2, 4, 128, 16, 0, 100, 16),
    ([777], [300], 2, 3, 128, 64, 0, 90, 10),          # prompts
    ([2000, 129, 150], [150, 129, 1], 1, 7, 64, 32, 0, 130, 70),
    ([1100], [400], 2, 2, 256, 32, 50.0, 64, 1),
    ([900, 310], [200, 11], 3, 1, 96, 16, 0, 333, 200),
    ([400], [400], 1, 6, 128, 128, 0, 20, 3),
]


def run(both, q, lens, new, hq, dim, f16, window, sinks, cap, workspace=None):
    import torch
    rows = sum(new)
    out = torch.full((rows + 1, hq * dim + 3), 7.0, device="cuda", dtype=torch.float16 if f16 else torch.float32)
    qt = dev(q)
    both.gpu.attend(qt.data_ptr(), hq * dim, hq, out.data_ptr(), hq * dim + 3, rows, max(new), scale=dim ** -0.5,
                    softcap=cap, window=window, sinks=sinks, out_f16=f16, workspace=workspace)
    got = host(out)
    assert np.all(got[rows] == 7) and np.all(got[:, hq * dim:] == 7)
    return got[:rows, :hq * dim].reshape(rows, hq, dim)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("k", range(len(CASES)))
def test_sinks(k, fmt, f16):
    lens, new, heads, group, dim, page, cap, window, sinks = CASES[k]
    note(f"sinks {CASES[k]} {fmt} f16={f16}")
    rng = np.random.default_rng(90 + k)
    both = Both(rng, len(lens), max(1, -(-max(lens) // page)), heads, dim, page, fmt)
    fill(both, rng, lens)
    both.same()
    both.call(lens, new)
    hq = heads * group
    q = (2 * rng.standard_normal((sum(new), hq, dim))).astype(np.float32)
    got = run(both, q, lens, new, hq, dim, f16, window, sinks, cap)
    want, tol = ref.attend(both.ref, q, lens, new, dim ** -0.5, cap, window, sinks)
    check(got, want, tol, f16)
    assert np.array_equal(run(both, q, lens, new, hq, dim, f16, window, sinks, cap), got)  # the same bits again


def test_reference_agrees_with_the_plain_one():
    """Without sinks the two references are the same numbers."""
    rng = np.random.default_rng(2)
    both = Both(rng, 2, 6, 2, 64, 16, "i8")
    fill(both, rng, [90, 40])
    q = rng.standard_normal((7, 4, 64)).astype(np.float32)
    for window in (0, 20):
        a, ta = both.ref.attend(q, [90, 40], [5, 2], 0.125, 0.0, window)
        b, tb = ref.attend(both.ref, q, [90, 40], [5, 2], 0.125, 0.0, window)
        assert np.allclose(a, b, rtol=1e-12, atol=1e-14) and np.allclose(ta, tb, rtol=1e-9)


@pytest.mark.parametrize("new", [1, 40])
def test_pages_given_back(new):
    """The middle of a conversation in no page: nothing of it is read as a token."""
    import torch
    note(f"sinks with pages given back new={new}")
    rng = np.random.default_rng(6)
    n, window, sinks, page = 1000, 100, 20, 16
    both = Both(rng, 1, 64, 2, 128, page, "i8")
    fill(both, rng, [n])
    both.call([n], [new])
    q = (2 * rng.standard_normal((new, 6, 128))).astype(np.float32)
    full = run(both, q, [n], [new], 6, 128, False, window, sinks, 0.0)
    first = (n - new - window + 1) // page
    both.ref.table[0, 2:first] = -1
    both.gpu.page_table.copy_(torch.from_numpy(both.ref.table))
    got = run(both, q, [n], [new], 6, 128, False, window, sinks, 0.0)
    assert np.array_equal(got, full)
    want, tol = ref.attend(both.ref, q, [n], [new], 128 ** -0.5, 0.0, window, sinks)
    check(got, want, tol, False)
    # and the first page too: its tokens are no longer seen, the window is
    both.ref.table[0, 0] = 10 ** 6
    both.gpu.page_table.copy_(torch.from_numpy(both.ref.table))
    got = run(both, q, [n], [new], 6, 128, False, window, sinks, 0.0)
    want, tol = ref.attend(both.ref, q, [n], [new], 128 ** -0.5, 0.0, window, sinks)
    check(got, want, tol, False)


@pytest.mark.parametrize("new", [1, 60])
def test_lengths_past_the_table(new):
    """A sequence longer than its table: the first tokens are still seen, by rows whose
    window lies behind the table too."""
    note(f"sinks past the table new={new}")
    rng = np.random.default_rng(7)
    both = Both(rng, 2, 4, 1, 64, 16, "e4m3")
    fill(both, rng, [64, 64])
    both.call([500, 64], [new, new])
    q = rng.standard_normal((2 * new, 3, 64)).astype(np.float32)
    got = run(both, q, None, [new, new], 3, 64, False, 100, 10, 0.0)
    want, tol = ref.attend(both.ref, q, [500, 64], [new, new], 0.125, 0.0, 100, 10)
    check(got, want, tol, False)


def test_without_a_window_and_without_sinks():
    """sinks change nothing where everything is seen, or where there are none."""
    note("sinks without a window")
    rng = np.random.default_rng(8)
    both = Both(rng, 2, 20, 1, 128, 16, "i8")
    lens, new = [300, 200], [1, 1]
    fill(both, rng, lens)
    both.call(lens, new)
    q = rng.standard_normal((2, 4, 128)).astype(np.float32)
    plain = run(both, q, lens, new, 4, 128, False, 0, 0, 0.0)
    assert np.array_equal(run(both, q, lens, new, 4, 128, False, 0, 40, 0.0), plain)
    # as many first tokens as there are: nothing is hidden, however short the window
    want, tol = ref.attend(both.ref, q, lens, new, 128 ** -0.5)
    check(run(both, q, lens, new, 4, 128, False, 1, 2 ** 31 - 1, 0.0), want, tol, False)
    check(run(both, q, lens, new, 4, 128, False, 2 ** 31 - 1, 2 ** 31 - 1, 0.0), want, tol, False)


@pytest.mark.parametrize("new", [1, 50])
def test_stream_graph_and_chain(new):
    """A recorded call and a captured one replay on new lengths; the op of a chain."""
    import torch
    from modgrad_amd.q4k import Chain
    note(f"sinks recorded new={new}")
    rng = np.random.default_rng(9)
    heads, hq, dim, page, window, sinks = 2, 4, 64, 16, 60, 9
    both = Both(rng, 3, 40, heads, dim, page, "e4m3")
    lens = [400, 150, 620]
    fill(both, rng, lens)
    rows = 3 * new
    qt = torch.empty(rows, hq * dim, device="cuda")
    outs = [torch.empty(rows, hq * dim, device="cuda") for _ in range(2)]
    both.call(lens, [new] * 3)
    ws = [both.gpu.attention_workspace(hq, rows, new) for _ in range(2)]
    s = torch.cuda.Stream()
    chain = Chain.from_ops([both.gpu.op_attend(qt.data_ptr(), hq * dim, hq, outs[0].data_ptr(), hq * dim, rows, new,
                                               ws[0], window=window, sinks=sinks)])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        both.gpu.attend(qt.data_ptr(), hq * dim, hq, outs[1].data_ptr(), hq * dim, rows, new, window=window,
                        sinks=sinks, workspace=ws[1], stream=s)
    for now in ([400, 150, 620], [new, 100, 300], [350, new, 610]):
        q = rng.standard_normal((rows, hq, dim)).astype(np.float32)
        qt.copy_(torch.from_numpy(q.reshape(rows, -1)))
        both.length.copy_(torch.tensor(now, dtype=torch.int32))
        torch.cuda.synchronize()
        chain.launch()
        g.replay()
        want, tol = ref.attend(both.ref, q, now, [new] * 3, dim ** -0.5, 0.0, window, sinks)
        for o in outs:
            check(host(o).reshape(q.shape), want, tol, False)


def test_many_sequences():
    """Hundreds of ragged sequences, windows and first tokens in equal runs of tiles."""
    note("sinks: 300 sequences")
    rng = np.random.default_rng(10)
    lens = [int(n) for n in rng.integers(1, 260, 300)]
    both = Both(rng, 300, 17, 1, 64, 16, "i8")
    fill(both, rng, lens)
    new = [1] * 300
    both.call(lens, new)
    q = rng.standard_normal((300, 2, 64)).astype(np.float32)
    got = run(both, q, lens, new, 2, 64, False, 70, 33, 0.0)
    want, tol = ref.attend(both.ref, q, lens, new, 0.125, 0.0, 70, 33)
    check(got, want, tol, False)
