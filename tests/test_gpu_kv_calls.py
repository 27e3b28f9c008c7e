"""Calls on the 8-bit cache at the edges of what its documentation allows."""
import numpy as np
import pytest

from tests import kv_reference as ref
from tests.gpu_util import dev, host
from tests.test_gpu_kvcache import Both, check, fill, note, random_cache, torch_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 3])
@pytest.mark.parametrize("place", [False, True])
def test_append_copies_the_queries_of_idle_slots(new, place):
    """Without a rotary table q is copied as it is, at positions before the first
    token too (an idle slot, more rows than tokens)."""
    import torch
    note(f"append without a table, idle slots new={new} in place={place}")
    rng = np.random.default_rng(new)
    both = Both(rng, 4, 2, 1, 64, 16, "i8")
    lens, rows = [0, 5, new - 1, 32], 4 * new
    both.call(lens, [new] * 4, new == 1)
    kv = torch.randn(rows, 128, device="cuda")
    q = rng.standard_normal((rows, 2 * 64)).astype(np.float32)
    qt = dev(q)
    out = qt if place else torch.full((rows, 128), 7.0, device="cuda")
    both.gpu.append(kv.data_ptr(), kv.data_ptr() + 256, 128, rows, new, q=qt.data_ptr(), q_stride=128,
                    q_out=out.data_ptr(), q_out_stride=128, n_q_heads=2)
    assert np.array_equal(host(out), q)


def test_attention_of_a_large_batch_with_long_tables():
    """A piece of 2048 tokens beside hundreds of slots whose tables hold 131072
    tokens: more tiles than 32 bits count, of which few are there."""
    import torch
    from modgrad_amd.kvcache import KvCache
    note("attention of a large batch with long tables")
    rng = np.random.default_rng(1)
    both = Both(rng, 3, 40, 2, 64, 64, "i8")
    gen = random_cache(both, 1)
    seqs, lens, news = 600, [0] * 600, [0] * 600
    table = np.full((seqs, 2048), -1, np.int32)
    for b, at, n, m in ((0, 17, 2100, 2048), (1, 300, 900, 1), (2, 599, 2500, 130)):
        table[at, :40], lens[at], news[at] = both.ref.table[b], n, m
    cache = KvCache.wrap(both.k, both.v, both.ks, both.vs, dev(table), dev(np.array(lens, np.int32)),
                         dev(np.concatenate([[0], np.cumsum(news)]).astype(np.int32)), "i8")
    rows, hq = sum(news), 16
    q = torch.randn(rows, hq, 64, generator=gen, device="cuda") * 2
    want, tol = torch_attention(both, q, [2100, 900, 2500], [2048, 1, 130], 0.125)
    for f16 in (False, True):
        out = torch.full((rows + 1, hq, 64), 7.0, device="cuda", dtype=torch.float16 if f16 else torch.float32)
        cache.attend(q.data_ptr(), hq * 64, hq, out.data_ptr(), hq * 64, rows, 2048, out_f16=f16)
        check(host(out[:rows]).astype(np.float64), host(want), host(tol), f16)
        assert bool((out[rows] == 7.0).all())


def test_set_lengths_without_counts_reaches_recorded_calls():
    """A chain recorded with counts, replayed after lengths were set with one new
    token each: the rows are those of one each."""
    import torch
    from modgrad_amd.kvcache import KvCache
    from modgrad_amd.q4k import Chain
    note("set_lengths without counts under a recorded call")
    rng = np.random.default_rng(2)
    c, fresh = (KvCache.new(n_pages=8, page_tokens=16, n_kv_heads=1, head_dim=64, n_seqs=2, max_pages=4) for _ in range(2))
    x = dev(rng.standard_normal((8, 2, 64)).astype(np.float32))
    q = dev(rng.standard_normal((8, 4, 64)).astype(np.float32))
    outs = [torch.zeros(8, 4, 64, device="cuda") for _ in range(2)]
    c.set_lengths([5, 3], [5, 3])
    ws = c.attention_workspace(4, 8, 8)
    chain = Chain.from_ops([c.op_append(x.data_ptr(), x.data_ptr() + 256, 128, 8, 8),
                            c.op_attend(q.data_ptr(), 256, 4, outs[0].data_ptr(), 256, 8, 8, ws)])
    for lens, new in (([5, 3], [5, 3]), ([6, 4], None), ([7, 5], None), ([9, 11], [2, 6])):
        c.set_lengths(lens, new)
        chain.launch()
        fresh.set_lengths(lens, new)
        rows, most = (2, 1) if new is None else (8, 6)
        fresh.append(x.data_ptr(), x.data_ptr() + 256, 128, rows, most)
        fresh.attend(q.data_ptr(), 256, 4, outs[1].data_ptr(), 256, rows, most)
        for a, b in ((c.k, fresh.k), (c.v, fresh.v), (c.k_scale, fresh.k_scale), (c.v_scale, fresh.v_scale),
                     (outs[0][:rows], outs[1][:rows])):
            assert np.array_equal(host(a), host(b)), (lens, new)


@pytest.mark.parametrize("lens", [[48, 48], [16, 65], [32, 80]])
def test_set_lengths_that_are_refused_take_no_pages(lens):
    """More pages than there are, or than a table has: none are taken for the
    sequences before the one that does not fit."""
    from modgrad_amd.kvcache import KvCache
    from modgrad_amd.q4k import BackendError
    note(f"refused lengths {lens}")
    c = KvCache.new(n_pages=5, page_tokens=16, n_kv_heads=1, head_dim=64, n_seqs=2, max_pages=4)
    c.set_lengths([7, 9])
    was = host(c.page_table).copy()
    with pytest.raises(BackendError):
        c.set_lengths(lens)
    assert len(c._free) == 3 and np.array_equal(host(c.page_table), was) and list(host(c.seq_len)) == [7, 9]
    c.set_lengths([64, 9])
    assert len(c._free) == 0


def test_workspaces_elsewhere_are_refused():
    """Memory of the host, and a view that says more bytes than it has."""
    import torch
    from modgrad_amd.kvcache import KvCache
    from modgrad_amd.q4k import BackendError
    note("workspaces elsewhere")
    c = KvCache.new(4, 16, 1, 64, 1, 4)
    c.set_lengths([5])
    n = c.attention_workspace(1, 1, 1).nbytes
    p = torch.zeros(64, device="cuda").data_ptr()
    for ws in (torch.empty(n, dtype=torch.uint8), torch.zeros(1, dtype=torch.uint8, device="cuda").expand(n)):
        with pytest.raises(BackendError):
            c.attend(p, 64, 1, p, 64, 1, 1, workspace=ws)
        with pytest.raises(BackendError):
            c.op_attend(p, 64, 1, p, 64, 1, 1, ws)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("new,n", [(1, 100), (1, 1500), (60, 100), (60, 1500)])
@pytest.mark.parametrize("loud", [0, 2, 5])
def test_attention_over_pages_of_all_loudness(loud, new, n, dim, fmt):
    """A page of V whose scale is 2^118 among others of 0.02, 1e-8 and 0: the quiet
    tokens' values vanish beside it, their part of the probabilities does not."""
    import torch
    note(f"pages of all loudness loud={loud} new={new} n={n} dim={dim} {fmt}")
    rng = np.random.default_rng(loud + dim)
    both = Both(rng, 1, -(-n // 16), 1, dim, 16, fmt)
    fill(both, rng, [n])
    ids = both.ref.table[0]
    both.ref.vs[ids[1]] *= np.float32(1e-8)
    both.ref.vs[ids[3]], both.ref.v[ids[3]] = 0, 0
    both.ref.vs[ids[loud]] = 2.0 ** 118
    both.vs.copy_(torch.from_numpy(both.ref.vs))
    both.v.copy_(torch.from_numpy(both.ref.v))
    q = rng.standard_normal((new, 4, dim)).astype(np.float32)
    both.call([n], [new], new == 1)
    out = torch.full((new, 4, dim), 7.0, device="cuda")
    both.gpu.attend(dev(q).data_ptr(), 4 * dim, 4, out.data_ptr(), 4 * dim, new, new)
    want, tol = both.ref.attend(q, [n], [new], dim ** -0.5)
    # A probability goes into the products times its page's scale, as w of 2^14 and
    # more (or 2^13.5) for the row's largest, in two f16 halves: the second one's step
    # is 2^-24 at the least, so that w is off by up to 2^-25, 2^-38 of the largest.
    k, _, _ = both.ref.read(0, 0, n)
    sc = dim ** -0.5 * q.reshape(-1, dim).astype(np.float64) @ k.T
    sc[np.arange(n) > n - new + np.arange(new).repeat(4)[:, None]] = -np.inf
    p = np.exp(sc - sc.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    largest = (p * both.ref.vs[ids, 0].astype(np.float64).repeat(16)[:n]).max(1)
    tol += (n * 2.0 ** -38 * ref.MOST[fmt] * largest).reshape(new, 4, 1)
    check(host(out).astype(np.float64), want, tol, False)
