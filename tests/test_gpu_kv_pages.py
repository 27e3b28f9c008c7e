"""A cache that hands its pages out, as a server runs it: a prompt whose pages a batch shares,
slots that leave and join it; a conversation whose middle is given back behind its first
tokens. Against the 64-bit reference over the cache's bytes."""
import numpy as np
import pytest

from tests import kv_attend_reference as ref
from tests.gpu_util import dev, host
from tests.test_gpu_kvcache import check, note
from tests.test_gpu_layer_ops import reference_of

pytestmark = pytest.mark.gpu


def step(cache, rng, lens, new, hq, heads, dim, stream=None, **attend):
    """Appends new random tokens and attends; the results against the reference."""
    import torch
    rows = sum(new)
    kv = rng.standard_normal((rows, 2, heads, dim)).astype(np.float32)
    q = (2 * rng.standard_normal((rows, hq, dim))).astype(np.float32)
    kt, qt, out = dev(kv), dev(q), torch.empty(rows, hq * dim, device="cuda")
    torch.cuda.synchronize()
    cache.set_lengths(lens, new, stream=stream)
    cache.append(kt.data_ptr(), kt.data_ptr() + 4 * heads * dim, 2 * heads * dim, rows, max(new), stream=stream)
    cache.attend(qt.data_ptr(), hq * dim, hq, out.data_ptr(), hq * dim, rows, max(new), stream=stream, **attend)
    torch.cuda.synchronize()
    want, tol = ref.attend(reference_of(cache), q, lens, new, dim ** -0.5, 0.0, attend.get("window", 0),
                           attend.get("sinks", 0))
    check(host(out).reshape(want.shape), want, tol, False)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_batch_that_shares_a_prompt(fmt):
    import torch
    from modgrad_amd.kvcache import KvCache
    note(f"a batch that shares a prompt {fmt}")
    rng = np.random.default_rng(61)
    seqs, heads, hq, dim, page, prefix = 20, 2, 6, 64, 32, 1024
    stream = torch.cuda.Stream()
    cache = KvCache.new(prefix // page + 4 * seqs, page, heads, dim, seqs, prefix // page + 4, fmt=fmt)
    lens = [prefix + 5] + [0] * (seqs - 1)
    step(cache, rng, lens, lens, hq, heads, dim, stream=stream)
    for b in range(1, seqs - 1):
        cache.share(b, 0, prefix, stream=stream)
        lens[b] = prefix
    free = len(cache._free)
    for _ in range(3):
        new = [int(n) for n in rng.integers(1, 9, seqs - 1)] + [0]
        lens = [a + b for a, b in zip(lens, new)]
        step(cache, rng, lens, new, hq, heads, dim, stream=stream, shared=prefix)
    common = host(cache.page_table)[1, :prefix // page].copy()
    # the first one leaves: the prompt stays, and another joins behind it
    cache.release(0, stream=stream)
    lens[0] = 0
    cache.share(seqs - 1, 5, prefix, stream=stream)
    lens[seqs - 1] = prefix
    for _ in range(2):
        new = [0] + [int(n) for n in rng.integers(1, 9, seqs - 1)]
        lens = [a + b for a, b in zip(lens, new)]
        step(cache, rng, lens, new, hq, heads, dim, stream=stream, shared=prefix)
    assert np.array_equal(host(cache.page_table)[seqs - 1, :len(common)], common)
    # a stranger has pages of its own
    lens[0], new = 40, [40] + [1] * (seqs - 1)
    lens[1:] = [n + 1 for n in lens[1:]]
    step(cache, rng, lens, new, hq, heads, dim, stream=stream)
    assert not set(host(cache.page_table)[0, :2]) & set(common) and len(cache._free) < free
    for b in range(seqs):
        cache.release(b, stream=stream)
    assert len(cache._free) == cache.n_pages and np.all(host(cache.page_table) == -1)


def test_conversation_without_its_middle():
    from modgrad_amd.kvcache import KvCache
    note("a conversation without its middle")
    rng = np.random.default_rng(62)
    heads, hq, dim, page, window, sinks = 2, 8, 128, 16, 100, 20
    cache = KvCache.new(14, page, heads, dim, 1, 40)  # 14 pages for 640 positions
    n = 0
    for m in [60, 1, 1, 30] + [25] * 18:
        n += m
        # rows of this step see the first 20 and from n - m - window + 1 on
        cache.give_back(0, 32, max(32, n - m - window + 1))
        step(cache, rng, [n], [m], hq, heads, dim, window=window, sinks=sinks)
    assert n > 500 and np.all(host(cache.page_table)[0, 2:20] == -1)
