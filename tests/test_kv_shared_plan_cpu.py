"""How attention behind a shared prefix is gone about (mgq_kv_attention_shared_plan): the
sizes of the GPU tests take the ways that their names say. Host only, no GPU."""
import ctypes

import pytest

from modgrad_amd import _lib
from tests.test_kvcache_cpu import INVALID, cache


@pytest.fixture(scope="module")
def L():
    return _lib.load()


def ask(c, hq, n, new, shared, kind=0):
    p = _lib.KvSharedPlan()
    made = _lib.load().mgq_kv_attention_shared_plan(ctypes.byref(c), hq, kind, n, new, shared, ctypes.byref(p))
    assert made in (0, INVALID)
    return p if made == 0 else None


def cache_of(seqs, heads, dim, page, fmt, max_pages):
    return cache(page_stride=heads * page * dim, page_tokens=page, n_kv_heads=heads, head_dim=dim, format=fmt, n_seqs=seqs,
                 max_pages=max_pages)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("fmt", [0, 1])
def test_ways_of_the_gpu_tests(fmt, kind):
    from tests.test_gpu_kv_shared_reach import CASES, layout
    for name, (way, prefix, seqs, _, heads, group, dim, page, _) in CASES.items():
        own, lens, new, ahead = layout(name)
        n = sum(new) + 2 * ahead
        c = cache_of(seqs, heads, dim, page, fmt, -(-(prefix + max(own)) // page))
        p = ask(c, heads * group, n, max(new), prefix, kind)
        assert p.way == way, name
        assert p.tiles == prefix // 64
        blocks = -(-n * group // (16 if way == _lib.SHARED_FEW else 128))
        assert p.blocks == blocks
        if way == _lib.SHARED_RUNS:  # some run goes on into the next block
            assert any(r * p.run // p.tiles != (min((r + 1) * p.run, blocks * p.tiles) - 1) // p.tiles
                       for r in range(-(-blocks * p.tiles // p.run)))
            assert blocks > 2 and p.tiles % p.run


def test_plain(L):
    """Short prefixes, and none: what the plain call does."""
    c = cache(max_pages=40, n_seqs=64)
    for shared in (0, 63, 64):
        p = ask(c, 4, 320, 5, shared)
        assert (p.way, p.tiles, p.blocks, p.run) == (_lib.SHARED_PLAIN, 0, 0, 0)
        assert p.own_groups > 0
    assert ask(c, 4, 320, 5, 2048).way != _lib.SHARED_PLAIN


def test_refuses(L):
    c = cache()
    for bad in (dict(hq=3), dict(n=0), dict(new=0), dict(shared=-1), dict(kind=2), dict(kind=-1), dict(n=1 << 28)):
        args = dict(hq=4, n=7, new=5, shared=128, kind=0)
        args.update(bad)
        assert ask(c, **args) is None
    assert L.mgq_kv_attention_shared_plan(ctypes.byref(c), 4, 0, 7, 5, 128, None) == INVALID
    assert ask(cache(head_dim=80), 4, 7, 5, 128) is None
    p = _lib.KvSharedPlan()
    assert L.mgq_kv_attention_shared_plan(None, 4, 0, 7, 5, 128, ctypes.byref(p)) == INVALID
