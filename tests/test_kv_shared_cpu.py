"""launch_kv_attention_shared_ex refuses bad arguments before any device call (no GPU)."""
import ctypes

import pytest

from modgrad_amd import _lib
from tests.test_kvcache_cpu import BAD_CACHE, BAD_CALL, FAKE, INVALID, cache


@pytest.fixture(scope="module")
def L():
    return _lib.load()


def size(L, c, hq=4, n=7, new=5, shared=128):
    return L.mgq_kv_attention_shared_workspace_bytes(ctypes.byref(c), hq, n, new, shared)


def attend(L, c, q=FAKE, qs=512, hq=4, out=FAKE, os=512, kind=0, n=7, new=5, scale=0.1, cap=0.0, shared=128, ws=FAKE,
           nbytes=1 << 40, win=0):
    op = _lib.KvAttentionSharedArgs(_lib.KvAttentionArgs(c, q, out, ws, nbytes, qs, os, hq, kind, n, new, win, scale, cap),
                                    shared)
    d, chain = _lib.OpDesc(op=_lib.OP_KV_ATTENTION_SHARED, w=ctypes.addressof(op)), ctypes.c_void_p()
    made = L.mgq_chain_create_ops(ctypes.byref(d), 1, ctypes.byref(chain))
    assert chain.value is None
    if win:
        return made
    assert made == L.launch_kv_attention_shared_ex(ctypes.byref(c), q, qs, hq, out, os, kind, n, new, scale, cap, shared,
                                                   ws, nbytes, None)
    return made


@pytest.mark.parametrize("bad", BAD_CACHE + BAD_CALL)
def test_bad_cache(L, bad):
    assert attend(L, cache(**bad)) == INVALID
    if bad in BAD_CACHE:
        assert size(L, cache(**bad)) == 0


@pytest.mark.parametrize("bad", [
    dict(shared=-1), dict(shared=-2 ** 31), dict(q=None), dict(qs=511), dict(out=FAKE + 2), dict(os=511), dict(kind=2),
    dict(hq=3), dict(n=0), dict(new=8), dict(scale=float("nan")), dict(cap=-1.0), dict(ws=None), dict(ws=FAKE + 8),
    dict(nbytes=0), dict(win=5), dict(win=-1)])
def test_refuses(L, bad):
    assert attend(L, cache(), **bad) == INVALID


def test_workspace(L):
    c, big = cache(max_pages=40, n_seqs=64), dict(n=320, shared=1024)
    plain = L.mgq_kv_attention_workspace_bytes(ctypes.byref(c), 4, 5)
    need = size(L, c, **big)
    assert need > plain > 0 and need % 16 == 0
    assert attend(L, c, nbytes=need - 1, **big) == INVALID
    # no whole tile of 64 tokens, or so few that every sequence reads them: the plain call's
    assert size(L, c, n=320, shared=63) == plain and size(L, c, n=320, shared=64) == plain
    assert size(L, c, n=320, shared=2 ** 31 - 1) == size(L, c, n=320, shared=40 * 64)
    for bad in (dict(hq=3), dict(n=0), dict(n=-1), dict(new=0), dict(shared=-1), dict(n=1 << 28)):
        assert size(L, c, **bad) == 0
    # room for the states of every block of 128 query rows and its parts of the prefix
    big = cache(n_seqs=64, max_pages=4096, n_kv_heads=4, page_stride=4 * 64 * 128)
    assert size(L, big, hq=28, n=64 * 300, new=300, shared=100000) >= 64 * 300 * 28 * 130 * 4


def test_refuses_null(L):
    assert L.mgq_kv_attention_shared_workspace_bytes(None, 4, 7, 5, 128) == 0
    assert L.launch_kv_attention_shared_ex(None, FAKE, 512, 4, FAKE, 512, 0, 7, 5, 0.1, 0.0, 128, FAKE, 1 << 40,
                                           None) == INVALID
    d, chain = _lib.OpDesc(op=_lib.OP_KV_ATTENTION_SHARED), ctypes.c_void_p()
    assert L.mgq_chain_create_ops(ctypes.byref(d), 1, ctypes.byref(chain)) == INVALID


def test_sizes_that_go_through_the_prefix_once(L):
    """The GPU tests of those paths are of sizes that take them: room for their states."""
    from tests.test_gpu_kv_shared_paths import CASES, WAYS
    cases = [(prefix, seqs, new, heads, group, dim, page) for prefix, seqs, _, new, heads, group, dim, page, _ in
             CASES.values()] + [(1024, seqs, new, 4, group, 64, 16) for seqs, new, group in WAYS.values()]
    for prefix, seqs, new, heads, group, dim, page in cases:
        for fmt in (0, 1):
            c = cache(page_stride=heads * page * dim, page_tokens=page, n_kv_heads=heads, head_dim=dim, format=fmt,
                      n_seqs=seqs, max_pages=prefix // page + 100)
            plain = L.mgq_kv_attention_workspace_bytes(ctypes.byref(c), heads * group, new)
            assert size(L, c, hq=heads * group, n=seqs * new, new=new, shared=prefix) > plain
