"""launch_kv_attention_sinks_ex refuses bad arguments before any device call (no GPU)."""
import ctypes

import pytest

from modgrad_amd import _lib
from tests.test_kvcache_cpu import BAD_CACHE, BAD_CALL, FAKE, INVALID, cache


@pytest.fixture(scope="module")
def L():
    return _lib.load()


def attend(L, c, q=FAKE, qs=512, hq=4, out=FAKE, os=512, kind=0, n=7, new=5, scale=0.1, cap=0.0, win=9, sinks=4,
           ws=FAKE, nbytes=1 << 40):
    op = _lib.KvAttentionSinksArgs(_lib.KvAttentionArgs(c, q, out, ws, nbytes, qs, os, hq, kind, n, new, win, scale, cap),
                                   sinks)
    d, chain = _lib.OpDesc(op=_lib.OP_KV_ATTENTION_SINKS, w=ctypes.addressof(op)), ctypes.c_void_p()
    codes = (L.mgq_chain_create_ops(ctypes.byref(d), 1, ctypes.byref(chain)),
             L.launch_kv_attention_sinks_ex(ctypes.byref(c), q, qs, hq, out, os, kind, n, new, scale, cap, win, sinks, ws,
                                            nbytes, None))
    assert chain.value is None
    return codes


@pytest.mark.parametrize("bad", BAD_CACHE + BAD_CALL)
def test_bad_cache(L, bad):
    assert attend(L, cache(**bad)) == (INVALID, INVALID)


@pytest.mark.parametrize("bad", [
    dict(sinks=-1), dict(sinks=-2 ** 31), dict(win=-1), dict(q=None), dict(qs=511), dict(out=FAKE + 2), dict(os=511),
    dict(kind=2), dict(hq=3), dict(n=0), dict(new=8), dict(scale=float("nan")), dict(cap=-1.0), dict(ws=None),
    dict(ws=FAKE + 8), dict(nbytes=0)])
def test_refuses(L, bad):
    assert attend(L, cache(), **bad) == (INVALID, INVALID)


def test_refuses_null(L):
    assert L.launch_kv_attention_sinks_ex(None, FAKE, 512, 4, FAKE, 512, 0, 7, 5, 0.1, 0.0, 9, 4, FAKE, 1 << 40,
                                          None) == INVALID
    d, chain = _lib.OpDesc(op=_lib.OP_KV_ATTENTION_SINKS), ctypes.c_void_p()
    assert L.mgq_chain_create_ops(ctypes.byref(d), 1, ctypes.byref(chain)) == INVALID
