"""launch_block_norm_ex and modgrad_amd.norm refuse bad arguments before any device
call (no GPU)."""
import ctypes

import pytest

from modgrad_amd import _lib

INVALID = _lib.hipErrorInvalidValue
FAKE = 0x10000  # never dereferenced: every call below fails validation first
NORM = dict(post_w=FAKE, norm_w=FAKE, h_scale=1.0, x_scale=1.0, eps=1e-6, hidden=64)
CALL = dict(h=FAKE, h_stride=64, x=2 * FAKE, x_stride=64, gate=3 * FAKE, gate_stride=0, h_out=4 * FAKE, h_out_stride=64,
            y=5 * FAKE, y_stride=64, y_type=0, rows=3)
NAN, INF = float("nan"), float("inf")
BAD = [
    dict(post_w=FAKE + 2), dict(norm_w=FAKE + 1), dict(norm_w=None), dict(h_scale=NAN), dict(h_scale=INF),
    dict(x_scale=-INF), dict(x_scale=NAN), dict(eps=-1e-6), dict(eps=NAN), dict(eps=INF), dict(hidden=0),
    dict(hidden=-4), dict(hidden=(1 << 30) + 1, h_stride=1 << 31, x_stride=1 << 31, h_out_stride=1 << 31, y_stride=1 << 31),
    dict(h=None), dict(h=FAKE + 2), dict(x=2 * FAKE + 2), dict(x=None), dict(x=None, gate=None), dict(x=None, post_w=None),
    dict(gate=3 * FAKE + 1), dict(h_out=4 * FAKE + 2), dict(y=5 * FAKE + 2), dict(y=5 * FAKE + 1, y_type=1),
    dict(h_out=None, y=None), dict(h_stride=63), dict(x_stride=63), dict(gate_stride=63), dict(gate_stride=-64),
    dict(h_out_stride=63), dict(y_stride=63), dict(y_type=2), dict(y_type=-1), dict(rows=0), dict(rows=-1),
    dict(h_out=FAKE, h_out_stride=65), dict(h_out=2 * FAKE), dict(y=2 * FAKE), dict(y=FAKE), dict(y=4 * FAKE),
    dict(y=3 * FAKE), dict(h_out=3 * FAKE)]


@pytest.fixture(scope="module")
def L():
    return _lib.load()


@pytest.mark.parametrize("bad", BAD)
def test_refuses(L, bad):
    n = dict(NORM, post_w=6 * FAKE, norm_w=7 * FAKE)
    n.update({k: v for k, v in bad.items() if k in n})
    c = dict(CALL)
    c.update({k: v for k, v in bad.items() if k in c})
    norm = _lib.BlockNorm(**n)
    assert L.launch_block_norm_ex(ctypes.byref(norm), *c.values(), None) == INVALID
    d = dict(c)
    args = _lib.BlockNormArgs(norm, d["h"], d["x"], d["gate"], d["h_out"], d["y"], d["h_stride"], d["x_stride"],
                              d["gate_stride"], d["h_out_stride"], d["y_stride"], d["y_type"], d["rows"])
    op = _lib.OpDesc(op=_lib.OP_BLOCK_NORM, w=ctypes.addressof(args))
    out = ctypes.c_void_p()
    assert L.mgq_chain_create_ops(ctypes.byref(op), 1, ctypes.byref(out)) == INVALID and out.value is None


def test_refuses_null(L):
    assert L.launch_block_norm_ex(None, *CALL.values(), None) == INVALID
    op, out = _lib.OpDesc(op=_lib.OP_BLOCK_NORM), ctypes.c_void_p()
    assert L.mgq_chain_create_ops(ctypes.byref(op), 1, ctypes.byref(out)) == INVALID
