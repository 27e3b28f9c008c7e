"""Positions of several axes: refusals before any device call, sections from GGUF
files, and the reference's own pins (no GPU)."""
import ctypes

import numpy as np
import pytest

from modgrad_amd import _lib
from tests import rope_axes_reference as ref
from tests.test_kvcache_cpu import cache

INVALID = _lib.hipErrorInvalidValue
FAKE = 0x10000  # never dereferenced: every call below fails validation first


@pytest.fixture(scope="module")
def L():
    return _lib.load()


def axes(pos=FAKE, pos_stride=7, n_axes=3, sections=(16, 24, 24, 0), order=0, own=0):
    return _lib.RopeAxes(pos, pos_stride, n_axes, (ctypes.c_int * 4)(*sections), order, own)


BAD = [dict(pos=None), dict(pos=FAKE + 2), dict(pos_stride=6), dict(pos_stride=-7), dict(n_axes=0), dict(n_axes=5),
       dict(n_axes=2), dict(sections=(16, 24, 25, 0)), dict(sections=(16, -24, 72, 0)), dict(sections=(0, 0, 0, 0)),
       dict(sections=(16, 24, 23, 0)), dict(order=2), dict(order=-1), dict(own=2), dict(own=-1),
       dict(own=1, sections=(65, 0, 0, 0)), dict(own=1, sections=(64, 1, 0, 0)), dict(sections=(2 ** 31 - 1,) * 4)]


@pytest.mark.parametrize("bad", BAD)
def test_refuses(L, bad):
    a, r, c = axes(**bad), _lib.Rope(FAKE, 8, 128, 1), cache()
    out = ctypes.c_void_p()

    def create(op, args):
        d = _lib.OpDesc(op=op, w=ctypes.addressof(args))
        return L.mgq_chain_create_ops(ctypes.byref(d), 1, ctypes.byref(out))
    assert L.launch_rope_axes_ex(FAKE, FAKE, ctypes.byref(a), ctypes.byref(r), 7, 1, 128, 128, 128, None) == INVALID
    assert L.launch_kv_append_axes_ex(ctypes.byref(c), ctypes.byref(r), ctypes.byref(a), FAKE, FAKE, 256, FAKE, 512,
                                      FAKE, 512, 4, 7, 5, None) == INVALID
    assert create(_lib.OP_ROPE_AXES, _lib.RopeAxesArgs(FAKE, FAKE, a, r, 7, 1, 128, 128, 128)) == INVALID
    append = _lib.KvAppendArgs(c, r, FAKE, FAKE, FAKE, FAKE, 256, 512, 512, 4, 7, 5)
    assert create(_lib.OP_KV_APPEND_AXES, _lib.KvAppendAxesArgs(append, a)) == INVALID
    assert out.value is None


@pytest.mark.parametrize("bad", [dict(table=None), dict(table=FAKE + 2), dict(n_pos=0), dict(rot_dim=0),
                                 dict(rot_dim=126), dict(rot_dim=130), dict(style=2)])
def test_refuses_table(L, bad):
    r = _lib.Rope(**dict(dict(table=FAKE, n_pos=8, rot_dim=128, style=1), **bad))
    a, c = axes(), cache()
    assert L.launch_rope_axes_ex(FAKE, FAKE, ctypes.byref(a), ctypes.byref(r), 7, 1, 128, 128, 128, None) == INVALID
    assert L.launch_kv_append_axes_ex(ctypes.byref(c), ctypes.byref(r), ctypes.byref(a), FAKE, FAKE, 256, FAKE, 512,
                                      FAKE, 512, 4, 7, 5, None) == INVALID


def test_refuses_null_and_rows(L):
    a, r, c = axes(), _lib.Rope(FAKE, 8, 128, 1), cache()
    turn = lambda x=FAKE, y=FAKE, a=ctypes.byref(a), r=ctypes.byref(r), n=7, h=1, d=128, xs=128, ys=128: \
        L.launch_rope_axes_ex(x, y, a, r, n, h, d, xs, ys, None)  # noqa: E731
    for bad in (dict(x=None), dict(y=FAKE + 2), dict(a=None), dict(r=None), dict(n=0), dict(h=0), dict(d=126),
                dict(d=127), dict(xs=127), dict(ys=127), dict(ys=130), dict(n=8)):
        assert turn(**bad) == INVALID, bad
    add = lambda c=ctypes.byref(c), a=ctypes.byref(a), r=ctypes.byref(r), k=FAKE, n=7, new=5, kvs=256: \
        L.launch_kv_append_axes_ex(c, r, a, k, FAKE, kvs, FAKE, 512, FAKE, 512, 4, n, new, None)  # noqa: E731
    for bad in (dict(c=None), dict(a=None), dict(r=None), dict(k=None), dict(n=8), dict(new=0), dict(new=8), dict(kvs=255)):
        assert add(**bad) == INVALID, bad
    for op in (_lib.OP_ROPE_AXES, _lib.OP_KV_APPEND_AXES):
        d, out = _lib.OpDesc(op=op), ctypes.c_void_p()
        assert L.mgq_chain_create_ops(ctypes.byref(d), 1, ctypes.byref(out)) == INVALID


def test_python_refuses():
    from modgrad_amd.kvcache import RopeAxes
    from modgrad_amd.q4k import BackendError
    for bad in (dict(sections=[]), dict(sections=[1] * 5), dict(sections=[4, -1]), dict(sections=[0, 0]),
                dict(sections=[257]), dict(sections=[4], order="rows")):
        with pytest.raises(BackendError):
            RopeAxes(**bad)


@pytest.mark.parametrize("vtype,values,want", [(5, [16, 24, 24, 0], [16, 24, 24, 0]), (4, [11, 11, 10], [11, 11, 10])])
def test_sections_from_gguf(tmp_path, vtype, values, want):
    from modgrad_amd.gguf import GgufFile, write_gguf
    from modgrad_amd.kvcache import RopeAxes
    path = str(tmp_path / "m.gguf")
    write_gguf(path, [("general.architecture", 8, "llama"),
                      ("llama.rope.dimension_sections", 9, (vtype, values))], [])
    a = RopeAxes.from_gguf(GgufFile.open(path), "turns")
    assert a.sections == want and a.order == "turns" and not a.own


def test_sections_from_gguf_refuses(tmp_path):
    from modgrad_amd.gguf import GgufFile, write_gguf
    from modgrad_amd.kvcache import RopeAxes
    from modgrad_amd.q4k import BackendError
    for i, meta in enumerate(([], [("llama.rope.dimension_sections", 4, 16)],
                              [("llama.rope.dimension_sections", 9, (6, [1.5]))])):
        path = str(tmp_path / f"m{i}.gguf")
        write_gguf(path, [("general.architecture", 8, "llama")] + meta, [])
        with pytest.raises(BackendError):
            RopeAxes.from_gguf(GgufFile.open(path))


def test_reference_shares():
    assert ref.pairs([2, 1, 3], "blocks", False) == [(0, 0), (0, 1), (1, 2), (2, 3), (2, 4), (2, 5)]
    assert ref.pairs([2, 1, 3], "turns", False) == [(0, 0), (1, 1), (2, 2), (0, 3), (2, 4), (2, 5)]
    assert ref.pairs([2, 0, 3], "turns", True) == [(0, 0), (2, 0), (0, 1), (2, 1), (2, 2)]
    # one axis is the plain rotation
    from tests.kv_reference import rotate
    rng = np.random.default_rng(1)
    x, table = rng.standard_normal((3, 2, 10)), rng.standard_normal((5, 4, 2)).astype(np.float32)
    pos = np.array([[4, 0, 2]])
    for half in (False, True):
        want = np.stack([rotate(x[t], table[pos[0, t]], half) for t in range(3)])
        assert np.array_equal(ref.turn(x, pos, table, [4], "turns", False, half), want)
