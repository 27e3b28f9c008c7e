"""The rotary and key/value-cache entry points refuse bad arguments before any
device call; the reference implementation's own pins (no GPU)."""
import ctypes

import numpy as np
import pytest

from modgrad_amd import _lib
from tests import kv_reference as ref

INVALID = _lib.hipErrorInvalidValue
FAKE = 0x10000  # never dereferenced: every call below fails validation first


@pytest.fixture(scope="module")
def L():
    return _lib.load()


def cache(**kw):
    f = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, page_table=FAKE, seq_len=FAKE, cu_tokens=FAKE,
             page_stride=2 * 64 * 128, n_pages=10, page_tokens=64, n_kv_heads=2, head_dim=128, format=0, n_seqs=3,
             max_pages=4)
    f.update(kw)
    return _lib.KvCacheDesc(**f)


BAD_CACHE = [dict(k=None), dict(v=None), dict(k=FAKE + 8), dict(v=FAKE + 4), dict(k_scale=None), dict(v_scale=FAKE + 2),
             dict(page_stride=2 * 64 * 128 - 16), dict(page_stride=2 * 64 * 128 + 8), dict(page_stride=-16),
             dict(page_stride=(1 << 60) & ~15), dict(n_pages=0), dict(n_pages=-1), dict(page_tokens=0),
             dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=256), dict(n_kv_heads=0), dict(head_dim=80),
             dict(head_dim=512), dict(head_dim=0), dict(format=2), dict(format=-1)]
BAD_CALL = [dict(page_table=None), dict(page_table=FAKE + 1), dict(seq_len=None), dict(seq_len=FAKE + 2),
            dict(cu_tokens=FAKE + 2), dict(n_seqs=0), dict(n_seqs=-1), dict(max_pages=0), dict(max_pages=1 << 24)]


def append(L, c, rope=None, k=FAKE, v=FAKE, kvs=256, q=FAKE, qs=512, qo=FAKE, qos=512, hq=4, n=7, new=5):
    return L.launch_kv_append_ex(ctypes.byref(c), rope and ctypes.byref(rope), k, v, kvs, q, qs, qo, qos, hq, n, new,
                                 None)


def attend(L, c, q=FAKE, qs=512, hq=4, out=FAKE, os=512, kind=0, n=7, new=5, scale=0.1, cap=0.0, win=0, ws=FAKE,
           nbytes=1 << 40):
    return L.launch_kv_attention_ex(ctypes.byref(c), q, qs, hq, out, os, kind, n, new, scale, cap, win, ws, nbytes,
                                    None)


@pytest.mark.parametrize("bad", BAD_CACHE + BAD_CALL)
def test_bad_cache(L, bad):
    c = cache(**bad)
    assert append(L, c) == INVALID
    assert attend(L, c) == INVALID
    if bad in BAD_CACHE:
        assert L.launch_kv_dequant_ex(ctypes.byref(c), FAKE, 1, FAKE, FAKE, None) == INVALID
        assert L.mgq_kv_attention_workspace_bytes(ctypes.byref(c), 4, 1) == 0


def test_null_structs(L):
    assert L.launch_kv_append_ex(None, None, FAKE, FAKE, 256, None, 0, None, 0, 0, 7, 5, None) == INVALID
    assert L.launch_kv_attention_ex(None, FAKE, 512, 4, FAKE, 512, 0, 7, 5, 0.1, 0.0, 0, FAKE, 1 << 40, None) == INVALID
    assert L.launch_kv_dequant_ex(None, FAKE, 1, FAKE, FAKE, None) == INVALID
    assert L.mgq_kv_attention_workspace_bytes(None, 4, 1) == 0
    assert L.launch_rope_ex(FAKE, FAKE, FAKE, None, 1, 1, 64, 64, 64, None) == INVALID
    assert L.launch_rope_table_ex(FAKE, 4, 0, 64, None, None) == INVALID


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(k=FAKE + 2), dict(kvs=255), dict(qs=511),
                                 dict(qos=511), dict(qo=None), dict(q=None), dict(q=FAKE + 1), dict(hq=0), dict(hq=-4),
                                 dict(qs=600), dict(n=0), dict(n=-1), dict(new=0), dict(new=8)])
def test_append_refuses(L, bad):
    assert append(L, cache(), **bad) == INVALID


@pytest.mark.parametrize("bad", [dict(scale=3e38), dict(cap=3e38), dict(scale=1e20, cap=1e-20),
                                 dict(scale=0.1, cap=1e-45)])
def test_attention_refuses_factors_past_f32(L, bad):
    assert attend(L, cache(), **bad) == INVALID


def test_one_token_each_needs_a_row_each(L):
    c = cache(cu_tokens=None)
    assert append(L, c, n=7, new=1) == INVALID  # 3 sequences
    assert append(L, c, n=3, new=2) == INVALID
    assert attend(L, c, n=7, new=1) == INVALID


@pytest.mark.parametrize("bad", [dict(table=None), dict(table=FAKE + 2), dict(n_pos=0), dict(n_pos=255), dict(rot_dim=0),
                                 dict(rot_dim=63), dict(rot_dim=-2), dict(rot_dim=130), dict(rot_dim=514),
                                 dict(style=2), dict(style=-1)])
def test_append_refuses_rope(L, bad):
    # 4 pages of 64 tokens: positions to 255
    f = dict(table=FAKE, n_pos=256, rot_dim=128, style=0)
    f.update(bad)
    assert append(L, cache(), _lib.Rope(**f)) == INVALID
    if "n_pos" not in bad or bad["n_pos"] == 0:
        assert L.launch_rope_ex(FAKE, FAKE, FAKE, ctypes.byref(_lib.Rope(**f)), 1, 1, 128, 128, 128, None) == INVALID


@pytest.mark.parametrize("bad", [(None, FAKE, FAKE, 1, 2, 128, 256, 256), (FAKE, FAKE + 2, FAKE, 1, 2, 128, 256, 256),
                                 (FAKE, FAKE, None, 1, 2, 128, 256, 256), (FAKE, FAKE, FAKE, 0, 2, 128, 256, 256),
                                 (FAKE, FAKE, FAKE, 1, 0, 128, 256, 256), (FAKE, FAKE, FAKE, 1, 2, 127, 256, 256),
                                 (FAKE, FAKE, FAKE, 1, 2, 128, 255, 256), (FAKE, FAKE, FAKE, 1, 2, 128, 256, 255),
                                 (FAKE, FAKE, FAKE, 1, 2, 128, 256, 300),
                                 (FAKE, 2 * FAKE, FAKE, 2 ** 31 - 1, 2 ** 23, 128, 2 ** 30, 2 ** 30)])
def test_rope_refuses(L, bad):
    x, y, pos, n, heads, dim, xs, ys = bad
    r = _lib.Rope(FAKE, 8, 64, 0)
    assert L.launch_rope_ex(x, y, pos, ctypes.byref(r), n, heads, dim, xs, ys, None) == INVALID


@pytest.mark.parametrize("bad", [dict(base=0.0), dict(base=-1.0), dict(base=float("nan")), dict(base=float("inf")),
                                 dict(freq_scale=0.0), dict(freq_scale=float("nan")), dict(ext_factor=float("nan")),
                                 dict(ext_factor=1.0, orig_ctx=0.0), dict(ext_factor=1.0, base=1.0),
                                 dict(ext_factor=1.0, beta_fast=0.0), dict(ext_factor=1.0, beta_slow=-1.0),
                                 dict(attn_factor=float("inf")), dict(factors=FAKE + 2)])
def test_rope_table_refuses(L, bad):
    f = dict(base=1e4, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0, orig_ctx=4096.0,
             factors=None)
    f.update(bad)
    assert L.launch_rope_table_ex(FAKE, 8, 0, 64, ctypes.byref(_lib.RopeScaling(**f)), None) == INVALID


def test_rope_table_refuses_sizes(L):
    s = _lib.RopeScaling(1e4, 1.0, 0.0, 1.0, 32.0, 1.0, 0.0, None)
    for t, n, first, rot in ((None, 8, 0, 64), (FAKE + 1, 8, 0, 64), (FAKE, 0, 0, 64), (FAKE, 8, -1, 64),
                             (FAKE, 8, 2 ** 31 - 4, 64), (FAKE, 8, 0, 0), (FAKE, 8, 0, 63), (FAKE, 8, 0, 514)):
        assert L.launch_rope_table_ex(t, n, first, rot, ctypes.byref(s), None) == INVALID


@pytest.mark.parametrize("bad", [dict(q=None), dict(q=FAKE + 2), dict(qs=511), dict(out=None), dict(out=FAKE + 2),
                                 dict(out=FAKE + 1, kind=1), dict(os=511), dict(kind=2), dict(kind=-1), dict(hq=3),
                                 dict(hq=0), dict(n=0), dict(new=0), dict(new=8), dict(scale=float("nan")),
                                 dict(scale=float("inf")), dict(scale=-0.5), dict(cap=-1.0), dict(cap=float("nan")),
                                 dict(cap=float("inf")), dict(win=-1), dict(ws=None), dict(ws=FAKE + 8),
                                 dict(nbytes=0), dict(new=1 << 28, n=1 << 28)])
def test_attention_refuses(L, bad):
    assert attend(L, cache(), **bad) == INVALID


def test_attention_workspace(L):
    c = cache()
    need = L.mgq_kv_attention_workspace_bytes(ctypes.byref(c), 4, 5)
    assert need > 0
    assert attend(L, c, nbytes=need - 1) == INVALID
    for bad in (dict(n_seqs=0), dict(max_pages=0), dict(max_pages=1 << 24)):
        assert L.mgq_kv_attention_workspace_bytes(ctypes.byref(cache(**bad)), 4, 5) == 0
    assert L.mgq_kv_attention_workspace_bytes(ctypes.byref(c), 3, 5) == 0
    assert L.mgq_kv_attention_workspace_bytes(ctypes.byref(c), 4, 0) == 0


def test_dequant_refuses(L):
    c = ctypes.byref(cache())
    for pages, n, k, v in ((None, 1, FAKE, FAKE), (FAKE, 0, FAKE, FAKE), (FAKE, -1, FAKE, FAKE), (FAKE, 1, None, FAKE),
                           (FAKE, 1, FAKE, FAKE + 2), (FAKE + 1, 1, FAKE, FAKE), (FAKE, 1 << 30, FAKE, FAKE)):
        assert L.launch_kv_dequant_ex(c, pages, n, k, v, None) == INVALID


def test_chain_ops_refuse(L):
    out = ctypes.c_void_p()

    def create(op, args):
        d = _lib.OpDesc(op=op, w=None if args is None else ctypes.addressof(args))
        return L.mgq_chain_create_ops(ctypes.byref(d), 1, ctypes.byref(out))

    for op in (_lib.OP_ROPE, _lib.OP_KV_APPEND, _lib.OP_KV_ATTENTION):
        assert create(op, None) == INVALID
    rope = _lib.Rope(FAKE, 256, 64, 0)
    assert create(_lib.OP_ROPE, _lib.RopeArgs(FAKE, FAKE, FAKE, rope, 0, 2, 128, 256, 256)) == INVALID
    assert create(_lib.OP_KV_APPEND, _lib.KvAppendArgs(cache(head_dim=100), rope, FAKE, FAKE, FAKE, FAKE, 256, 512,
                                                       512, 4, 7, 5)) == INVALID
    assert create(_lib.OP_KV_ATTENTION, _lib.KvAttentionArgs(cache(), FAKE, FAKE, FAKE, 16, 512, 512, 4, 0, 7, 5, 0,
                                                             0.1, 0.0)) == INVALID
    assert out.value is None


# ------------------------------------------------ the reference's own pins --

def test_reference_codes():
    g = ref.grid("e4m3")
    fine = ~np.isnan(g)
    assert g[0x7E] == 448.0 and g[0x08] == 2.0 ** -6 and g[0x01] == 2.0 ** -9 and np.isnan(g[0x7F])
    assert np.array_equal(ref.code(g[fine], "e4m3")[1:128 - 1], np.arange(256)[fine][1:128 - 1])
    # ties go to the even code, past the largest it saturates
    assert list(ref.code([2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0, 464.0, 1e9, -np.inf, np.nan], "e4m3")) \
        == [0, 2, 0x58, 0x5A, 0x7E, 0x7E, 0xFE, 0]
    assert list(ref.code([0.5, 1.5, -2.5, 126.5, 200.0, np.nan], "i8").view(np.int8)) == [0, 2, -2, 126, 127, 0]


def test_reference_attention_is_a_mean_of_v():
    rng = np.random.default_rng(3)
    c = ref.Cache(np.zeros((3, 1, 16, 64), np.uint8), np.zeros((3, 1, 64, 16), np.uint8), np.zeros((3, 1), np.float32),
                  np.zeros((3, 1), np.float32), np.array([[2, 0]]), "i8")
    x = rng.integers(-127, 128, (20, 1, 64)).astype(np.float64)
    x[0], x[16] = 127, -127  # both pages get scale 1
    c.append(0, 0, x, x)
    k, v, there = c.read(0, 0, 20)
    assert there.all() and np.array_equal(k, x[:, 0]) and np.array_equal(v, x[:, 0])
    out, _ = c.attend(np.zeros((1, 2, 64)), [20], [1], 1.0)
    assert np.allclose(out[0, 1], x[:, 0].mean(0))
    out, _ = c.attend(np.zeros((1, 2, 64)), [20], [1], 1.0, window=5)
    assert np.allclose(out[0, 0], x[15:, 0].mean(0))


# ------------------------------------------------------- frequencies by GGUF --

def _gguf(tmp_path, meta):
    from modgrad_amd.gguf import GgufFile, write_gguf
    path = str(tmp_path / "m.gguf")
    write_gguf(path, [("general.architecture", 8, "llama")] + meta, [])
    return GgufFile.open(path)


@pytest.mark.parametrize("meta,want", [
    ([], dict(base=1e4, freq_scale=1.0, ext_factor=0.0, orig_ctx=0.0)),
    ([("llama.rope.freq_base", 6, 5e5)], dict(base=5e5, freq_scale=1.0, ext_factor=0.0)),
    ([("llama.rope.scaling.type", 8, "linear"), ("llama.rope.scaling.factor", 6, 8.0)],
     dict(base=1e4, freq_scale=0.125, ext_factor=0.0)),
    ([("llama.rope.scaling.type", 8, "yarn"), ("llama.rope.scaling.factor", 6, 4.0),
      ("llama.rope.scaling.original_context_length", 4, 32768), ("llama.rope.scaling.attn_factor", 6, 1.5)],
     dict(freq_scale=0.25, ext_factor=1.0, orig_ctx=32768.0, attn_factor=1.5, beta_fast=32.0, beta_slow=1.0)),
])
def test_rope_scaling_from_gguf(tmp_path, meta, want):
    from modgrad_amd.kvcache import RopeScaling
    c = RopeScaling.from_gguf(_gguf(tmp_path, meta)).c
    assert {k: getattr(c, k) for k in want} == want and not c.factors


def test_rope_scaling_from_gguf_refuses(tmp_path):
    from modgrad_amd.kvcache import RopeScaling
    from modgrad_amd.q4k import BackendError
    for meta in ([("llama.rope.scaling.type", 8, "longer")],
                 [("llama.rope.scaling.type", 8, "yarn"), ("llama.rope.scaling.factor", 6, 4.0)]):
        with pytest.raises(BackendError):
            RopeScaling.from_gguf(_gguf(tmp_path, meta))


@pytest.mark.parametrize("meta,scale", [
    ([("scaling.factor", 6, 4.0)], 0.25),                                  # a factor without a type is linear
    ([("scale_linear", 6, 2.0)], 0.5),                                     # the older key
    ([("scaling.factor", 6, 4.0), ("scale_linear", 6, 2.0)], 0.25),        # the newer one counts
    ([("scaling.type", 8, "linear"), ("scale_linear", 6, 8.0)], 0.125),
    ([("scaling.type", 8, "none"), ("scaling.factor", 6, 4.0)], 1.0),
    ([("scale_linear", 6, 1.0)], 1.0)])
def test_rope_scaling_from_gguf_without_a_type(tmp_path, meta, scale):
    from modgrad_amd.kvcache import RopeScaling
    c = RopeScaling.from_gguf(_gguf(tmp_path, [(f"llama.rope.{k}", t, v) for k, t, v in meta])).c
    assert (c.freq_scale, c.ext_factor, c.base) == (scale, 0.0, 1e4)


def test_rope_scaling_from_gguf_yarn_by_the_older_factor(tmp_path):
    from modgrad_amd.kvcache import RopeScaling
    c = RopeScaling.from_gguf(_gguf(tmp_path, [("llama.rope.scaling.type", 8, "yarn"), ("llama.rope.scale_linear", 6, 4.0),
                                               ("llama.rope.scaling.original_context_length", 4, 4096)])).c
    assert (c.freq_scale, c.ext_factor, c.orig_ctx) == (0.25, 1.0, 4096.0)


@pytest.mark.parametrize("meta", [
    [("scaling.type", 8, "linear"), ("scaling.factor", 4, 4)],             # whole numbers where the format has floats
    [("freq_base", 4, 500000)],
    [("scaling.type", 8, "yarn"), ("scaling.factor", 6, 4.0), ("scaling.original_context_length", 4, 4096),
     ("scaling.yarn_beta_fast", 6, 16.0)],                                 # a ramp of another shape
])
def test_rope_scaling_from_gguf_refuses_what_it_would_pass_over(tmp_path, meta):
    from modgrad_amd.kvcache import RopeScaling
    from modgrad_amd.q4k import BackendError
    with pytest.raises(BackendError):
        RopeScaling.from_gguf(_gguf(tmp_path, [(f"llama.rope.{k}", t, v) for k, t, v in meta]))


def test_rope_scaling_from_gguf_takes_the_finetuned_flag(tmp_path):
    from modgrad_amd.kvcache import RopeScaling
    c = RopeScaling.from_gguf(_gguf(tmp_path, [
        ("llama.rope.scaling.type", 8, "yarn"), ("llama.rope.scaling.factor", 6, 4.0),
        ("llama.rope.scaling.original_context_length", 4, 4096), ("llama.rope.scaling.finetuned", 7, True)])).c
    assert (c.freq_scale, c.ext_factor) == (0.25, 1.0)


def test_attention_takes_large_batches(L):
    """Long pieces for many sequences of large tables: the number of tiles is no
    limit where each work-group has rows of one sequence; rows and work-groups are."""
    size = lambda hq, new, **kw: L.mgq_kv_attention_workspace_bytes(  # noqa: E731
        ctypes.byref(cache(**kw)), hq, new)
    big = dict(n_seqs=256, max_pages=131072 // 64, n_kv_heads=8, page_stride=8 * 64 * 128)
    assert size(64, 2048, **big) > 0 and size(64, 8192, **big) > 0
    assert size(64, 1, **big) > 0 and size(64, 6, **big) > 0
    assert size(64, 1 << 26, **big) == 0              # 2^29 rows of a kv head
    assert size(64, 131072, **{**big, "n_seqs": 4096}) == 0  # 2^31 groups of 16 rows and heads


def test_attention_refuses_more_tiles_than_its_runs_can_count(L):
    """Few query rows: the tiles are cut into 512 equal runs, whose ends are counted
    in 32 bits."""
    tiles = (1 << 24) - 1  # of a sequence
    for seqs, fits in ((127, True), (128, False)):
        run = -(-seqs * tiles // 512)
        assert (512 * run < 2 ** 31) == fits and seqs * tiles < 2 ** 31
        c = cache(n_seqs=seqs, max_pages=tiles, n_kv_heads=1)
        assert (L.mgq_kv_attention_workspace_bytes(ctypes.byref(c), 1, 1) > 0) == fits


@pytest.mark.parametrize("factors", [dict(n=31), dict(n=33), dict(dtype="float64"), dict(step=2), dict()])
def test_rope_table_refuses_factors(factors):
    """Too few or too many, of another type, not next to one another, of the host."""
    import torch
    from modgrad_amd.kvcache import RopeScaling, kern
    from modgrad_amd.q4k import BackendError
    n, step = factors.get("n", 32), factors.get("step", 1)
    f = torch.ones(n * step, dtype=getattr(torch, factors.get("dtype", "float32")))[::step]
    with pytest.raises(BackendError, match="factors|tensors on"):  # before the library sees them
        kern.rope_table(FAKE, 0, 0, 64, RopeScaling(factors=f))
