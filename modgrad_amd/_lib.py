"""ctypes binding of libmodgrad_q4k.so (the C ABI in include/modgrad_q4k.h).

There is no fallback: if the library is missing or does not export every
declared symbol, loading raises. Build it with `python -m modgrad_amd.build`.
"""
from __future__ import annotations

import ctypes
import os
import re

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libmodgrad_q4k.so")
HEADER = os.path.join(os.path.dirname(HERE), "include", "modgrad_q4k.h")

hipSuccess = 0
hipErrorInvalidValue = 1
hipErrorNotSupported = 801

P = ctypes.c_void_p
I = ctypes.c_int
S = ctypes.c_size_t
F = ctypes.c_float
L = ctypes.c_int64
D = ctypes.c_double

SIGNATURES = {
    "launch_dequant_q4k": (I, [P, I, P]),
    "launch_matvec_q4k": (I, [P, P, P, I, I]),
    "launch_matvec_q4k_ex": (I, [P, P, P, I, I, I, P]),
    "launch_matvec_q4k_bias_ex": (I, [P, P, P, P, I, I, I, P]),
    "launch_quantize_q8_1": (I, [P, P, P, P, I]),
    "launch_matvec_q5k": (I, [P, P, P, I, I]),
    "launch_matvec_q6k": (I, [P, P, P, I, I]),
    "launch_matvec_q6k_dp4a": (I, [P, P, P, P, P, I, I]),
    "launch_matvec_q5k_ex": (I, [P, P, P, I, I, P]),
    "launch_matvec_q6k_ex": (I, [P, P, P, I, I, P]),
    "launch_matvec_q6k_dp4a_ex": (I, [P, P, P, P, P, I, I, P]),
    "launch_matvec_q4k_dp4a": (I, [P, P, P, P, P, I, I]),
    "launch_quantize_q8_1_ex": (I, [P, P, P, P, I, P]),
    "launch_matvec_q4k_dp4a_ex": (I, [P, P, P, P, P, I, I, P]),
    "launch_dequant_q4k_ex": (I, [P, I, P, P]),
    "mgq_batched_workspace_bytes": (S, [I, I]),
    "launch_matvec_q4k_batched": (I, [P, P, P, I, I, I, P, S, P]),
    "launch_matvec_q4k_batched_noalloc": (I, [P, P, P, I, I, I, P]),
    "launch_gemm_q4k_f16": (I, [P, P, P, I, I, I, P]),
    "mgq_gemm_tile": (I, [I, I, I, I, P, P, P]),
    "launch_quantize_matvec_q4k_dp4a_ex": (I, [P, P, P, I, I, P]),
    "launch_rms_norm": (I, [P, P, P, I, I, F]),
    "launch_rms_norm_ex": (I, [P, P, P, I, I, F, P]),
    "launch_geglu": (I, [P, P, P, I]),
    "launch_glu_ex": (I, [P, P, P, I, I, P]),
    "launch_residual_add": (I, [P, P, I]),
    "launch_residual_add_ex": (I, [P, P, I, P]),
    "launch_scale": (I, [P, F, I]),
    "launch_scale_ex": (I, [P, F, I, P]),
    "launch_matvec_q4k_rmsnorm_ex": (I, [P, P, P, F, P, I, I, P]),
    "launch_matvec_q6k_rmsnorm_ex": (I, [P, P, P, F, P, I, I, P]),
    "launch_matvec_q4k_glu_ex": (I, [P, P, P, P, F, I, P, I, I, P]),
    "launch_block_norm_ex": (I, [P, P, L, P, L, P, L, P, L, P, L, I, I, P]),
    "launch_rope_table_ex": (I, [P, I, I, I, P, P]),
    "launch_rope_ex": (I, [P, P, P, P, I, I, I, L, L, P]),
    "launch_rope_axes_ex": (I, [P, P, P, P, I, I, I, L, L, P]),
    "launch_kv_append_axes_ex": (I, [P, P, P, P, P, L, P, L, P, L, I, I, I, P]),
    "launch_kv_append_ex": (I, [P, P, P, P, L, P, L, P, L, I, I, I, P]),
    "launch_kv_dequant_ex": (I, [P, P, I, P, P, P]),
    "mgq_kv_attention_workspace_bytes": (S, [P, I, I]),
    "launch_kv_attention_sinks_ex": (I, [P, P, L, I, P, L, I, I, I, F, F, I, I, P, S, P]),
    "mgq_kv_attention_shared_workspace_bytes": (S, [P, I, I, I, I]),
    "mgq_kv_attention_shared_plan": (I, [P, I, I, I, I, I, P]),
    "launch_kv_attention_shared_ex": (I, [P, P, L, I, P, L, I, I, I, F, F, I, P, S, P]),
    "launch_kv_attention_ex": (I, [P, P, L, I, P, L, I, I, I, F, F, I, P, S, P]),
    "mgq_chain_create": (I, [P, I, P]),
    "mgq_chain_create_ex": (I, [P, I, I, P]),
    "mgq_chain_create_ops": (I, [P, I, P]),
    "mgq_chain_info": (I, [P, P, P]),
    "mgq_chain_launch": (I, [P, P]),
    "mgq_chain_destroy": (I, [P]),
    "mgq_prepare": (I, []),
    "mgq_version": (ctypes.c_char_p, []),
}

ACT_GELU_TANH = 0
ACT_SILU = 1
LAYOUT_ROWS = 0
LAYOUT_FLAT = 1
CHAIN_AUTO = 0
CHAIN_GRAPH = 1
CHAIN_PERSISTENT = 2
CHAIN_EAGER = 3
OP_MATVEC = 0
OP_MATVEC_NORM = 1
OP_MATVEC_GLU = 2
OP_RMS_NORM = 3
OP_GLU = 4
OP_RESIDUAL_ADD = 5
OP_QUANTIZE_Q8_1 = 6
OP_MATVEC_DP4A = 7
OP_QUANTIZE_MATVEC_DP4A = 8
OP_ROPE = 9
OP_KV_APPEND = 10
OP_KV_ATTENTION = 11
OP_BLOCK_NORM = 12
OP_ROPE_AXES = 13
OP_KV_APPEND_AXES = 14
OP_KV_ATTENTION_SINKS = 15
OP_KV_ATTENTION_SHARED = 16
SHARED_PLAIN = 0
SHARED_FEW = 1
SHARED_PARTS = 2
SHARED_RUNS = 3
AXES_BLOCKS = 0
AXES_TURNS = 1
ROPE_INTERLEAVED = 0
ROPE_HALF = 1
KV_I8 = 0
KV_E4M3 = 1
OUT_F32 = 0
OUT_F16 = 1
DTYPE_Q4_K = 12
DTYPE_Q5_K = 13
DTYPE_Q6_K = 14


class GemvDesc(ctypes.Structure):
    """mgq_gemv_desc."""
    _fields_ = [("w_q4", P), ("x", P), ("y", P), ("out_dim", I), ("blocks_per_row", I)]


class OpDesc(ctypes.Structure):
    """mgq_op_desc (one kernel of an op chain)."""
    _fields_ = [("op", I), ("dtype", I), ("layout", I), ("act", I), ("w", P), ("w2", P),
                ("x", P), ("x2", P), ("norm_w", P), ("y", P), ("out_dim", I), ("in_dim", I),
                ("rows", I), ("eps", F), ("xq", P), ("xd", P), ("xsum", P)]


class RopeScaling(ctypes.Structure):
    """mgq_rope_scaling."""
    _fields_ = [("base", D), ("freq_scale", D), ("ext_factor", D), ("attn_factor", D),
                ("beta_fast", D), ("beta_slow", D), ("orig_ctx", D), ("factors", P)]


class Rope(ctypes.Structure):
    """mgq_rope."""
    _fields_ = [("table", P), ("n_pos", I), ("rot_dim", I), ("style", I)]


class KvCacheDesc(ctypes.Structure):
    """mgq_kv_cache."""
    _fields_ = [("k", P), ("v", P), ("k_scale", P), ("v_scale", P), ("page_table", P),
                ("seq_len", P), ("cu_tokens", P), ("page_stride", L), ("n_pages", I),
                ("page_tokens", I), ("n_kv_heads", I), ("head_dim", I), ("format", I),
                ("n_seqs", I), ("max_pages", I)]


class RopeArgs(ctypes.Structure):
    """mgq_rope_args (OP_ROPE)."""
    _fields_ = [("x", P), ("y", P), ("pos", P), ("rope", Rope), ("n_tokens", I), ("n_heads", I),
                ("head_dim", I), ("x_stride", L), ("y_stride", L)]


class KvAppendArgs(ctypes.Structure):
    """mgq_kv_append_args (OP_KV_APPEND)."""
    _fields_ = [("cache", KvCacheDesc), ("rope", Rope), ("k", P), ("v", P), ("q", P),
                ("q_out", P), ("kv_stride", L), ("q_stride", L), ("q_out_stride", L),
                ("n_q_heads", I), ("n_tokens", I), ("max_new", I)]


class KvAttentionArgs(ctypes.Structure):
    """mgq_kv_attention_args (OP_KV_ATTENTION)."""
    _fields_ = [("cache", KvCacheDesc), ("q", P), ("out", P), ("workspace", P),
                ("workspace_bytes", S), ("q_stride", L), ("out_stride", L), ("n_q_heads", I),
                ("out_type", I), ("n_tokens", I), ("max_new", I), ("window", I), ("scale", F),
                ("softcap", F)]


class RopeAxes(ctypes.Structure):
    """mgq_rope_axes."""
    _fields_ = [("pos", P), ("pos_stride", L), ("n_axes", I), ("sections", I * 4), ("order", I), ("own", I)]


class RopeAxesArgs(ctypes.Structure):
    """mgq_rope_axes_args (OP_ROPE_AXES)."""
    _fields_ = [("x", P), ("y", P), ("axes", RopeAxes), ("rope", Rope), ("n_tokens", I), ("n_heads", I),
                ("head_dim", I), ("x_stride", L), ("y_stride", L)]


class KvAppendAxesArgs(ctypes.Structure):
    """mgq_kv_append_axes_args (OP_KV_APPEND_AXES)."""
    _fields_ = [("append", KvAppendArgs), ("axes", RopeAxes)]


class KvAttentionSinksArgs(ctypes.Structure):
    """mgq_kv_attention_sinks_args (OP_KV_ATTENTION_SINKS)."""
    _fields_ = [("attention", KvAttentionArgs), ("sinks", I)]


class KvAttentionSharedArgs(ctypes.Structure):
    """mgq_kv_attention_shared_args (OP_KV_ATTENTION_SHARED)."""
    _fields_ = [("attention", KvAttentionArgs), ("shared_tokens", I)]


class KvSharedPlan(ctypes.Structure):
    """mgq_kv_shared_plan."""
    _fields_ = [("way", I), ("tiles", I), ("blocks", I), ("run", I), ("own_groups", L), ("join_groups", L)]


class BlockNorm(ctypes.Structure):
    """mgq_block_norm."""
    _fields_ = [("post_w", P), ("norm_w", P), ("h_scale", F), ("x_scale", F), ("eps", F), ("hidden", I)]


class BlockNormArgs(ctypes.Structure):
    """mgq_block_norm_args (OP_BLOCK_NORM)."""
    _fields_ = [("norm", BlockNorm), ("h", P), ("x", P), ("gate", P), ("h_out", P), ("y", P), ("h_stride", L),
                ("x_stride", L), ("gate_stride", L), ("h_out_stride", L), ("y_stride", L), ("y_type", I), ("rows", I)]


class HipError(RuntimeError):
    def __init__(self, fn: str, code: int):
        super().__init__(f"{fn} returned hipError {code}")
        self.code = code


_lib = None


def declared_symbols() -> list[str]:
    """Function names declared in include/modgrad_q4k.h."""
    text = open(HEADER).read()
    return re.findall(r"^\s*(?:hipError_t|const char \*)\s*\*?\s*(\w+)\s*\(", text, re.M)


def load() -> ctypes.CDLL:
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(
            f"{LIB_PATH} is missing: build it with `python -m modgrad_amd.build` "
            "(there is no CPU fallback)")
    lib = ctypes.CDLL(LIB_PATH)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)  # AttributeError if the symbol is not exported
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


def check(fn: str, code: int) -> None:
    if code != hipSuccess:
        raise HipError(fn, code)
