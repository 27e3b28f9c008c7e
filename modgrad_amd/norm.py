"""The norms around a block of a decoder layer with what lies between them (the
reference's launch_rms_norm, launch_scale, launch_residual_add and the next
block's launch_rms_norm, crates/modgrad-gemma/src/rocm_gemma.rs:429-489), in one
launch over the C ABI.

    norm = BlockNorm(3584, 1e-6, post_w=w1, norm_w=w2, x_scale=0.22)
    norm.apply(h, x, rows, y=y)             # h += 0.22 norm(x) w1; y = norm(h) w2
    Chain.from_ops([..., norm.op(h, x, 1, y=y), ...])

Addresses are device pointers as in modgrad_amd.q4k.kern, the weights tensors that
the object keeps. `stream` is a torch stream, None the null stream.
"""
from __future__ import annotations

import ctypes

from . import _lib
from .q4k import BackendError, _torch, kern
from .kvcache import _elsewhere, _on_device, _on_gpu, _op


class BlockNorm:
    """Weights and factors of (mgq_block_norm)
      z = x r(x) post_w, h' = h_scale h + x_scale gate z, y = h' r(h') norm_w,
    r(a) = 1 / sqrt(mean(a^2) + eps). post_w, norm_w: f32 tensors [hidden], or None
    for no norm there; gate: an f32 tensor [hidden] of one gate for each channel."""

    def __init__(self, hidden: int, eps: float, post_w=None, norm_w=None, gate=None, h_scale: float = 1.0,
                 x_scale: float = 1.0):
        self.device = None
        for t, name in ((post_w, "post_w"), (norm_w, "norm_w"), (gate, "gate")):
            if t is None:
                continue
            if tuple(t.shape) != (hidden,) or t.dtype != _torch().float32 or not t.is_contiguous():
                raise BackendError("Runtime", f"block norm: {name}: {hidden} contiguous f32 expected")
            if self.device is not None and t.device != self.device:
                raise BackendError("Runtime", "block norm: tensors on different devices")
            self.device = t.device
        self.hidden, self.post_w, self.norm_w, self.gate = hidden, post_w, norm_w, gate
        self._look = self.device is not None and _elsewhere(self.device)
        self._gate = 0 if gate is None else gate.data_ptr()
        self.desc = _lib.BlockNorm(None if post_w is None else post_w.data_ptr(),
                                   None if norm_w is None else norm_w.data_ptr(), h_scale, x_scale, eps, hidden)
        self._ref = ctypes.byref(self.desc)

    def _rows(self, h, x, h_out, y, gate, gate_stride, strides):
        d = self.hidden
        h_stride, x_stride, h_out_stride, y_stride = (d if s is None else s for s in strides)
        if h_out is None:
            h_out, h_out_stride = h, h_stride
        if not gate:
            gate, gate_stride = (self._gate if x else 0), 0
        elif self._gate:
            raise BackendError("Runtime", "block norm: a gate for each channel and one for each row")
        return (h, h_stride, x, x_stride, gate, d if gate_stride is None else gate_stride, h_out, h_out_stride, y,
                y_stride)

    def apply(self, h: int, x: int, rows: int, h_out: int | None = None, y: int = 0, y_f16: bool = False,
              gate: int = 0, gate_stride: int | None = None, h_stride: int | None = None, x_stride: int | None = None,
              h_out_stride: int | None = None, y_stride: int | None = None, stream=None) -> None:
        """h' to h_out (None: to h itself, 0: nowhere) and its norm to y (0: nowhere)
        for `rows` rows; x 0: no block's result, only h_scale h and its norm. gate: a
        row of gates for each row. Strides in values, hidden by default."""
        if self._look:
            _on_device(self.device)
        kern.block_norm(self._ref, *self._rows(h, x, h_out, y, gate, gate_stride,
                                               (h_stride, x_stride, h_out_stride, y_stride)),
                        _lib.OUT_F16 if y_f16 else _lib.OUT_F32, rows, stream)

    def op(self, h: int, x: int, rows: int, h_out: int | None = None, y: int = 0, y_f16: bool = False,
           gate: int = 0, gate_stride: int | None = None, h_stride: int | None = None, x_stride: int | None = None,
           h_out_stride: int | None = None, y_stride: int | None = None) -> "_lib.OpDesc":
        """apply as a descriptor of an op chain (q4k.Chain.from_ops)."""
        _on_gpu(self.device)
        h, hs, x, xs, gate, gs, ho, hos, y, ys = self._rows(h, x, h_out, y, gate, gate_stride,
                                                            (h_stride, x_stride, h_out_stride, y_stride))
        return _op(_lib.OP_BLOCK_NORM, _lib.BlockNormArgs(
            self.desc, h, x or None, gate or None, ho or None, y or None, hs, xs, gs, hos, ys,
            _lib.OUT_F16 if y_f16 else _lib.OUT_F32, rows))
