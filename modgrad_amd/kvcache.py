"""Rotary positions and a paged 8-bit key/value cache: what a decoder needs
between the matvecs of a layer (the reference's launch_rope_neox, copy and
sdpa_decode sequence, crates/modgrad-gemma/src/rocm_gemma.rs:448-469), over the
C ABI.

  RopeScaling   frequencies of a rotary table, from numbers or GGUF metadata
  RopeTable     a table of (cos, sin) on the device, and its application
  RopeAxes      positions of several axes (time, height, width) on such a table
  KvCache       pages of 8-bit keys and values, their scales and page tables;
                append, attend, dequant, and the same as op-chain descriptors

    rope = RopeTable.from_gguf(g, n_pos=8192, half=True)
    cache = KvCache.new(n_pages=512, page_tokens=64, n_kv_heads=4, head_dim=128,
                        n_seqs=8, max_pages=128)
    cache.set_lengths([n0 + 1, n1 + 1, ...])           # the new tokens included
    cache.append(k, v, kv_stride, 8, 1, rope=rope, q=q, q_stride=qs, n_q_heads=28)
    cache.attend(q, qs, 28, out, 28 * 128, 8, 1)
    cache.share(1, 0, 4096)                            # slot 1 behind slot 0's first 4096 tokens

Addresses are device pointers as in modgrad_amd.q4k.kern; torch only allocates.
`stream` is a torch stream, None the null stream; page tables and lengths are
written on it too, so a step's set_lengths is given the stream of its launches.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

from . import _lib
from .gguf import GgmlType
from .q4k import BackendError, _torch, kern


def _stream(stream):
    """A context in which torch allocates and writes on the launches' stream:
    memory freed there is used again behind the launches, not beside them."""
    cuda = _torch().cuda
    return cuda.stream(cuda.default_stream() if stream is None else stream)


def _elsewhere(device) -> bool:
    """Whether a call has to look (_on_device) if its tensors are on the current
    device: there is nothing else with one GPU, and looking costs a microsecond."""
    return device.type != "cuda" or _torch().cuda.device_count() > 1


def _on_device(device) -> None:
    """Launches go to the current device: the tensors have to be there."""
    if device.type != "cuda":
        raise BackendError("Runtime", f"tensors on {device}")
    cuda = _torch().cuda
    if device.index != cuda.current_device():
        raise BackendError("Runtime", f"tensors on {device}, the current device is "
                                      f"cuda:{cuda.current_device()}")


def _on_gpu(device) -> None:
    """A recorded launch goes to the device that is current then; host memory is never there."""
    if device is not None and device.type != "cuda":
        raise BackendError("Runtime", f"tensors on {device}")


FORMATS = {"i8": _lib.KV_I8, "e4m3": _lib.KV_E4M3}


class RopeScaling:
    """Frequencies of a rotary table (mgq_rope_scaling). `factors`: a device
    f32 tensor of rot_dim/2 divisors (a GGUF file's rope_freqs.weight)."""

    def __init__(self, base: float = 10000.0, freq_scale: float = 1.0, ext_factor: float = 0.0,
                 attn_factor: float = 1.0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 orig_ctx: float = 0.0, factors=None):
        self.factors = factors
        self.c = _lib.RopeScaling(base, freq_scale, ext_factor, attn_factor, beta_fast, beta_slow,
                                  orig_ctx, None if factors is None else factors.data_ptr())
        self.ref = ctypes.byref(self.c)

    def check(self, rot_dim: int) -> None:
        """The divisors are read as rot_dim/2 floats of the current device."""
        f = self.factors
        if f is None:
            return
        if f.numel() != rot_dim // 2 or str(f.dtype) != "torch.float32" or not f.is_contiguous():
            raise BackendError("Runtime", f"rope factors: {rot_dim // 2} contiguous f32 expected")
        _on_device(f.device)

    @classmethod
    def from_gguf(cls, g, factors=None) -> "RopeScaling":
        """From an opened GgufFile's <arch>.rope.* keys: freq_base,
        scaling.type ("none", "linear", "yarn"; a factor without a type is
        linear), scaling.factor (older files: rope.scale_linear),
        scaling.attn_factor, scaling.original_context_length. Keys that would
        change the angles in another way (further rope.scaling.* ones of a
        "yarn" file, numbers of another type) are refused, not passed over."""
        arch = g.architecture()

        def number(key):
            m = g.meta(f"{arch}.rope.{key}")
            x = 0.0 if m is None else m.as_f32()
            if x is None:
                raise BackendError("Unsupported", f"{arch}.rope.{key} is not a float")
            return x

        base = number("freq_base") or 10000.0
        m = g.meta(f"{arch}.rope.scaling.type")
        kind = m.as_str() if m is not None else "linear"
        factor = number("scaling.factor") or number("scale_linear") or 1.0
        attn = number("scaling.attn_factor") or 1.0
        if kind not in ("none", "linear", "yarn"):
            raise BackendError("Unsupported", f"rope scaling type {kind!r}")
        if kind == "none" or factor == 1.0:
            return cls(base, attn_factor=attn, factors=factors)
        if kind == "linear":
            return cls(base, freq_scale=1.0 / factor, attn_factor=attn, factors=factors)
        known = ("type", "factor", "attn_factor", "original_context_length", "finetuned")
        for key in g.metadata:
            if key.startswith(f"{arch}.rope.scaling.") and key.split(".rope.scaling.")[1] not in known:
                raise BackendError("Unsupported", key)
        orig = g.meta_u32(f"{arch}.rope.scaling.original_context_length")
        if not orig:
            raise BackendError("Runtime", f"missing {arch}.rope.scaling.original_context_length")
        return cls(base, freq_scale=1.0 / factor, ext_factor=1.0, attn_factor=attn,
                   orig_ctx=float(orig), factors=factors)


class RopeAxes:
    """How the pairs of a head are shared out among several axes of positions
    (mgq_rope_axes): sections[a] pairs for axis a, in "blocks" one after another, or in
    "turns" of one pair for each axis that has some left. own: every axis has the
    table's columns from the first on (a picture's rows and columns), instead of the
    pair's. With one, RopeTable.apply and KvCache.append take positions
    [n_axes][pos_stride]."""

    ORDERS = {"blocks": _lib.AXES_BLOCKS, "turns": _lib.AXES_TURNS}

    def __init__(self, sections, order: str = "blocks", own: bool = False):
        self.sections = [int(n) for n in sections]
        if order not in self.ORDERS or not 1 <= len(self.sections) <= 4 or min(self.sections) < 0 \
                or not 1 <= sum(self.sections) <= 256:
            raise BackendError("Runtime", f"rope axes: sections {self.sections}, {order!r}")
        self.order, self.own = order, bool(own)

    @classmethod
    def from_gguf(cls, g, order: str = "blocks") -> "RopeAxes":
        """Of a GGUF model's <arch>.rope.dimension_sections. Whether its axes lie in
        blocks or take turns is the architecture's, and no key of the file says it."""
        key = f"{g.architecture()}.rope.dimension_sections"
        m = g.meta(key)
        values = m.value if m is not None and isinstance(m.value, list) else []
        sections = [v.value for v in values]
        if not sections or not all(isinstance(n, int) and not isinstance(n, bool) for n in sections):
            raise BackendError("Unsupported", f"{key}: whole numbers expected")
        return cls(sections, order)

    def at(self, pos: int, pos_stride: int) -> "_lib.RopeAxes":
        """With the positions of a call: device ints, axis a of row t at
        pos[a * pos_stride + t]."""
        n = len(self.sections)
        return _lib.RopeAxes(pos or None, pos_stride, n, (_lib.I * 4)(*self.sections), self.ORDERS[self.order], self.own)


class RopeTable:
    """(cos, sin) of positions 0 .. n_pos-1 on the device, f32
    [n_pos][rot_dim/2][2]. half: pairs (i, i + rot_dim/2); else (2i, 2i+1)."""

    def __init__(self, n_pos: int, rot_dim: int, half: bool, scaling: RopeScaling | None = None,
                 stream=None):
        if n_pos <= 0 or rot_dim <= 0 or rot_dim % 2:
            raise BackendError("Runtime", f"rope table of {n_pos} positions, {rot_dim} dims")
        torch = _torch()
        scaling = scaling or RopeScaling()
        with _stream(stream):
            t = torch.empty(n_pos, rot_dim // 2, 2, dtype=torch.float32, device="cuda")
        kern.rope_table(t.data_ptr(), n_pos, 0, rot_dim, scaling, stream)
        self._hold(t, half)

    @classmethod
    def wrap(cls, table, half: bool) -> "RopeTable":
        """Of an existing device tensor [n_pos, rot_dim/2, 2], f32."""
        if table.dim() != 3 or table.shape[2] != 2 or not table.is_contiguous() \
                or table.dtype != _torch().float32:
            raise BackendError("Runtime", "rope table: contiguous f32 [n_pos, rot_dim/2, 2] expected")
        r = cls.__new__(cls)
        r._hold(table, half)
        return r

    @classmethod
    def from_gguf(cls, g, n_pos: int, half: bool, stream=None) -> "RopeTable":
        """For a GGUF model: its rotated dims (<arch>.rope.dimension_count),
        scaling and, where the file holds them, the divisors of its
        rope_freqs.weight. Which dims pair up is the architecture's, and no key
        of the file says it."""
        torch = _torch()
        arch = g.architecture()
        rot = g.meta_u32(f"{arch}.rope.dimension_count") or g.meta_u32(f"{arch}.attention.key_length")
        if not rot:
            emb, heads = g.meta_u32(f"{arch}.embedding_length"), g.meta_u32(f"{arch}.attention.head_count")
            if not emb or not heads:
                raise BackendError("Runtime", f"missing {arch}.rope.dimension_count")
            rot = emb // heads
        factors = None
        if "rope_freqs.weight" in g.tensors:
            if g.tensors["rope_freqs.weight"].dtype != GgmlType.F32:
                raise BackendError("Unsupported", "rope_freqs.weight is not F32")
            raw = np.frombuffer(g.tensor_bytes("rope_freqs.weight"), np.float32).copy()
            with _stream(stream):
                factors = torch.from_numpy(raw).cuda()
        return cls(n_pos, rot, half, RopeScaling.from_gguf(g, factors), stream)

    def _hold(self, table, half: bool) -> None:
        self.table, self.half, self.device = table, bool(half), table.device
        self._look = _elsewhere(self.device)
        self.n_pos, self.rot_dim = table.shape[0], 2 * table.shape[1]
        self.desc = _lib.Rope(table.data_ptr(), self.n_pos, self.rot_dim,
                              _lib.ROPE_HALF if half else _lib.ROPE_INTERLEAVED)
        self.ref = ctypes.byref(self.desc)

    def apply(self, x: int, y: int, pos: int, n_tokens: int, n_heads: int, head_dim: int,
              x_stride: int | None = None, y_stride: int | None = None, stream=None,
              axes: RopeAxes | None = None, pos_stride: int | None = None) -> None:
        """y = x, [n_tokens][n_heads][head_dim] f32 turned to positions pos; with
        axes, pos is [n_axes][pos_stride] (n_tokens by default)."""
        if self._look:
            _on_device(self.device)
        row = n_heads * head_dim
        if axes is not None:
            at = axes.at(pos, n_tokens if pos_stride is None else pos_stride)
            kern.rope_axes(x, y, ctypes.byref(at), self.ref, n_tokens, n_heads, head_dim,
                           row if x_stride is None else x_stride, row if y_stride is None else y_stride, stream)
            return
        kern.rope(x, y, pos, self.ref, n_tokens, n_heads, head_dim,
                  row if x_stride is None else x_stride, row if y_stride is None else y_stride,
                  stream)

    def op(self, x: int, y: int, pos: int, n_tokens: int, n_heads: int, head_dim: int,
           x_stride: int | None = None, y_stride: int | None = None, axes: RopeAxes | None = None,
           pos_stride: int | None = None) -> "_lib.OpDesc":
        """apply as a descriptor of an op chain (q4k.Chain.from_ops)."""
        _on_gpu(self.device)
        row = n_heads * head_dim
        if axes is not None:
            return _op(_lib.OP_ROPE_AXES, _lib.RopeAxesArgs(
                x, y, axes.at(pos, n_tokens if pos_stride is None else pos_stride), self.desc, n_tokens, n_heads,
                head_dim, row if x_stride is None else x_stride, row if y_stride is None else y_stride))
        return _op(_lib.OP_ROPE, _lib.RopeArgs(
            x, y, pos, self.desc, n_tokens, n_heads, head_dim,
            row if x_stride is None else x_stride, row if y_stride is None else y_stride))


def _op(kind: int, args) -> "_lib.OpDesc":
    d = _lib.OpDesc(op=kind, w=ctypes.addressof(args))
    d._args = args  # read when the chain is created
    return d


def _workspace(workspace, device) -> None:
    """A call writes all of its workspace: it has to be memory of the cache's device."""
    if workspace.device != device or not workspace.is_contiguous():
        raise BackendError("Runtime", f"workspace: contiguous memory on {device} expected")


def _without_window(window: int, sinks: int) -> None:
    if window or sinks:
        raise BackendError("Unsupported", "attention over a shared prefix with a window")


class KvCache:
    """One layer's paged 8-bit cache and the page tables of n_seqs slots
    (mgq_kv_cache)."""

    def __init__(self, k, v, k_scale, v_scale, page_table, seq_len, cu_tokens, fmt: str):
        torch = _torch()
        if fmt not in FORMATS:
            raise BackendError("Unsupported", f"cache format {fmt!r}")
        if k.dim() != 4 or v.dim() != 4 or k.dtype != torch.uint8 or v.dtype != torch.uint8:
            raise BackendError("Runtime", "cache: uint8 [pages, heads, tokens, dim] k and "
                                          "[pages, heads, dim, tokens] v expected")
        pages, heads, tokens, dim = k.shape
        if tuple(v.shape) != (pages, heads, dim, tokens) or k.stride()[1:] != (tokens * dim, dim, 1) \
                or v.stride()[1:] != (tokens * dim, tokens, 1) or k.stride(0) != v.stride(0):
            raise BackendError("Runtime", "cache: k and v differ in pages, or a page's heads are "
                                          "not contiguous")
        for t, name, shape, dt in ((k_scale, "k_scale", (pages, heads), torch.float32),
                                   (v_scale, "v_scale", (pages, heads), torch.float32),
                                   (seq_len, "seq_len", tuple(page_table.shape[:1]), torch.int32)):
            if tuple(t.shape) != shape or t.dtype != dt or not t.is_contiguous():
                raise BackendError("Runtime", f"cache: {name}: contiguous {dt} {shape} expected")
        if page_table.dim() != 2 or page_table.dtype != torch.int32 or not page_table.is_contiguous():
            raise BackendError("Runtime", "cache: page_table: contiguous int32 [n_seqs, max_pages]")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.page_table, self.seq_len, self.cu_tokens = page_table, seq_len, None
        self.format, self.device = fmt, k.device
        self.n_pages, self.n_kv_heads, self.page_tokens, self.head_dim = pages, heads, tokens, dim
        self.n_seqs, self.max_pages = page_table.shape
        self.desc = _lib.KvCacheDesc(
            k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
            page_table.data_ptr(), seq_len.data_ptr(), None, k.stride(0), pages, tokens, heads, dim,
            FORMATS[fmt], self.n_seqs, self.max_pages)
        self.use_cu_tokens(cu_tokens)
        for t in (v, k_scale, v_scale, page_table, seq_len):
            if t.device != self.device:
                raise BackendError("Runtime", "cache: tensors on different devices")
        self._look = _elsewhere(self.device)
        self._own_cu = None
        self._ref = ctypes.byref(self.desc)
        self._free = None
        self._held = [[] for _ in range(self.n_seqs)]  # pages of each slot, None where given back
        self._users = [0] * self.n_pages               # slots that have a page

    @classmethod
    def wrap(cls, k, v, k_scale, v_scale, page_table, seq_len, cu_tokens=None,
             fmt: str = "i8") -> "KvCache":
        """Of existing tensors: k uint8 [pages, heads, tokens, dim], v uint8
        [pages, heads, dim, tokens], scales f32 [pages, heads], page_table
        int32 [n_seqs, max_pages], seq_len int32 [n_seqs], cu_tokens int32
        [n_seqs + 1] or None (one new token per sequence)."""
        return cls(k, v, k_scale, v_scale, page_table, seq_len, cu_tokens, fmt)

    @classmethod
    def new(cls, n_pages: int, page_tokens: int, n_kv_heads: int, head_dim: int, n_seqs: int,
            max_pages: int, fmt: str = "i8", stream=None) -> "KvCache":
        """An empty cache whose pages reserve(), share(), give_back() and release() hand
        out and take back. Its table is theirs to write: pages entered by hand would be
        given out or taken back beside them (wrap() is for tables of one's own)."""
        torch = _torch()
        with _stream(stream):
            try:
                k = torch.zeros(n_pages, n_kv_heads, page_tokens, head_dim, dtype=torch.uint8, device="cuda")
                v = torch.zeros(n_pages, n_kv_heads, head_dim, page_tokens, dtype=torch.uint8, device="cuda")
            except torch.cuda.OutOfMemoryError as e:
                raise BackendError("OutOfMemory", f"cache of {n_pages} pages") from e
            c = cls(k, v, torch.zeros(n_pages, n_kv_heads, device="cuda"),
                    torch.zeros(n_pages, n_kv_heads, device="cuda"),
                    torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device="cuda"),
                    torch.zeros(n_seqs, dtype=torch.int32, device="cuda"), None, fmt)
        c._free = list(range(n_pages - 1, -1, -1))
        return c

    # -- pages and lengths ---------------------------------------------------
    def _short(self, seq: int, n_tokens: int) -> int:
        """Pages that slot `seq` lacks for n_tokens positions."""
        need = -(-n_tokens // self.page_tokens)
        if need > self.max_pages:
            raise BackendError("Runtime", f"reserve: {n_tokens} tokens need {need} pages, a "
                                          f"sequence has {self.max_pages}")
        return max(0, need - len(self._held[seq]))

    def _afford(self, short: int) -> None:
        if short > len(self._free):
            raise BackendError("OutOfMemory", f"reserve: {short} pages, {len(self._free)} free")

    def _own_pages(self, what: str, *seqs) -> None:
        if self._free is None:
            raise BackendError("Unsupported", f"{what}: the cache wraps tables of the caller's")
        for seq in seqs:
            if not 0 <= seq < self.n_seqs:
                raise BackendError("Runtime", f"{what}: sequence {seq}")

    def _write(self, seq: int, first: int, pages, stream) -> None:
        with _stream(stream):
            self.page_table[seq, first: first + len(pages)] = _torch().tensor(pages, dtype=_torch().int32)

    def _leave(self, pages) -> None:
        """Pages that one slot less has; those that none has are free."""
        for p in pages:
            self._users[p] -= 1
        self._free += [p for p in pages if self._users[p] == 0]

    def reserve(self, seq: int, n_tokens: int, stream=None) -> None:
        """Pages for the first n_tokens positions of slot `seq`."""
        self._own_pages("reserve", seq)
        if n_tokens < 0:
            raise BackendError("Runtime", f"reserve: {n_tokens} tokens of sequence {seq}")
        short, held = self._short(seq, n_tokens), self._held[seq]
        self._afford(short)
        if short:
            new = [self._free.pop() for _ in range(short)]
            for p in new:
                self._users[p] = 1
            self._write(seq, len(held), new, stream)
            held += new

    def share(self, seq: int, other: int, n_tokens: int, stream=None) -> None:
        """Slot `seq`, which has no pages yet, begins with those of the first n_tokens
        positions (whole pages) of slot `other`: what attend(shared=n_tokens) reads once for
        both. A page is free again when no slot has it; new tokens go behind it."""
        self._own_pages("share", seq, other)
        n = n_tokens // self.page_tokens
        pages = self._held[other][:max(n, 0)]
        if seq == other or self._held[seq] or n_tokens < 0 or n_tokens % self.page_tokens or len(pages) < n \
                or None in pages:
            raise BackendError("Runtime", f"share: {n_tokens} tokens of sequence {other} with {seq}: whole pages that "
                                          "the one has and the other has none of")
        for p in pages:
            self._users[p] += 1
        self._held[seq] = pages
        if pages:
            self._write(seq, 0, pages, stream)

    def give_back(self, seq: int, first: int, end: int, stream=None) -> None:
        """Pages of slot `seq` that lie in positions first .. end-1, which no call looks at
        any more (behind the first tokens and ahead of a window)."""
        self._own_pages("give_back", seq)
        if not 0 <= first <= end:
            raise BackendError("Runtime", f"give_back: positions {first} to {end}")
        held = self._held[seq]
        slots = range(-(-first // self.page_tokens), min(end // self.page_tokens, len(held)))
        self._leave([held[i] for i in slots if held[i] is not None])
        for i in slots:
            held[i] = None
        if slots:
            self._write(seq, slots[0], [-1] * len(slots), stream)

    def release(self, seq: int, stream=None) -> None:
        """Gives the pages of slot `seq` back, those that other slots have to them, and
        leaves it idle."""
        self._own_pages("release", seq)
        self._leave([p for p in self._held[seq] if p is not None])
        self._held[seq] = []
        with _stream(stream):
            self.page_table[seq] = -1
            self.seq_len[seq] = 0

    def set_lengths(self, lengths, new=None, stream=None) -> None:
        """Tokens of every slot with the next call's new ones, and how many of
        them are new (None: one each); pages are reserved for them. New tokens do
        not lie in pages that are shared or were given back. The tensors
        stay in place, so that recorded calls replay on the new values: one that
        was recorded with counts takes any that fit its n_tokens and max_new, one
        that was recorded with one each stays at that."""
        torch = _torch()
        lengths = [int(n) for n in lengths]
        counts = None if new is None else [int(n) for n in new]
        if len(lengths) != self.n_seqs or (counts is not None and len(counts) != self.n_seqs):
            raise BackendError("Runtime", f"set_lengths: {self.n_seqs} sequences")
        for n, m in zip(lengths, counts or [0] * self.n_seqs):
            if not 0 <= m <= n < 2 ** 30:
                raise BackendError("Runtime", f"set_lengths: {n} tokens, {m} of them new")
        if self._free is not None:
            for b, (n, m) in enumerate(zip(lengths, counts or [min(n, 1) for n in lengths])):
                for p in self._held[b][(n - m) // self.page_tokens: -(-n // self.page_tokens)] if m else ():
                    if p is None or self._users[p] > 1:
                        raise BackendError("Runtime", f"set_lengths: new tokens {n - m} to {n} of sequence {b} in a page "
                                                      f"that {'was given back' if p is None else 'others read'}")
            self._afford(sum(self._short(b, n) for b, n in enumerate(lengths)))  # all of them or none
            for b, n in enumerate(lengths):
                self.reserve(b, n, stream)
        with _stream(stream):
            self.seq_len.copy_(torch.tensor(lengths, dtype=torch.int32))
            if counts is not None and self._own_cu is None:
                self._own_cu = torch.empty(self.n_seqs + 1, dtype=torch.int32, device=self.device)
            if self._own_cu is not None:  # one each: for the calls that were recorded with counts
                starts = np.cumsum([0] + (counts or [1] * self.n_seqs))
                self._own_cu.copy_(torch.tensor(starts, dtype=torch.int32))
            self.use_cu_tokens(None if counts is None else self._own_cu)

    def use_cu_tokens(self, cu_tokens) -> None:
        """The device tensor [n_seqs + 1] that says which rows of a call are
        whose, or None for one row each."""
        if cu_tokens is not None:
            if tuple(cu_tokens.shape) != (self.n_seqs + 1,) or cu_tokens.dtype != _torch().int32 \
                    or not cu_tokens.is_contiguous() or cu_tokens.device != self.device:
                raise BackendError("Runtime", f"cu_tokens: contiguous int32 [{self.n_seqs + 1}] expected")
        self.cu_tokens = cu_tokens
        self.desc.cu_tokens = None if cu_tokens is None else cu_tokens.data_ptr()

    # -- operators -----------------------------------------------------------
    def append(self, k: int, v: int, kv_stride: int, n_tokens: int, max_new: int, rope=None,
               q: int = 0, q_stride: int = 0, q_out: int | None = None, q_out_stride: int | None = None,
               n_q_heads: int = 0, stream=None, axes: RopeAxes | None = None, pos: int = 0,
               pos_stride: int | None = None) -> None:
        """Rows of k and v (n_kv_heads*head_dim floats, kv_stride apart) into
        the cache, k rotated by `rope` (a RopeTable); q, if given, rotated to
        q_out (in place by default). With axes, the rows' positions are pos
        [n_axes][pos_stride] (n_tokens by default), not their places."""
        if self._look:
            _on_device(self.device)
        if rope is not None and (self._look or rope._look) and rope.device != self.device:
            raise BackendError("Runtime", f"rope table on {rope.device}, cache on {self.device}")
        if axes is None and pos:
            raise BackendError("Runtime", "append: positions without axes")
        if axes is not None:
            at = axes.at(pos, n_tokens if pos_stride is None else pos_stride)
            kern.kv_append_axes(self._ref, None if rope is None else rope.ref, ctypes.byref(at), k, v, kv_stride, q,
                                q_stride, q if q_out is None else q_out,
                                q_stride if q_out_stride is None else q_out_stride, n_q_heads, n_tokens, max_new, stream)
            return
        kern.kv_append(self._ref, None if rope is None else rope.ref, k, v, kv_stride, q, q_stride,
                       q if q_out is None else q_out, q_stride if q_out_stride is None else q_out_stride,
                       n_q_heads, n_tokens, max_new, stream)

    def attention_workspace(self, n_q_heads: int, n_tokens: int, max_new: int, shared: int = 0):
        """A device tensor for attend's workspace (any call with these sizes; with
        `shared`, any with no more sequences, tokens, new and shared tokens)."""
        if shared:
            n = kern.kv_attention_shared_workspace_bytes(self._ref, n_q_heads, n_tokens, max_new, shared)
        else:
            n = kern.kv_attention_workspace_bytes(self._ref, n_q_heads, max_new)
        if n == 0 or n_tokens <= 0:
            raise BackendError("Runtime", f"attention of {n_q_heads} heads, {max_new} new tokens")
        return _torch().empty(n, dtype=_torch().uint8, device=self.device)

    def attend(self, q: int, q_stride: int, n_q_heads: int, out: int, out_stride: int,
               n_tokens: int, max_new: int, scale: float | None = None, softcap: float = 0.0,
               window: int = 0, out_f16: bool = False, workspace=None, stream=None, sinks: int = 0,
               shared: int = 0) -> None:
        """out = attention of q's rows over the cache (scale: head_dim^-0.5); with a
        window the first `sinks` positions of a sequence stay visible behind it.
        shared: so many first positions of all sequences lie in the same pages, which are
        read once for all (without a window; the workspace is one for `shared`).
        Without a workspace, a fresh one comes from torch's caching allocator,
        of the launch stream."""
        if self._look:
            _on_device(self.device)
        if workspace is None:
            with _stream(stream):
                workspace = self.attention_workspace(n_q_heads, n_tokens, max_new, shared)
        else:
            _workspace(workspace, self.device)
        scale = 1.0 / math.sqrt(self.head_dim) if scale is None else scale
        kind = _lib.OUT_F16 if out_f16 else _lib.OUT_F32
        if shared:
            _without_window(window, sinks)
            kern.kv_attention_shared(self._ref, q, q_stride, n_q_heads, out, out_stride, kind, n_tokens, max_new, scale,
                                     softcap, shared, workspace.data_ptr(), workspace.nbytes, stream)
            return
        if sinks:
            kern.kv_attention_sinks(self._ref, q, q_stride, n_q_heads, out, out_stride, kind, n_tokens, max_new, scale,
                                    softcap, window, sinks, workspace.data_ptr(), workspace.nbytes, stream)
            return
        kern.kv_attention(self._ref, q, q_stride, n_q_heads, out, out_stride, kind, n_tokens, max_new, scale, softcap,
                          window, workspace.data_ptr(), workspace.nbytes, stream)

    def dequant(self, pages: int, n: int, k_out: int, v_out: int, stream=None) -> None:
        """n pages (device int32 ids) as f32 [n][kv head][token][dim]."""
        if self._look:
            _on_device(self.device)
        kern.kv_dequant(self._ref, pages, n, k_out, v_out, stream)

    # -- the same as descriptors of an op chain (q4k.Chain.from_ops) ----------
    def op_append(self, k: int, v: int, kv_stride: int, n_tokens: int, max_new: int, rope=None,
                  q: int = 0, q_stride: int = 0, q_out: int | None = None,
                  q_out_stride: int | None = None, n_q_heads: int = 0, axes: RopeAxes | None = None, pos: int = 0,
                  pos_stride: int | None = None) -> "_lib.OpDesc":
        _on_gpu(self.device)
        if rope is not None and rope.device != self.device:
            raise BackendError("Runtime", f"rope table on {rope.device}, cache on {self.device}")
        args = _lib.KvAppendArgs(
            self.desc, _lib.Rope() if rope is None else rope.desc, k, v, q or None,
            (q if q_out is None else q_out) or None, kv_stride, q_stride,
            q_stride if q_out_stride is None else q_out_stride, n_q_heads, n_tokens, max_new)
        if axes is None:
            if pos:
                raise BackendError("Runtime", "append: positions without axes")
            return _op(_lib.OP_KV_APPEND, args)
        return _op(_lib.OP_KV_APPEND_AXES, _lib.KvAppendAxesArgs(
            args, axes.at(pos, n_tokens if pos_stride is None else pos_stride)))

    def op_attend(self, q: int, q_stride: int, n_q_heads: int, out: int, out_stride: int,
                  n_tokens: int, max_new: int, workspace, scale: float | None = None,
                  softcap: float = 0.0, window: int = 0, out_f16: bool = False, sinks: int = 0,
                  shared: int = 0) -> "_lib.OpDesc":
        """The workspace has to outlive the chain."""
        _on_gpu(self.device)
        _workspace(workspace, self.device)
        args = _lib.KvAttentionArgs(
            self.desc, q, out, workspace.data_ptr(), workspace.numel() * workspace.element_size(),
            q_stride, out_stride, n_q_heads, _lib.OUT_F16 if out_f16 else _lib.OUT_F32, n_tokens,
            max_new, window, 1.0 / math.sqrt(self.head_dim) if scale is None else scale, softcap)
        if shared:
            _without_window(window, sinks)
            return _op(_lib.OP_KV_ATTENTION_SHARED, _lib.KvAttentionSharedArgs(args, shared))
        if sinks:
            return _op(_lib.OP_KV_ATTENTION_SINKS, _lib.KvAttentionSinksArgs(args, sinks))
        return _op(_lib.OP_KV_ATTENTION, args)
