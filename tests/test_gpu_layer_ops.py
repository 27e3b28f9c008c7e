"""A layer's operators together, as a decoder runs them: a recorded step of norms, Q4_K
matvecs, an append at positions of three axes and attention with first tokens that stay
visible; and a batch behind one prompt, its prefix written once and shared."""
import numpy as np
import pytest

from tests import kv_attend_reference as attend_ref
from tests import kv_reference as kv_ref
from tests import rope_axes_reference as axes_ref
from tests.gpu_util import dev, host, random_q4k_bytes
from tests.test_gpu_block_norm import check as check_norm
from tests.test_gpu_kvcache import check as check_attention
from tests.test_gpu_kvcache import note, rope_table_ref

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, HIDDEN = 4, 2, 64, 512
SECTIONS = (8, 12, 12)


def reference_of(cache):
    """The cache's bytes as they are, for the 64-bit attention."""
    return kv_ref.Cache(host(cache.k), host(cache.v), host(cache.k_scale), host(cache.v_scale), host(cache.page_table),
                        cache.format)


def test_recorded_decode_step():
    import torch
    from modgrad_amd.kvcache import KvCache, RopeAxes, RopeTable
    from modgrad_amd.norm import BlockNorm
    from modgrad_amd.q4k import Chain, kern, op_matvec
    from modgrad_amd import _lib
    note("a recorded decode step")
    rng = np.random.default_rng(1)
    row = (HEADS + 2 * KV) * DIM
    w_qkv, w_o = (dev(random_q4k_bytes(rng, n * k // 256)) for n, k in ((row, HIDDEN), (HIDDEN, HEADS * DIM)))
    weights = [rng.uniform(0.5, 1.5, HIDDEN).astype(np.float32) for _ in range(3)]
    pre, post, after = map(dev, weights)
    gate = rng.uniform(0.2, 1.0, HIDDEN).astype(np.float32)
    first = BlockNorm(HIDDEN, 1e-6, norm_w=pre)
    join = BlockNorm(HIDDEN, 1e-6, post_w=post, norm_w=after, gate=dev(gate), x_scale=0.5)
    table = rope_table_ref(100, 2 * sum(SECTIONS)).astype(np.float32)
    rope, axes = RopeTable.wrap(dev(table), True), RopeAxes(SECTIONS)
    window, sinks, eps = 40, 6, 1e-6

    def side():
        b = {"cache": KvCache.new(12, 16, KV, DIM, 1, 12, fmt="i8"), "h": torch.empty(1, HIDDEN, device="cuda"),
             "pos": torch.empty(3, 1, dtype=torch.int32, device="cuda")}
        for name, n in (("x", HIDDEN), ("qkv", row), ("q", HEADS * DIM), ("att", HEADS * DIM), ("o", HIDDEN), ("y", HIDDEN)):
            b[name] = torch.empty(1, n, device="cuda")
        b["cache"].set_lengths([1])
        b["ws"] = b["cache"].attention_workspace(HEADS, 1, 1)
        b["at"] = {k: t.data_ptr() for k, t in b.items() if isinstance(t, torch.Tensor)}
        return b

    def append_args(b):
        at = b["at"]
        return (at["qkv"] + 4 * HEADS * DIM, at["qkv"] + 4 * (HEADS + KV) * DIM, row, 1, 1), dict(
            rope=rope, q=at["qkv"], q_stride=row, q_out=at["q"], q_out_stride=HEADS * DIM, n_q_heads=HEADS, axes=axes,
            pos=at["pos"])

    def attend_args(b):
        at = b["at"]
        return (at["q"], HEADS * DIM, HEADS, at["att"], HEADS * DIM, 1, 1), dict(window=window, sinks=sinks,
                                                                                 workspace=b["ws"])
    a, b = side(), side()
    at, (pa, pk), (ta, tk) = a["at"], append_args(a), attend_args(a)
    chain = Chain.from_ops([
        first.op(at["h"], 0, 1, h_out=0, y=at["x"]),
        op_matvec(_lib.DTYPE_Q4_K, w_qkv.data_ptr(), at["x"], at["qkv"], row, HIDDEN),
        a["cache"].op_append(*pa, **pk), a["cache"].op_attend(*ta, **tk),
        op_matvec(_lib.DTYPE_Q4_K, w_o.data_ptr(), at["att"], at["o"], HIDDEN, HEADS * DIM),
        join.op(at["h"], at["o"], 1, y=at["y"])])
    for step in range(70):
        h = rng.standard_normal((1, HIDDEN)).astype(np.float32)
        p = np.array([[step], [step // 3 + 2], [step % 7]], np.int32)
        for s in (a, b):
            s["h"].copy_(torch.from_numpy(h))
            s["pos"].copy_(torch.from_numpy(p))
            s["cache"].set_lengths([step + 1])
        chain.launch()
        bt, (qa, qk), (ua, uk) = b["at"], append_args(b), attend_args(b)
        first.apply(bt["h"], 0, 1, h_out=0, y=bt["x"])
        kern.matvec_q4k(w_qkv.data_ptr(), bt["x"], bt["qkv"], row, HIDDEN // 256)
        b["cache"].append(*qa, **qk)
        b["cache"].attend(*ua, **uk)
        kern.matvec_q4k(w_o.data_ptr(), bt["att"], bt["o"], HIDDEN, HEADS * DIM // 256)
        join.apply(bt["h"], bt["o"], 1, y=bt["y"])
        for name in ("x", "qkv", "q", "att", "o", "h", "y"):
            assert np.array_equal(host(a[name]), host(b[name])), (step, name)
        assert np.array_equal(host(a["cache"].k), host(b["cache"].k))
        if step % 10 and step != 69:
            continue
        # each operator's results from what it was given
        check_norm(h, None, None, None, weights[0], 1.0, 1.0, eps, None, host(a["x"]))
        qkv = host(a["qkv"]).reshape(HEADS + 2 * KV, DIM)
        q = axes_ref.turn(qkv[None, :HEADS], p, table, SECTIONS, "blocks", False, True)
        assert np.all(np.abs(host(a["q"]).reshape(q.shape) - q) <= 2.0 ** -24 * np.abs(q) + 1e-15)
        want, tol = attend_ref.attend(reference_of(a["cache"]), host(a["q"]).reshape(1, HEADS, DIM), [step + 1], [1],
                                      DIM ** -0.5, 0.0, window, sinks)
        check_attention(host(a["att"]).reshape(want.shape), want, tol, False)
        check_norm(h, host(a["o"]), weights[1], gate, weights[2], 1.0, 0.5, eps, host(a["h"]), host(a["y"]))


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_batch_behind_one_prompt(fmt):
    """A prompt with a picture is written once; the sequences' tables begin with its pages."""
    import torch
    from modgrad_amd.kvcache import KvCache, RopeAxes, RopeTable
    from modgrad_amd.norm import BlockNorm
    note(f"a batch behind one prompt {fmt}")
    rng = np.random.default_rng(2)
    seqs, prefix, page, heads, group = 24, 1024, 32, 2, 3
    hq, hidden = heads * group, 384
    row = (hq + 2 * heads) * DIM
    common = prefix // page
    cache = KvCache.new(common + 3 * seqs, page, heads, DIM, seqs, common + 3, fmt=fmt)
    table = rope_table_ref(1200, 2 * sum(SECTIONS)).astype(np.float32)
    rope, axes = RopeTable.wrap(dev(table), True), RopeAxes(SECTIONS, "turns")
    # the prompt, as sequence 0's
    x = dev(rng.standard_normal((prefix, row)).astype(np.float32))
    pos = rng.integers(0, 1000, (3, prefix)).astype(np.int32)
    cache.set_lengths([prefix] + [0] * (seqs - 1), [prefix] + [0] * (seqs - 1))
    q = torch.empty(prefix, hq * DIM, device="cuda")
    pt = dev(pos)
    cache.append(x.data_ptr() + 4 * hq * DIM, x.data_ptr() + 4 * (hq + heads) * DIM, row, prefix, prefix, rope=rope,
                 q=x.data_ptr(), q_stride=row, q_out=q.data_ptr(), q_out_stride=hq * DIM, n_q_heads=hq, axes=axes,
                 pos=pt.data_ptr())
    # the others begin with its pages, and have three of their own
    t = host(cache.page_table).copy()
    used = set(t[0, :common])
    free = [p for p in range(cache.n_pages) if p not in used]
    t[:, :common] = t[0, :common]
    t[:, common:] = np.array(free[:3 * seqs], np.int32).reshape(seqs, 3)
    wrapped = KvCache.wrap(cache.k, cache.v, cache.k_scale, cache.v_scale, dev(t), cache.seq_len, fmt=fmt)
    weights = [rng.uniform(0.5, 1.5, hidden).astype(np.float32) for _ in range(2)]
    norm = BlockNorm(hidden, 1e-6, post_w=dev(weights[0]), norm_w=dev(weights[1]))
    lens = [prefix] * seqs
    for step in range(4):
        new = [1] * seqs if step % 2 else [int(n) for n in rng.integers(0, 20, seqs)]
        lens = [a + b for a, b in zip(lens, new)]
        rows = sum(new)
        x = dev(rng.standard_normal((rows, row)).astype(np.float32))
        pos = rng.integers(0, 1200, (3, rows)).astype(np.int32)
        pt, q = dev(pos), torch.empty(rows, hq * DIM, device="cuda")
        wrapped.set_lengths(lens, None if step % 2 else new)
        wrapped.append(x.data_ptr() + 4 * hq * DIM, x.data_ptr() + 4 * (hq + heads) * DIM, row, rows, max(new), rope=rope,
                       q=x.data_ptr(), q_stride=row, q_out=q.data_ptr(), q_out_stride=hq * DIM, n_q_heads=hq, axes=axes,
                       pos=pt.data_ptr())
        out = torch.empty(rows, hq * DIM, device="cuda")
        wrapped.attend(q.data_ptr(), hq * DIM, hq, out.data_ptr(), hq * DIM, rows, max(new), shared=prefix)
        want = axes_ref.turn(host(x)[:, :hq * DIM].reshape(rows, hq, DIM), pos, table, SECTIONS, "turns", False, True)
        assert np.all(np.abs(host(q).reshape(want.shape) - want) <= 2.0 ** -24 * np.abs(want) + 1e-15)
        want, tol = attend_ref.attend(reference_of(wrapped), host(q).reshape(rows, hq, DIM), lens, new, DIM ** -0.5)
        check_attention(host(out).reshape(want.shape), want, tol, False)
        alone = torch.empty_like(out)
        wrapped.attend(q.data_ptr(), hq * DIM, hq, alone.data_ptr(), hq * DIM, rows, max(new))
        check_attention(host(alone).reshape(want.shape), want, tol, False)
        # the block's end: its result normalized into the stream, that normalized for the next
        h = rng.standard_normal((rows, hidden)).astype(np.float32)
        ht, y = dev(h), torch.empty(rows, hidden, device="cuda", dtype=torch.float16)
        norm.apply(ht.data_ptr(), out.data_ptr(), rows, y=y.data_ptr(), y_f16=True)
        check_norm(h, host(out), weights[0], None, weights[1], 1.0, 1.0, 1e-6, host(ht), host(y))
