"""The norms around a block (launch_block_norm_ex, modgrad_amd.norm) against their
formulas in 64 bits.

Tolerances, in steps of f32 (2^-24 of a value each). The factor r is a 64-bit root rounded
to f32; z takes it and is multiplied by r, the weight and the gate: 4 roundings. h_scale h is
one, the sum with x_scale z (fused) another: |h'| + |h_scale h| + 4 |x_scale gate z| of them.
y is compared with the norm of the h' that came back: the factor, its product and the
weight's, 3 roundings, and half a step of f16 (2^-11). Where h' does not come back, an h'
that is off by d moves y by r w d and, through the mean, by |y| rms(d) / rms(h'). What falls
below the least numbers adds 2^-145 (2^-25 in f16)."""
import numpy as np
import pytest

from modgrad_amd import _lib
from tests.gpu_util import dev, host

pytestmark = pytest.mark.gpu
STEP = 1.001 * 2.0 ** -24  # and what products of roundings add


def note(msg):
    print(f"[case] {msg}", flush=True)


def rstd(a, eps):
    return 1.0 / np.sqrt((a * a).mean(1, keepdims=True) + np.float64(np.float32(eps)))


def check(h, x, post_w, gate, norm_w, h_scale, x_scale, eps, h_got, y_got):
    f = np.float64
    z = 0.0
    if x is not None:
        z = x.astype(f)
        if post_w is not None:
            z = z * rstd(z, eps) * post_w
        if gate is not None:
            z = z * gate
        z = f(np.float32(x_scale)) * z
    a = f(np.float32(h_scale)) * h.astype(f)
    want = a + z
    d = STEP * (np.abs(want) + np.abs(a) + 4 * np.abs(z)) + 2.0 ** -145
    if h_got is not None:
        assert h_got.dtype == np.float32
        assert np.all(np.abs(h_got - want) <= d)
    if y_got is not None:
        of = (want if h_got is None else h_got).astype(f)
        r = rstd(of, eps)
        y = of * r * norm_w
        half = y_got.dtype == np.float16
        tol = (3 * STEP + (2.0 ** -11 if half else 0)) * np.abs(y) + (2.0 ** -25 if half else 2.0 ** -145)
        if h_got is None:
            rms = lambda v: np.sqrt((v * v).mean(1, keepdims=True))  # noqa: E731
            tol += 1.001 * (r * np.abs(norm_w) * d + np.abs(y) * rms(d) / rms(of))
        assert np.all(np.abs(y_got - y) <= tol)


def inputs(rows, hidden, seed=0, gates=0):
    rng = np.random.default_rng([rows, hidden, seed])
    h = (3 * rng.standard_normal((rows, hidden))).astype(np.float32)
    h[:, ::97] *= 20
    x = rng.standard_normal((rows, hidden)).astype(np.float32)
    w1, w2 = (rng.uniform(0.2, 2, hidden).astype(np.float32) for _ in range(2))
    gate = rng.standard_normal((rows if gates == 2 else 1, hidden)).astype(np.float32) if gates else None
    return h, x, w1, w2, gate


# around each variant's limits: a wavefront, four quads of it, a work-group of 256 and
# of 1024 threads, longer rows; odd ends
@pytest.mark.parametrize("rows,hidden", [
    (1, 1), (1, 2), (3, 3), (5, 4), (2, 63), (7, 255), (4, 256), (9, 257), (1, 896), (37, 1023), (2, 1024), (3, 1025),
    (1, 3584), (6, 3583), (5, 4096), (2, 4097), (3, 4864), (1, 16384), (2, 16385), (1, 18944), (2, 40003),
    (1100, 250), (1500, 897), (1200, 3585), (1031, 5001)])
@pytest.mark.parametrize("f16", [False, True])
def test_sizes(rows, hidden, f16):
    import torch
    from modgrad_amd.norm import BlockNorm
    note(f"norm rows={rows} hidden={hidden} f16={f16}")
    gates = (rows + hidden) % 3
    h, x, w1, w2, gate = inputs(rows, hidden, gates=gates)
    eps, hs, xs = 1e-5, 0.75, 0.31
    n = BlockNorm(hidden, eps, post_w=dev(w1), norm_w=dev(w2), gate=dev(gate[0]) if gates == 1 else None, h_scale=hs,
                  x_scale=xs)
    ht, xt, gt = dev(h), dev(x), dev(gate) if gates == 2 else None
    ho = torch.full((rows + 1, hidden), 7.0, device="cuda")
    y = torch.full((rows + 1, hidden), 7.0, device="cuda", dtype=torch.float16 if f16 else torch.float32)
    n.apply(ht.data_ptr(), xt.data_ptr(), rows, h_out=ho.data_ptr(), y=y.data_ptr(), y_f16=f16,
            gate=gt.data_ptr() if gates == 2 else 0)
    got, yg = host(ho), host(y)
    assert np.all(got[rows] == 7) and np.all(yg[rows] == 7) and np.array_equal(host(ht), h)
    check(h, x, w1, gate, w2, hs, xs, eps, got[:rows], yg[:rows])
    # in place
    n.apply(ht.data_ptr(), xt.data_ptr(), rows, y=y.data_ptr(), y_f16=f16, gate=gt.data_ptr() if gates == 2 else 0)
    assert np.array_equal(host(ht), got[:rows]) and np.array_equal(host(y), yg)


@pytest.mark.parametrize("hidden", [130, 1500, 20001])
@pytest.mark.parametrize("parts", ["x", "post", "gate", "pre", "x+pre", "post+pre", "only h", "y alone"])
def test_parts(parts, hidden):
    """Each norm, the gate, the block's result and each output left out."""
    import torch
    from modgrad_amd.norm import BlockNorm
    note(f"norm {parts} hidden={hidden}")
    rows = 5
    h, x, w1, w2, gate = inputs(rows, hidden, 1, gates=1)
    post, pre = "post" in parts, "pre" in parts or parts == "y alone"
    use_x, use_gate = parts not in ("pre", "only h"), parts == "gate"
    n = BlockNorm(hidden, 1e-6, post_w=dev(w1) if post else None, norm_w=dev(w2) if pre else None,
                  gate=dev(gate[0]) if use_gate else None, h_scale=1.5)
    ht, xt = dev(h), dev(x)
    ho, y = (torch.full((rows, hidden), 7.0, device="cuda") for _ in range(2))
    n.apply(ht.data_ptr(), xt.data_ptr() if use_x else 0, rows, h_out=0 if parts == "y alone" else ho.data_ptr(),
            y=y.data_ptr() if pre else 0)
    got, yg = host(ho), host(y)
    if parts == "y alone":
        assert np.all(got == 7)
        got = None
    if not pre:
        assert np.all(yg == 7)
        yg = None
    check(h, x if use_x else None, w1 if post else None, gate if use_gate else None, w2, 1.5, 1.0, 1e-6, got, yg)


@pytest.mark.parametrize("hidden", [60, 1001, 17000])
@pytest.mark.parametrize("off", [0, 1, 2, 3])
def test_strides(hidden, off):
    """Rows apart, at every alignment of a float; what lies between them stays."""
    import torch
    from modgrad_amd.norm import BlockNorm
    note(f"norm hidden={hidden} off={off}")
    rows, gaps = 4, (3, 5, 1, 2, 7)
    h, x, w1, w2, gate = inputs(rows, hidden, 2, gates=2)
    n = BlockNorm(hidden, 1e-6, post_w=dev(w1), norm_w=dev(w2))

    def spread(a, gap):
        b = np.full(off + rows * (hidden + gap), 9.0, np.float32)
        b[off:].reshape(rows, -1)[:, :hidden] = a
        return dev(b)
    ht, xt, gt = spread(h, gaps[0]), spread(x, gaps[1]), spread(gate, gaps[2])
    ho = torch.full((off + rows * (hidden + gaps[3]),), 7.0, device="cuda")
    y = torch.full((off + rows * (hidden + gaps[4]),), 7.0, device="cuda", dtype=torch.float16)
    n.apply(ht.data_ptr() + 4 * off, xt.data_ptr() + 4 * off, rows, h_out=ho.data_ptr() + 4 * off,
            y=y.data_ptr() + 2 * off, y_f16=True, gate=gt.data_ptr() + 4 * off, gate_stride=hidden + gaps[2],
            h_stride=hidden + gaps[0], x_stride=hidden + gaps[1], h_out_stride=hidden + gaps[3],
            y_stride=hidden + gaps[4])
    got, yg = (host(t)[off:].reshape(rows, -1) for t in (ho, y))
    assert np.all(host(ho)[:off] == 7) and np.all(host(y)[:off] == 7)
    assert np.all(got[:, hidden:] == 7) and np.all(yg[:, hidden:] == 7)
    check(h, x, w1, gate, w2, 1.0, 1.0, 1e-6, got[:, :hidden], yg[:, :hidden])


@pytest.mark.parametrize("hidden", [100, 2000, 20000])
def test_far_values(hidden):
    """Rows whose squares leave f32 on either side, a row of zeros."""
    import torch
    from modgrad_amd.norm import BlockNorm
    note(f"norm far values hidden={hidden}")
    h, x, w1, w2, _ = inputs(6, hidden, 3)
    scale = np.array([1e25, 1e-25, 1e-38, 1.0, 1e30, 0.0], np.float32)[:, None]
    h, x = h * scale, x * scale[::-1]
    for eps in (1e-6, 0.0):
        n = BlockNorm(hidden, eps, post_w=dev(w1), norm_w=dev(w2))
        ho, y = (torch.empty(6, hidden, device="cuda") for _ in range(2))
        ht, xt = dev(h), dev(x)
        n.apply(ht.data_ptr(), xt.data_ptr(), 6, h_out=ho.data_ptr(), y=y.data_ptr())
        got, yg = host(ho), host(y)
        with np.errstate(all="ignore"):
            rows = slice(None) if eps else slice(1, 6)  # zeros over no eps: 0 times infinity
            check(h[rows], x[rows], w1, None, w2, 1.0, 1.0, eps, got[rows], yg[rows])
        if not eps:
            assert np.all(np.isnan(got[0])) and np.all(np.isnan(yg[0]))


def test_not_finite():
    """A NaN makes its row NaN; an infinity makes a NaN of its place and zeros of the
    others (finite over infinite); rows beside are as they were."""
    import torch
    from modgrad_amd.norm import BlockNorm
    note("norm not finite")
    h, x, w1, w2, _ = inputs(4, 700, 4)
    x[1, 5], h[2, 699], x[3, 0] = np.nan, np.nan, np.inf
    n = BlockNorm(700, 1e-6, post_w=dev(w1), norm_w=dev(w2))
    ho, y = (torch.empty(4, 700, device="cuda") for _ in range(2))
    ht, xt = dev(h), dev(x)
    n.apply(ht.data_ptr(), xt.data_ptr(), 4, h_out=ho.data_ptr(), y=y.data_ptr())
    got, yg = host(ho), host(y)
    check(h[:1], x[:1], w1, None, w2, 1.0, 1.0, 1e-6, got[:1], yg[:1])
    assert np.all(np.isnan(got[1])) and np.all(np.isnan(yg[1]))
    assert np.isnan(got[2]).sum() == 1 and np.all(np.isnan(yg[2]))
    assert np.isnan(got[3, 0]) and np.array_equal(got[3, 1:], h[3, 1:])


def test_f16_past_its_largest():
    import torch
    from modgrad_amd.norm import BlockNorm
    note("norm f16 past its largest")
    h = np.ones((1, 64), np.float32)
    w = np.full(64, 65519.0, np.float32)  # rounds down to 65504, 65520 up to infinity
    w[1::2] = 65520.0
    n = BlockNorm(64, 0.0, norm_w=dev(w))
    y = torch.empty(1, 64, device="cuda", dtype=torch.float16)
    ht = dev(h)
    n.apply(ht.data_ptr(), 0, 1, h_out=0, y=y.data_ptr(), y_f16=True)
    got = host(y)[0]
    assert np.all(got[::2] == 65504) and np.all(np.isinf(got[1::2]))


def test_stream_and_graph():
    """On another stream, and captured and replayed on new values."""
    import torch
    from modgrad_amd.norm import BlockNorm
    note("norm on a stream and in a graph")
    rows, hidden = 3, 3584
    h, x, w1, w2, _ = inputs(rows, hidden, 5)
    n = BlockNorm(hidden, 1e-6, post_w=dev(w1), norm_w=dev(w2))
    ht, xt = dev(h), dev(x)
    ho, y = (torch.empty(rows, hidden, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    call = lambda: n.apply(ht.data_ptr(), xt.data_ptr(), rows, h_out=ho.data_ptr(), y=y.data_ptr(), stream=s)  # noqa: E731
    call()
    s.synchronize()
    check(h, x, w1, None, w2, 1.0, 1.0, 1e-6, host(ho), host(y))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        call()
    for seed in range(3):
        h, x = inputs(rows, hidden, 6 + seed)[:2]
        ht.copy_(torch.from_numpy(h))
        xt.copy_(torch.from_numpy(x))
        ho.zero_()
        g.replay()
        check(h, x, w1, None, w2, 1.0, 1.0, 1e-6, host(ho), host(y))


def test_chain_op():
    """In an op chain between matvecs' buffers: the same bits as the call."""
    import torch
    from modgrad_amd.norm import BlockNorm
    from modgrad_amd.q4k import Chain, op_residual_add
    note("norm in a chain")
    hidden = 3584
    h, x, w1, w2, gate = inputs(1, hidden, 9, gates=1)
    n = BlockNorm(hidden, 1e-6, post_w=dev(w1), norm_w=dev(w2), gate=dev(gate[0]), x_scale=0.5)
    a, b, xt = dev(h), dev(h), dev(x)
    ya, yb = (torch.empty(1, hidden, device="cuda") for _ in range(2))
    chain = Chain.from_ops([n.op(a.data_ptr(), xt.data_ptr(), 1, y=ya.data_ptr()),
                            op_residual_add(a.data_ptr(), ya.data_ptr(), hidden),
                            n.op(a.data_ptr(), ya.data_ptr(), 1, y=xt.data_ptr())])
    x2 = dev(x)
    chain.launch()
    n.apply(b.data_ptr(), x2.data_ptr(), 1, y=yb.data_ptr())
    b += yb
    n.apply(b.data_ptr(), yb.data_ptr(), 1, y=x2.data_ptr())
    assert np.array_equal(host(a), host(b)) and np.array_equal(host(xt), host(x2))


def test_many_rows():
    """More rows than a launch has work-groups: 2^20 and some, of 4 values."""
    import torch
    from modgrad_amd.norm import BlockNorm
    note("norm of 2^22 + 5 rows")
    rows = (1 << 22) + 5
    h, x, w1, w2, _ = inputs(rows, 4, 10)
    n = BlockNorm(4, 1e-6, post_w=dev(w1), norm_w=dev(w2))
    ht, xt = dev(h), dev(x)
    ho, y = (torch.empty(rows, 4, device="cuda") for _ in range(2))
    n.apply(ht.data_ptr(), xt.data_ptr(), rows, h_out=ho.data_ptr(), y=y.data_ptr())
    check(h, x, w1, None, w2, 1.0, 1.0, 1e-6, host(ho), host(y))


def test_python_refusals():
    import torch
    from modgrad_amd.norm import BlockNorm
    from modgrad_amd.q4k import BackendError
    w = torch.ones(64, device="cuda")
    for bad in (dict(post_w=w[:63]), dict(norm_w=w.double()), dict(gate=torch.ones(128, device="cuda")[::2]),
                dict(post_w=w, norm_w=w.cpu())):
        with pytest.raises(BackendError):
            BlockNorm(64, 1e-6, **bad)
    n = BlockNorm(64, 1e-6, gate=w)
    with pytest.raises(BackendError):
        n.apply(w.data_ptr(), w.data_ptr(), 1, gate=w.data_ptr())
    with pytest.raises(BackendError):
        n.apply(w.data_ptr(), 0, 1, h_out=0)
    assert _lib.OP_BLOCK_NORM == 12
