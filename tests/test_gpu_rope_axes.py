"""Rotary positions of several axes on the GPU, alone and in an append to the cache,
against the 64-bit reference of tests/rope_axes_reference.py."""
import numpy as np
import pytest

from tests import rope_axes_reference as ref
from tests.gpu_util import dev, host
from tests.test_gpu_kvcache import Both, note, rope_table_ref

pytestmark = pytest.mark.gpu


def table_of(n_pos, sections, own):
    return rope_table_ref(n_pos, 2 * (max(sections) if own else sum(sections))).astype(np.float32)


def close(got, want):
    """One rounding to f32 (2^-24 relative) of a 64-bit value; NaN where NaN is due."""
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    assert np.all(np.abs(got - want)[fine] <= 2.0 ** -24 * np.abs(want)[fine] + 1e-15)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("order", ["blocks", "turns"])
@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,sections,gap,off", [
    (1, 28, 128, (16, 24, 24), 0, 0), (1, 1, 2, (1,), 0, 0), (7, 3, 80, (20, 20), 3, 1), (33, 2, 64, (11, 11, 10), 0, 0),
    (5, 4, 96, (0, 24, 0, 24), 5, 2), (9, 2, 128, (1, 2, 3, 4), 0, 3), (300, 5, 128, (24, 20, 20, 0), 16, 0),
    (4, 1, 512, (64, 64, 64, 64), 0, 0), (4, 1, 512, (3, 250, 1, 2), 0, 0), (2, 3, 72, (17, 19), 0, 0),
    (17, 2, 256, (5, 5, 5, 5), 0, 0), (3, 2, 66, (9, 0, 20), 0, 0)])
def test_turn(tokens, heads, dim, sections, gap, off, own, order, half):
    import torch
    from modgrad_amd.kvcache import RopeAxes, RopeTable
    note(f"axes tokens={tokens} heads={heads} dim={dim} {sections} {order} own={own} half={half} gap={gap} off={off}")
    rng = np.random.default_rng([tokens, dim, *sections])
    table = table_of(97, sections, own)
    rope, axes = RopeTable.wrap(dev(table), half), RopeAxes(sections, order, own)
    stride = heads * dim + gap
    x = rng.standard_normal(off + tokens * stride).astype(np.float32)
    pos = rng.integers(0, 97, (len(sections), tokens + off)).astype(np.int32)
    for a, n in enumerate(sections):
        if n == 0:
            pos[a] = -2 ** 31  # not read
    xt, pt = dev(x), dev(pos)
    yt = torch.full((tokens * (stride + 3),), 7.0, device="cuda")
    rope.apply(xt.data_ptr() + 4 * off, yt.data_ptr(), pt.data_ptr(), tokens, heads, dim, stride, stride + 3, axes=axes,
               pos_stride=tokens + off)
    rows = x[off:].reshape(tokens, stride)[:, :heads * dim].reshape(tokens, heads, dim)
    want = ref.turn(rows, pos[:, :tokens], table, sections, order, own, half)
    got = host(yt).reshape(tokens, stride + 3)
    assert np.all(got[:, heads * dim:] == 7.0)
    got = got[:, :heads * dim].reshape(tokens, heads, dim)
    close(got, want)
    assert np.array_equal(got[..., 2 * sum(sections):], rows[..., 2 * sum(sections):])
    rope.apply(xt.data_ptr() + 4 * off, xt.data_ptr() + 4 * off, pt.data_ptr(), tokens, heads, dim, stride, stride,
               axes=axes, pos_stride=tokens + off)
    again = host(xt)[off:].reshape(tokens, stride)
    assert np.array_equal(again[:, :heads * dim].reshape(got.shape), got)
    assert np.array_equal(again[:, heads * dim:], x[off:].reshape(tokens, stride)[:, heads * dim:])


def test_one_axis_is_the_plain_call():
    import torch
    from modgrad_amd.kvcache import RopeAxes, RopeTable
    note("axes: one axis, and the same position on three")
    rng = np.random.default_rng(3)
    for half in (False, True):
        rope = RopeTable.wrap(dev(rope_table_ref(50, 128).astype(np.float32)), half)
        x = torch.randn(6, 3, 128, device="cuda")
        p = dev(np.tile(rng.integers(0, 50, 6).astype(np.int32), (3, 1)))
        y, z, w = (torch.empty_like(x) for _ in range(3))
        rope.apply(x.data_ptr(), y.data_ptr(), p.data_ptr(), 6, 3, 128)
        rope.apply(x.data_ptr(), z.data_ptr(), p.data_ptr(), 6, 3, 128, axes=RopeAxes([64]))
        rope.apply(x.data_ptr(), w.data_ptr(), p.data_ptr(), 6, 3, 128, axes=RopeAxes([20, 30, 14], "turns"))
        assert np.array_equal(host(y), host(z)) and np.array_equal(host(y), host(w))


@pytest.mark.parametrize("dim,sections", [(64, (16, 16)), (66, (16, 17))])
def test_positions_outside_the_table(dim, sections):
    import torch
    from modgrad_amd.kvcache import RopeAxes, RopeTable
    note(f"axes: positions outside the table, dim={dim}")
    table = table_of(10, sections, False)
    rope = RopeTable.wrap(dev(table), True)
    pos = np.array([[9, 10, 0, -1, 2 ** 31 - 1, 3], [0, 0, -2 ** 31, 1, 2, 10]], np.int32)
    x, p = torch.ones(6, 1, dim, device="cuda"), dev(pos)
    y = torch.zeros(6, 1, dim, device="cuda")
    rope.apply(x.data_ptr(), y.data_ptr(), p.data_ptr(), 6, 1, dim, axes=RopeAxes(sections))
    got = host(y)
    close(got, ref.turn(np.ones((6, 1, dim)), pos, table, sections, "blocks", False, True))
    assert np.all(np.isnan(got[1:])) and np.all(np.isfinite(got[0]))


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("heads,qh,dim,sections,page,half,order,own", [
    (2, 14, 128, (16, 24, 24), 16, True, "blocks", False), (1, 3, 64, (11, 11, 10), 64, False, "turns", False),
    (2, 2, 96, (13, 0, 20), 32, True, "turns", True), (1, 2, 256, (40, 40, 41), 16, True, "blocks", True)])
def test_append_steps(fmt, heads, qh, dim, sections, page, half, order, own):
    """Prompts, single tokens and pieces at positions that are not their places: every
    byte and scale as the reference's."""
    import torch
    from modgrad_amd.kvcache import RopeAxes, RopeTable
    rng = np.random.default_rng(heads * 1000 + dim + page)
    both = Both(rng, 3, 4, heads, dim, page, fmt)
    table = table_of(23, sections, own)  # fewer positions than the cache has places
    rope, axes = RopeTable.wrap(dev(table), half), RopeAxes(sections, order, own)
    lens = [0, 0, 0]
    for step, new in enumerate([[page + 3, 0, 1], [1, 1, 1], [1, 2 * page, 0], [1, 1, 1], [2, 1, page], [1, 1, 1]]):
        note(f"axes append {fmt} heads={heads} dim={dim} page={page} {sections} {order} step={step} new={new}")
        lens = [a + b for a, b in zip(lens, new)]
        both.call(lens, new, new == [1, 1, 1] and step % 2 == 1)
        t = sum(new)
        row = (qh + 2 * heads) * dim + 5
        x = rng.standard_normal((t, row)).astype(np.float32) * np.float32(1.0 + step)
        x[:, ::7] *= 3
        pos = rng.integers(0, 23, (len(sections), t + 2)).astype(np.int32)
        if step == 4:
            pos[2, 1] = 23  # outside: its query is NaN, its key counts as 0
        xt, pt = dev(x), dev(pos)
        qo = torch.full((t + 1, qh * dim + 1), 7.0, device="cuda")
        both.gpu.append(xt.data_ptr() + 4 * qh * dim, xt.data_ptr() + 4 * (qh + heads) * dim, row, t, max(new),
                        rope=rope, q=xt.data_ptr(), q_stride=row, q_out=qo.data_ptr(), q_out_stride=qh * dim + 1,
                        n_q_heads=qh, axes=axes, pos=pt.data_ptr(), pos_stride=t + 2)
        q, k = (ref.turn(x[:, a * dim:b * dim].reshape(t, b - a, dim), pos[:, :t], table, sections, order, own, half)
                for a, b in ((0, qh), (qh, qh + heads)))
        v = x[:, (qh + heads) * dim:(qh + 2 * heads) * dim].reshape(t, heads, dim).astype(np.float64)
        at = 0
        for b in range(3):
            both.ref.append(b, lens[b] - new[b], k[at:at + new[b]], v[at:at + new[b]])
            at += new[b]
        both.same()
        got = host(qo)
        assert np.all(got[t] == 7.0) and np.all(got[:, qh * dim:] == 7.0)
        close(got[:t, :qh * dim].reshape(q.shape), q)


def test_append_without_queries_and_refusals():
    from modgrad_amd.kvcache import RopeAxes, RopeTable
    from modgrad_amd.q4k import BackendError
    note("axes append without queries")
    rng = np.random.default_rng(8)
    both = Both(rng, 2, 2, 1, 64, 16, "i8")
    sections = (10, 12, 10)
    table = table_of(9, sections, False)
    rope, axes = RopeTable.wrap(dev(table), True), RopeAxes(sections)
    both.call([5, 3], [5, 3])
    x = rng.standard_normal((8, 2, 1, 64)).astype(np.float32)
    pos = rng.integers(0, 9, (3, 8)).astype(np.int32)
    xt, pt = dev(x), dev(pos)
    both.gpu.append(xt.data_ptr(), xt.data_ptr() + 256, 128, 8, 5, rope=rope, axes=axes, pos=pt.data_ptr())
    k = ref.turn(x[:, 0], pos, table, sections, "blocks", False, True)
    both.ref.append(0, 0, k[:5], x[:5, 1].astype(np.float64))
    both.ref.append(1, 0, k[5:], x[5:, 1].astype(np.float64))
    both.same()
    for bad in (dict(rope=None, axes=axes, pos=pt.data_ptr()), dict(rope=rope, axes=axes), dict(rope=rope, pos=pt.data_ptr()),
                dict(rope=rope, axes=RopeAxes([10, 10]), pos=pt.data_ptr()),
                dict(rope=rope, axes=axes, pos=pt.data_ptr(), pos_stride=7)):
        with pytest.raises(BackendError):
            both.gpu.append(xt.data_ptr(), xt.data_ptr() + 256, 128, 8, 5, **bad)
    both.same()


def test_chain_and_graph():
    """Recorded in an op chain and in a captured graph, replayed on new positions."""
    import torch
    from modgrad_amd.kvcache import KvCache, RopeAxes, RopeTable
    from modgrad_amd.q4k import Chain
    note("axes in a chain and a graph")
    sections, heads, dim = (16, 24, 24), 2, 128
    table = table_of(40, sections, False)
    rope, axes = RopeTable.wrap(dev(table), True), RopeAxes(sections)
    caches = [KvCache.new(8, 16, heads, dim, 2, 4) for _ in range(3)]
    x = torch.empty(2, (4 + 2 * heads) * dim, device="cuda")
    pos = torch.empty(3, 2, dtype=torch.int32, device="cuda")
    qs = [torch.empty(2, 4 * dim, device="cuda") for _ in range(3)]
    y = [torch.empty(2, 4 * dim, device="cuda") for _ in range(3)]
    row, at, s = x.shape[1], x.data_ptr(), torch.cuda.Stream()
    for c in caches:
        c.set_lengths([1, 1])

    def args(i):
        return (at + 16 * dim, at + 4 * (4 + heads) * dim, row, 2, 1), dict(
            rope=rope, q=at, q_stride=row, q_out=qs[i].data_ptr(), q_out_stride=4 * dim, n_q_heads=4, axes=axes,
            pos=pos.data_ptr())
    turn = lambda i: (at, y[i].data_ptr(), pos.data_ptr(), 2, 4, dim, row, 4 * dim)  # noqa: E731
    a, k = args(0)
    chain = Chain.from_ops([rope.op(*turn(0), axes=axes), caches[0].op_append(*a, **k)])
    a, k = args(1)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        rope.apply(*turn(1), axes=axes, stream=s)
        caches[1].append(*a, **k, stream=s)
    rng = np.random.default_rng(4)
    for step in range(4):
        x.copy_(torch.from_numpy(rng.standard_normal(tuple(x.shape)).astype(np.float32)))
        p = rng.integers(0, 40, (3, 2)).astype(np.int32)
        pos.copy_(torch.from_numpy(p))
        for c in caches:
            c.set_lengths([step + 1, 2 * step + 1])
        torch.cuda.synchronize()
        chain.launch()
        g.replay()
        a, k = args(2)
        rope.apply(*turn(2), axes=axes)
        caches[2].append(*a, **k)
        want = ref.turn(host(x)[:, :4 * dim].reshape(2, 4, dim), p, table, sections, "blocks", False, True)
        for i in range(3):
            close(host(qs[i]).reshape(want.shape), want)
            assert np.array_equal(host(y[i]), host(qs[i]))
            assert np.array_equal(host(caches[i].k), host(caches[2].k))
            assert np.array_equal(host(caches[i].k_scale), host(caches[2].k_scale))
