"""Attention behind a shared prefix launches and asks for no more than the call's rows can
need, however ragged the batch (host only, no GPU)."""
import ctypes

import pytest

from modgrad_amd import _lib
from tests.test_kv_shared_plan_cpu import ask, cache_of
from tests.test_kvcache_cpu import INVALID

LAUNCH = (2 ** 32 - 1) // 256  # work-groups of 256 threads that one launch counts


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("fmt", [0, 1])
def test_launches_are_of_the_rows(fmt, kind):
    """One piece of 2048 tokens among 63 single tokens: 116 row blocks of 128 and 63 that are
    not full at most, of 4 heads; not 64 times those of the piece."""
    c = cache_of(64, 4, 128, 64, fmt, 400)
    p = ask(c, 28, 2111, 2048, 12000, kind)
    assert p.way != _lib.SHARED_PLAIN
    pairs = (2111 * 7 // 128 + 64) * 4
    assert p.own_groups <= pairs and p.join_groups <= 128 * pairs
    even = ask(c, 28, 64 * 2048, 2048, 12000, kind)  # all of them as long
    assert even.own_groups == 64 * 112 * 4


@pytest.mark.parametrize("seqs,heads,hq,n,new,shared", [
    (256, 8, 64, 8447, 8192, 12032), (256, 8, 64, 256 * 8192, 8192, 12032), (256, 8, 64, 256 * 4096, 4096, 20000),
    (1024, 8, 128, 1024 * 900, 900, 200000), (1 << 18, 8, 8, 1 << 18, 1, 20000), (1 << 16, 16, 256, 1 << 16, 1, 64000),
    (1 << 20, 1, 16, 1 << 20, 1, 8000), (512, 64, 64, 512 * 700, 700, 4096)])
def test_launches_are_counted(seqs, heads, hq, n, new, shared):
    for dim in (64, 128, 256):
        for kind in (0, 1):
            c = cache_of(seqs, heads, dim, 64, 0, -(-(shared + new) // 64) + 1)
            p = ask(c, hq, n, new, shared, kind)
            if p is not None and p.way != _lib.SHARED_PLAIN:
                assert 0 < p.join_groups <= LAUNCH and 0 < p.own_groups <= LAUNCH


def room(c, hq, n, new, shared):
    return _lib.load().mgq_kv_attention_shared_workspace_bytes(ctypes.byref(c), hq, n, new, shared)


def test_room_is_of_the_rows():
    """The same batch: own states of its row blocks (47.7 MB) and the prefix's (62 MB at two
    for each of 116 blocks), not the 1.9 GB of 64 such pieces."""
    c = cache_of(64, 4, 128, 64, 0, 400)
    assert room(c, 28, 2111, 2048, 12000) < 2.5e8
    # a sequence's last block is seldom full: no less than the rows take
    assert room(c, 28, 64 * 2048, 2048, 12000) >= 2 * 64 * 2048 * 28 * 130 * 4
    c = cache_of(256, 8, 128, 64, 0, 400)
    assert room(c, 64, 8447, 8192, 12032) < 1e9


def test_one_state_a_part():
    """64 prompts of 2048 tokens: a state of each row block for the prefix, one for the own
    tiles, 1.9 GB each."""
    c = cache_of(64, 4, 128, 64, 0, 400)
    states = 64 * 2048 * 28 * 130 * 4
    assert ask(c, 28, 64 * 2048, 2048, 12000).way == _lib.SHARED_PARTS
    assert 2 * states <= room(c, 28, 64 * 2048, 2048, 12000) < 2.02 * states


def needed(p, heads, dim, wide):
    """States that a call with this plan has, at least."""
    cuts = -(-p.tiles // p.run) if p.run else 0
    prefix = {_lib.SHARED_PLAIN: 0, _lib.SHARED_FEW: 16 * p.blocks * cuts, _lib.SHARED_PARTS: 128 * p.blocks * cuts,
              _lib.SHARED_RUNS: 256 * -(-p.blocks * p.tiles // max(1, p.run))}[p.way]
    own = 128 * p.own_groups if wide and p.join_groups else 0
    return (prefix * heads + own) * (dim + 2) * 4


def test_room_does_not_fall():
    """Memory for a batch does for every smaller one: fewer tokens, new tokens, sequences or
    shared tokens; and is enough for the states of the plan."""
    import random
    rng = random.Random(5)
    ways = set()
    for _ in range(6000):
        dim, fmt = rng.choice((64, 96, 128, 256)), rng.randrange(2)
        heads, group = rng.choice((1, 2, 4, 8, 16)), rng.choice((1, 2, 3, 7, 8, 16))
        size = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))  # noqa: E731
        seqs, new, shared = size(1, 300), size(1, 3000), size(1, 40000)
        n = max(new, rng.randrange(seqs, seqs * new + 1))
        low = lambda v: rng.choice((v, v, rng.randrange(1, v + 1), max(1, v - 1)))  # noqa: E731
        seqs2, new2, shared2 = low(seqs), low(new), low(shared)
        n2 = max(new2, low(n))
        large, small = (cache_of(b, heads, dim, 64, fmt, 40000 // 64 + 40) for b in (seqs, seqs2))
        hq = heads * group
        a, b = room(large, hq, n, new, shared), room(small, hq, n2, new2, shared2)
        assert 0 < b <= a, ((seqs, n, new, shared), (seqs2, n2, new2, shared2), heads, group, dim, fmt)
        plain = _lib.load().mgq_kv_attention_workspace_bytes(ctypes.byref(large), hq, new)
        for kind in (0, 1):
            p = ask(large, hq, n, new, shared, kind)
            ways.add(p.way)
            assert a >= plain and a >= needed(p, heads, dim, new * group > (32 if dim == 256 else 48))
    assert ways == {0, 1, 2, 3}


@pytest.mark.parametrize("way", ["plain", "sinks", "shared"])
def test_joins_that_no_launch_counts(way):
    """2^20 sequences of 16 rows: refused before the first of two launches, but where every
    row sees at most 8 tiles and none is joined."""
    from tests.test_kv_shared_cpu import FAKE
    L = _lib.load()

    def made(seqs, max_pages, window=0):
        c = cache_of(seqs, 1, 64, 64, 0, max_pages)
        c.cu_tokens = None
        args = _lib.KvAttentionArgs(c, FAKE, FAKE, FAKE, 1 << 45, 1024, 1024, 16, 0, seqs, 1, window, 0.1, 0.0)
        op = {"plain": lambda: args, "sinks": lambda: _lib.KvAttentionSinksArgs(args, 4),
              "shared": lambda: _lib.KvAttentionSharedArgs(args, 640)}[way]()
        kind = {"plain": _lib.OP_KV_ATTENTION, "sinks": _lib.OP_KV_ATTENTION_SINKS,
                "shared": _lib.OP_KV_ATTENTION_SHARED}[way]
        d, chain = _lib.OpDesc(op=kind, w=ctypes.addressof(op)), ctypes.c_void_p()
        code = L.mgq_chain_create_ops(ctypes.byref(d), 1, ctypes.byref(chain))
        if chain.value:  # recorded, never launched; without a device it is not even that
            L.mgq_chain_destroy(chain)
        return code
    assert made(1 << 20, 100) == INVALID
    fits = [made((1 << 20) - 1, 100), made(1 << 20, 8)]
    if way == "sinks":
        assert made(1 << 20, 100, 2000) == INVALID
        fits.append(made(1 << 20, 100, 300))  # 300 and 4: never more than 8 tiles
    assert INVALID not in fits
