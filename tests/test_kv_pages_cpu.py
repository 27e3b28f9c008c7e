"""Pages of a cache that hands them out: shared by several slots, given back from the middle
of one, free again when the last slot leaves them (host logic, no GPU)."""
import contextlib
import random

import pytest
import torch

from modgrad_amd import kvcache
from modgrad_amd.kvcache import KvCache
from modgrad_amd.q4k import BackendError

PAGE = 16


@pytest.fixture(autouse=True)
def without_a_gpu(monkeypatch):
    monkeypatch.setattr(kvcache, "_torch", lambda: torch)
    monkeypatch.setattr(kvcache, "_stream", lambda stream: contextlib.nullcontext())


def cache(pages=20, seqs=4, most=10):
    z = lambda *s, dtype=torch.uint8: torch.zeros(*s, dtype=dtype)  # noqa: E731
    c = KvCache.wrap(z(pages, 1, PAGE, 64), z(pages, 1, 64, PAGE), z(pages, 1, dtype=torch.float32),
                     z(pages, 1, dtype=torch.float32), torch.full((seqs, most), -1, dtype=torch.int32),
                     z(seqs, dtype=torch.int32))
    c._free = list(range(pages - 1, -1, -1))  # as KvCache.new leaves it
    return c


def rows(c):
    return c.page_table.tolist()


def consistent(c):
    """Every page is free or in some slots' lists, which the table holds."""
    used = [p for held in c._held for p in held if p is not None]
    assert sorted(c._free + list(set(used))) == list(range(c.n_pages))
    assert [used.count(p) for p in range(c.n_pages)] == c._users
    for b, held in enumerate(c._held):
        assert rows(c)[b] == [-1 if p is None else p for p in held] + [-1] * (c.max_pages - len(held))


def test_shared_pages_outlive_their_first_slot():
    c = cache()
    c.set_lengths([70, 0, 0, 0], [70, 0, 0, 0])
    c.share(1, 0, 64)
    c.share(2, 1, 32)
    common = rows(c)[0][:4]
    assert rows(c)[1][:5] == common + [-1] and rows(c)[2][:3] == common[:2] + [-1]
    consistent(c)
    c.set_lengths([71, 65, 33, 0], [1, 1, 1, 0])
    consistent(c)
    assert rows(c)[1][:4] == common and rows(c)[1][4] not in rows(c)[0]
    free = len(c._free)
    c.release(0)
    consistent(c)
    assert len(c._free) == free + 1 and not set(common) & set(c._free)  # only its own page is free
    c.reserve(3, 100)
    assert not set(rows(c)[3]) & set(common)
    c.release(1)
    assert set(common[2:]) <= set(c._free) and not set(common[:2]) & set(c._free)
    c.release(2)
    c.release(3)
    consistent(c)
    assert len(c._free) == c.n_pages


def test_given_back():
    c = cache()
    c.set_lengths([150, 0, 0, 0], [150, 0, 0, 0])
    was = rows(c)[0]
    c.give_back(0, 5, 100)  # pages 1 .. 5 lie in it
    assert rows(c)[0] == was[:1] + [-1] * 5 + was[6:]
    consistent(c)
    c.give_back(0, 5, 100)  # nothing is given back twice
    c.give_back(0, 100, 100)
    c.give_back(0, 33, 40)
    consistent(c)
    c.set_lengths([151, 0, 0, 0], [1, 0, 0, 0])
    c.give_back(0, 96, 2 ** 40)
    consistent(c)
    assert len(c._free) == c.n_pages - 1
    c.release(0)
    assert len(c._free) == c.n_pages and rows(c)[0] == [-1] * 10


def test_new_tokens_in_pages_of_others():
    c = cache()
    c.set_lengths([64, 0, 0, 0], [64, 0, 0, 0])
    c.share(1, 0, 64)
    before = (rows(c), list(c._free))
    for lengths, new in (([64, 64, 0, 0], [0, 1, 0, 0]), ([64, 64, 0, 0], [1, 0, 0, 0]), ([64, 64, 0, 0], None),
                         ([64, 66, 0, 0], [0, 3, 0, 0])):
        with pytest.raises(BackendError):
            c.set_lengths(lengths, new)
    assert (rows(c), c._free) == before
    c.set_lengths([50, 64, 0, 0], [0, 0, 0, 0])  # none new
    c.set_lengths([65, 66, 0, 0], [1, 2, 0, 0])
    c.release(1)
    c.set_lengths([65, 0, 0, 0], [5, 0, 0, 0])   # now its own again
    c.give_back(0, 0, 32)
    with pytest.raises(BackendError):
        c.set_lengths([32, 0, 0, 0], [1, 0, 0, 0])
    c.set_lengths([66, 0, 0, 0], [1, 0, 0, 0])
    consistent(c)


def test_refuses():
    c = cache()
    c.reserve(0, 64)
    c.reserve(1, 16)
    for bad in ((2, 0, 60), (2, 0, 80), (2, 0, -16), (2, 2, 16), (1, 0, 16), (4, 0, 16), (-1, 0, 16), (2, 4, 16),
                (2, -1, 16), (3, 2, 16)):
        with pytest.raises(BackendError):
            c.share(*bad)
    c.give_back(0, 16, 32)
    with pytest.raises(BackendError):
        c.share(2, 0, 48)  # a page of it was given back
    for bad in ((4, 0, 16), (-1, 0, 16), (0, -1, 16), (0, 32, 16)):
        with pytest.raises(BackendError):
            c.give_back(*bad)
    c.share(2, 0, 0)
    consistent(c)
    c._free = None  # of the caller's tables
    for f in (lambda: c.share(2, 0, 16), lambda: c.give_back(0, 0, 16), lambda: c.release(0), lambda: c.reserve(0, 1)):
        with pytest.raises(BackendError):
            f()


def test_any_order():
    rng = random.Random(3)
    c = cache(pages=30, seqs=5, most=8)
    for _ in range(3000):
        a, b, n = rng.randrange(5), rng.randrange(5), rng.randrange(0, 129)
        try:
            rng.choice((lambda: c.reserve(a, n), lambda: c.share(a, b, n // 16 * 16), lambda: c.give_back(a, n // 3, n),
                        lambda: c.release(a)))()
        except BackendError:
            pass
        consistent(c)
