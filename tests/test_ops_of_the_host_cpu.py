"""Tensors of the host make no op of a recorded chain: its kernels would read host memory."""
import pytest
import torch

from modgrad_amd import kvcache, norm
from modgrad_amd.kvcache import KvCache, RopeAxes, RopeTable
from modgrad_amd.norm import BlockNorm
from modgrad_amd.q4k import BackendError

FAKE = 0x10000


@pytest.fixture(autouse=True)
def without_a_gpu(monkeypatch):
    """The package's torch asks for a GPU; what is looked at here needs none."""
    for module in (kvcache, norm):
        monkeypatch.setattr(module, "_torch", lambda: torch)


def test_block_norm():
    w = torch.ones(64)
    for weights in (dict(post_w=w), dict(norm_w=w), dict(gate=w)):
        with pytest.raises(BackendError):
            BlockNorm(64, 1e-6, **weights).op(FAKE, FAKE, 1)
    assert BlockNorm(64, 1e-6).op(FAKE, FAKE, 1).op  # nothing of the object's to look at


def test_rope_table():
    table = RopeTable.wrap(torch.zeros(4, 8, 2), True)
    for kw in ({}, dict(axes=RopeAxes([4, 4]))):
        with pytest.raises(BackendError):
            table.op(FAKE, FAKE, FAKE, 1, 1, 64, **kw)


def test_cache():
    z = lambda *s, dtype=torch.uint8: torch.zeros(*s, dtype=dtype)  # noqa: E731
    c = KvCache.wrap(z(4, 2, 16, 64), z(4, 2, 64, 16), z(4, 2, dtype=torch.float32), z(4, 2, dtype=torch.float32),
                     z(3, 2, dtype=torch.int32), z(3, dtype=torch.int32))
    for kw in ({}, dict(axes=RopeAxes([4, 4]), pos=FAKE)):
        with pytest.raises(BackendError):
            c.op_append(FAKE, FAKE, 128, 3, 1, **kw)
    for kw in ({}, dict(window=5, sinks=5), dict(shared=64)):
        with pytest.raises(BackendError):
            c.op_attend(FAKE, 256, 4, FAKE, 256, 3, 1, z(1024), **kw)
