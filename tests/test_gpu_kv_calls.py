"""Calls on the 8-bit cache at the edges of what its documentation allows."""
import numpy as np
import pytest

from tests.gpu_util import dev, host
from tests.test_gpu_kvcache import Both, note

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 3])
@pytest.mark.parametrize("place", [False, True])
def test_append_copies_the_queries_of_idle_slots(new, place):
    """Without a rotary table q is copied as it is, at positions before the first
    token too (an idle slot, more rows than tokens)."""
    import torch
    note(f"append without a table, idle slots new={new} in place={place}")
    rng = np.random.default_rng(new)
    both = Both(rng, 4, 2, 1, 64, 16, "i8")
    lens, rows = [0, 5, new - 1, 32], 4 * new
    both.call(lens, [new] * 4, new == 1)
    kv = torch.randn(rows, 128, device="cuda")
    q = rng.standard_normal((rows, 2 * 64)).astype(np.float32)
    qt = dev(q)
    out = qt if place else torch.full((rows, 128), 7.0, device="cuda")
    both.gpu.append(kv.data_ptr(), kv.data_ptr() + 256, 128, rows, new, q=qt.data_ptr(), q_stride=128,
                    q_out=out.data_ptr(), q_out_stride=128, n_q_heads=2)
    assert np.array_equal(host(out), q)
