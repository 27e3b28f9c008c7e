"""Attention behind a shared prefix on each of its ways, asserted, with everything in one
batch: rows ahead of the first sequence and behind the last, an idle slot, sequences that
have only begun, holes in the common pages. Against tests/kv_attend_reference.py."""
import ctypes

import numpy as np
import pytest

from modgrad_amd import _lib
from tests import kv_attend_reference as ref
from tests.gpu_util import dev, host
from tests.test_gpu_kv_shared import build
from tests.test_gpu_kvcache import check, note

pytestmark = pytest.mark.gpu

FEW, PARTS, RUNS = _lib.SHARED_FEW, _lib.SHARED_PARTS, _lib.SHARED_RUNS
CASES = {
    # way, prefix, sequences, new tokens up to, kv heads, group, dim, page, softcap
    "few rows": (FEW, 1024, 20, 2, 4, 3, 64, 16, 0),
    "few rows, heads of 256": (FEW, 1024, 12, 3, 4, 5, 256, 32, 30.0),
    "single tokens, heads of 256": (PARTS, 704, 64, 1, 2, 8, 256, 32, 0),
    "several tokens": (PARTS, 1024, 40, 6, 4, 4, 96, 32, 0),
    "prompts": (PARTS, 1344, 5, 150, 4, 3, 64, 64, 50.0),
    "runs, few tokens each": (RUNS, 2240, 68, 3, 8, 16, 64, 32, 0),
    "runs, heads of 64": (RUNS, 1920, 11, 58, 8, 5, 64, 64, 30.0),
    "runs, heads of 128": (RUNS, 1920, 5, 43, 8, 16, 128, 128, 0),
    "runs, heads of 256": (RUNS, 1920, 9, 23, 4, 16, 256, 32, 0),
}


def layout(name):
    """(own tokens, lengths, new tokens, rows on either side that are nobody's)."""
    _, prefix, seqs, most, *_ = CASES[name]
    rng = np.random.default_rng(sum(map(ord, name)))
    new = [int(v) for v in rng.integers(max(1, (9 * most) // 10), most + 1, seqs)]
    new[0] = most
    own = [n + int(v) for n, v in zip(new, rng.integers(0, 70, seqs))]
    lens = [prefix + n for n in own]
    lens[-1], new[-1] = 0, 0                         # idle
    if seqs > 4:
        lens[1] = max(new[1], prefix // 3)           # on its way through the prefix
        lens[2] = new[2]                             # at its begin: sees no whole tile ahead
    return own, lens, new, 5


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("name", CASES)
def test_ways(name, f16, fmt):
    import torch
    way, prefix, seqs, _, heads, group, dim, page, cap = CASES[name]
    note(f"shared ways {name} {fmt} f16={f16}")
    rng = np.random.default_rng(7)
    own, lens, new, ahead = layout(name)
    both = build(rng, prefix, own, heads, dim, page, fmt)
    t = both.ref.table
    t[:, 1], t[:, prefix // page - 1] = -1, 10 ** 6  # holes in every list
    both.gpu.page_table.copy_(torch.from_numpy(t))
    both.call(lens, new)
    cu = ahead + np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    both.gpu.use_cu_tokens(dev(cu.astype(np.int32)))
    rows, hq = sum(new) + 2 * ahead, heads * group
    plan = _lib.KvSharedPlan()
    _lib.check("plan", _lib.load().mgq_kv_attention_shared_plan(ctypes.byref(both.gpu.desc), hq, int(f16), rows, max(new),
                                                                prefix, ctypes.byref(plan)))
    assert plan.way == way
    q = (2 * rng.standard_normal((rows, hq, dim))).astype(np.float32)
    q[:ahead] = np.nan
    q[rows - ahead:] = np.inf
    out = torch.full((rows, hq * dim), 7.0, device="cuda", dtype=torch.float16 if f16 else torch.float32)
    qt = dev(q)
    ws = both.gpu.attention_workspace(hq, rows, max(new), shared=prefix)
    ends = []
    for byte in (0, 255):  # what the workspace holds does not matter
        ws.fill_(byte)
        both.gpu.attend(qt.data_ptr(), hq * dim, hq, out.data_ptr(), hq * dim, rows, max(new), scale=dim ** -0.5,
                        softcap=cap, out_f16=f16, shared=prefix, workspace=ws)
        ends.append(host(out).reshape(rows, hq, dim))
    got = ends[0]
    assert np.array_equal(got, ends[1])
    assert np.all(got[:ahead] == 7) and np.all(got[rows - ahead:] == 7)
    mine = slice(ahead, rows - ahead)
    want, tol = ref.attend(both.ref, q[mine], lens, new, dim ** -0.5, cap)
    check(got[mine], want, tol, f16)
