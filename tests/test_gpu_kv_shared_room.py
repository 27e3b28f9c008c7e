"""Attention behind a shared prefix in batches whose sequences differ much in new tokens, and
with row starts that fall: work-groups and states are those of the call's rows."""
import numpy as np
import pytest

from tests import kv_attend_reference as ref
from tests.gpu_util import dev, host
from tests.test_gpu_kv_shared import build, run
from tests.test_gpu_kvcache import check, note

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("seqs,long,at,heads,group,dim,prefix", [
    (64, 300, 0, 2, 7, 128, 1024), (64, 300, 63, 2, 7, 128, 1024), (20, 180, 7, 4, 4, 64, 1408), (12, 70, 5, 2, 16, 256, 1024)])
def test_one_long_piece(seqs, long, at, heads, group, dim, prefix, fmt):
    note(f"shared: one piece of {long} among {seqs}, heads of {dim} {fmt}")
    rng = np.random.default_rng(51)
    new = [1] * seqs
    new[at] = long
    if seqs > 20:
        new[30] = 0
    own = [n + 9 for n in new]
    both = build(rng, prefix, own, heads, dim, 32, fmt)
    lens, hq = [prefix + n if m else 0 for n, m in zip(own, new)], heads * group
    q = (2 * rng.standard_normal((sum(new), hq, dim))).astype(np.float32)
    want, tol = ref.attend(both.ref, q, lens, new, dim ** -0.5)
    both.call(lens, new)
    for f16 in (False, True):
        ws = both.gpu.attention_workspace(hq, len(q), long, shared=prefix)
        ws.fill_(255)
        check(run(both, q, new, hq, dim, f16, prefix, workspace=ws), want, tol, f16)


@pytest.mark.parametrize("new", [40, 400])
def test_ranges_that_overlap(new):
    """Three sequences of one list claim the same rows: each would write the same, and no more
    row blocks have places than the rows of the call can make. What is written is right."""
    import torch
    note(f"shared: ranges that overlap new={new}")
    rng = np.random.default_rng(52)
    prefix, hq, dim = 1024 + new // 64 * 64, 16, 64
    both = build(rng, prefix, [64] * 6, 4, dim, 64, "i8")
    t = both.ref.table
    t[:] = t[0]
    both.gpu.page_table.copy_(torch.from_numpy(t))
    q = rng.standard_normal((new, hq, dim)).astype(np.float32)
    want, tol = ref.attend(both.ref, q, [prefix + 40] + [0] * 5, [new] + [0] * 5, 0.125)
    both.call([prefix + 40] * 6, [0] * 6)
    both.gpu.use_cu_tokens(dev(np.array([0, new, 0, new, 0, new, 0], np.int32)))
    qt, out = dev(q), torch.full((new + 1, hq * dim), 7.0, device="cuda")
    ws = both.gpu.attention_workspace(hq, new, new, shared=prefix)
    guard = torch.full((ws.nbytes + 4096,), 90, dtype=torch.uint8, device="cuda")
    part = guard[:ws.nbytes]
    both.gpu.attend(qt.data_ptr(), hq * dim, hq, out.data_ptr(), hq * dim, new, new, scale=0.125, shared=prefix,
                    workspace=part)
    got = host(out)
    assert np.all(got[new] == 7) and np.all(host(guard[ws.nbytes:]) == 90)
    check(got[:new].reshape(want.shape), want, tol, False)


def test_one_workspace_for_every_batch():
    """Memory for the largest batch, at its exact size, does for smaller ones on each way; what
    lies behind it stays."""
    import torch
    note("shared: one workspace for every batch")
    rng = np.random.default_rng(53)
    seqs, prefix, heads, group, dim = 40, 1344, 4, 4, 64
    hq, own = heads * group, [60] * seqs
    both = build(rng, prefix, own, heads, dim, 64, "i8")
    n = both.gpu.attention_workspace(hq, seqs * 60, 60, shared=prefix).nbytes
    guard = torch.empty(n + 4096, dtype=torch.uint8, device="cuda")
    for new, shared in (([60] * seqs, prefix), ([1] * seqs, prefix), ([3] * seqs, 1300), ([1, 0, 60] + [0] * 37, 700),
                        ([7] * seqs, 64), ([1] * 20 + [0] * 20, prefix)):
        guard.fill_(90)
        lens = [prefix + 60 if m else 0 for m in new]
        q = (2 * rng.standard_normal((sum(new), hq, dim))).astype(np.float32)
        want, tol = ref.attend(both.ref, q, lens, new, dim ** -0.5)
        both.call(lens, new)
        check(run(both, q, new, hq, dim, False, shared, workspace=guard[:n]), want, tol, False)
        assert bool((guard[n:] == 90).all())
