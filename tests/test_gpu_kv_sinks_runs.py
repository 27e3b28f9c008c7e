"""First tokens behind a window where the tiles of all rows are cut into equal runs, one for
each resident work-group (16 tiles a group and more): served batches. Against
tests/kv_attend_reference.py."""
import numpy as np
import pytest

from tests import kv_attend_reference as ref
from tests.test_gpu_kv_sinks import run
from tests.test_gpu_kvcache import Both, check, note

pytestmark = pytest.mark.gpu

CASES = {
    # sequences, tokens, new tokens, kv heads, group, dim, page, softcap, window, sinks
    "single tokens": (70, 2300, 1, 4, 3, 64, 64, 0, 2000, 70),
    "three tokens each": (50, 2100, 3, 2, 16, 64, 32, 30.0, 1800, 5),
    "heads of 128": (35, 2400, 1, 8, 2, 128, 128, 0, 2050, 64),
    "heads of 256": (20, 1900, 2, 4, 12, 256, 64, 0, 1700, 100),
}


def written(both, rng):
    """Every page as if tokens had been appended to all of it."""
    import torch
    for bytes_, scales, t, s in ((both.ref.k, both.ref.ks, both.k, both.ks), (both.ref.v, both.ref.vs, both.v, both.vs)):
        if both.ref.fmt == "i8":
            x = rng.integers(-127, 128, bytes_.shape, dtype=np.int8).view(np.uint8)
            at = rng.uniform(0.01, 0.03, scales.shape)
        else:  # below 2 either way: codes 0x00 .. 0x3f
            x = (rng.integers(0, 0x40, bytes_.shape, dtype=np.uint8) | rng.integers(0, 2, bytes_.shape, dtype=np.uint8) << 7)
            at = rng.uniform(0.5, 1.5, scales.shape)
        bytes_[:], scales[:] = x, at.astype(np.float32)
        t.copy_(torch.from_numpy(bytes_))
        s.copy_(torch.from_numpy(scales))


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("name", CASES)
def test_runs(name, fmt):
    seqs, most, m, heads, group, dim, page, cap, window, sinks = CASES[name]
    f16 = (fmt == "i8") == (dim == 64)
    note(f"sinks in runs {name} {fmt} f16={f16}")
    rng = np.random.default_rng(sum(map(ord, name)))
    both = Both(rng, seqs, -(-most // page), heads, dim, page, fmt)
    written(both, rng)
    lens = [int(n) for n in rng.integers(most - 64, most + 1, seqs)]
    lens[3] = m                      # just begun
    lens[5] = window + sinks // 2    # the window meets the first tokens
    new = [m] * seqs
    # tiles that the rows of a kv head go through, 16 query rows each
    first = [max(0, n - m - window + 1) // 64 for n in lens]
    tiles = [-(-n // 64) - f + min(f, -(-sinks // 64)) for n, f in zip(lens, first)]
    slots = 256 if dim == 256 else 512
    assert sum(tiles) * heads * -(-m * group // 16) >= 16 * slots and m * group <= (32 if dim == 256 else 48)
    hq = heads * group
    q = (2 * rng.standard_normal((seqs * m, hq, dim))).astype(np.float32)
    want, tol = ref.attend(both.ref, q, lens, new, dim ** -0.5, cap, window, sinks)
    both.call(lens, new, m == 1)
    got = run(both, q, lens, new, hq, dim, f16, window, sinks, cap)
    check(got, want, tol, f16)
    both.call(lens, new)
    assert np.array_equal(run(both, q, lens, new, hq, dim, f16, window, sinks, cap), got)  # and by row starts
