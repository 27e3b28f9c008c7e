"""The norms around a block for prompts: the work-groups of many rows (4 a CU and more), a
wavefront a row to 1024 values and 256 threads to 4096, with and without whole quads; and
rows of 8193 to 16384 values, which 1024 threads hold. Bounds: tests/test_gpu_block_norm.py."""
import numpy as np
import pytest

from tests.gpu_util import dev, host
from tests.test_gpu_block_norm import check, inputs, note

pytestmark = pytest.mark.gpu

# hidden sizes, rows beside 4 a CU (None: few rows)
SIZES = [(260, 0), (896, 3), (1021, 1), (1024, 5), (1028, 0), (2049, 2), (3584, 1), (4096, 3), (4100, 0),
         (8193, None), (9001, None), (12000, None), (16383, None), (8193, 1)]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("hidden,more", SIZES)
def test_rows(hidden, more, f16):
    import torch
    from modgrad_amd.norm import BlockNorm
    rows = 3 if more is None else 4 * torch.cuda.get_device_properties(0).multi_processor_count + more
    note(f"norm of a prompt rows={rows} hidden={hidden} f16={f16}")
    gates = hidden % 3
    h, x, w1, w2, gate = inputs(rows, hidden, 11, gates=gates)
    n = BlockNorm(hidden, 1e-5, post_w=dev(w1), norm_w=dev(w2), gate=dev(gate[0]) if gates == 1 else None, h_scale=0.75,
                  x_scale=0.31)
    ht, xt, gt = dev(h), dev(x), dev(gate) if gates == 2 else None
    ho = torch.full((rows + 1, hidden), 7.0, device="cuda")
    y = torch.full((rows + 1, hidden), 7.0, device="cuda", dtype=torch.float16 if f16 else torch.float32)
    n.apply(ht.data_ptr(), xt.data_ptr(), rows, h_out=ho.data_ptr(), y=y.data_ptr(), y_f16=f16,
            gate=gt.data_ptr() if gates == 2 else 0)
    got, yg = host(ho), host(y)
    assert np.all(got[rows] == 7) and np.all(yg[rows] == 7) and np.array_equal(host(ht), h)
    check(h, x, w1, gate, w2, 0.75, 0.31, 1e-5, got[:rows], yg[:rows])


@pytest.mark.parametrize("hidden", [896, 3584])
@pytest.mark.parametrize("parts", ["x", "post", "pre", "y alone"])
def test_parts(parts, hidden):
    """Each norm and each output left out, in place, rows apart."""
    import torch
    from modgrad_amd.norm import BlockNorm
    rows = 4 * torch.cuda.get_device_properties(0).multi_processor_count + 2
    note(f"norm of a prompt {parts} hidden={hidden}")
    h, x, w1, w2, _ = inputs(rows, hidden, 12)
    post, pre = parts == "post", parts in ("pre", "y alone")
    n = BlockNorm(hidden, 1e-6, post_w=dev(w1) if post else None, norm_w=dev(w2) if pre else None)
    wide = np.full((rows, hidden + 3), 9.0, np.float32)
    wide[:, :hidden] = h
    ht, xt, y = dev(wide), dev(x), torch.full((rows, hidden + 1), 7.0, device="cuda")
    n.apply(ht.data_ptr(), 0 if parts == "pre" else xt.data_ptr(), rows, h_out=0 if parts == "y alone" else None,
            y=y.data_ptr() if pre else 0, h_stride=hidden + 3, y_stride=hidden + 1)
    got, yg = host(ht), host(y)
    assert np.all(got[:, hidden:] == 9) and np.all(yg[:, hidden:] == 7)
    if parts == "y alone":
        assert np.array_equal(got, wide)
    if not pre:
        assert np.all(yg == 7)
    check(h, None if parts == "pre" else x, w1 if post else None, None, w2, 1.0, 1.0, 1e-6,
          None if parts == "y alone" else got[:, :hidden], yg[:, :hidden] if pre else None)
