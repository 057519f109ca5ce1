"""The microscaled (MX) operators at sizes and shapes where launches, tiles and strides change."""
import pytest
import torch

from ditserve_amd import mx

pytestmark = pytest.mark.gpu
DEV = "cuda"


def raw(m):
    return m.data.view(torch.uint8), m.scales.view(torch.uint8)


@pytest.mark.parametrize("op,cols", [("quantize", 32), ("quantize", 544), ("norm", 32)])
def test_more_rows_than_one_launch_dimension_holds(op, cols):
    """From 2^26 waves on a launch has 2^32 threads, which its first dimension does not hold: every row is
    written all the same.  Rows repeat with a period, so each is compared with its own of a small call."""
    rows, period = (1 << 26) // ((cols + 511) // 512 if op == "quantize" else 1) + 5, 4093
    g = torch.Generator(device=DEV).manual_seed(cols)
    few = torch.randn((period, cols), generator=g, device=DEV).to(torch.bfloat16)
    call = mx.quantize if op == "quantize" else mx.norm
    want = raw(call(few))
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device=DEV)
    whole = rows // period * period
    x[:whole].view(-1, period, cols).copy_(few)
    x[whole:].copy_(few[:rows - whole])
    out = mx.MXTensor.empty(rows, cols, DEV)
    for t in raw(out):
        t.fill_(0xAA)
    call(x, out=out)
    for got, ref in zip(raw(out), want):
        parts = got[:whole].view(-1, period, got.shape[1])
        for i in range(0, parts.shape[0], 1024):
            assert (parts[i:i + 1024] == ref).all(), i
        assert torch.equal(got[whole:], ref[:rows - whole])
