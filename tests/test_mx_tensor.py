"""MXTensor and the Python checks of the microscaled (MX) operators where nothing is launched (no GPU)."""
import pytest
import torch

from ditserve_amd import mx


def random_matrix(rows, cols, fmt):
    m = mx.MXTensor.empty(rows, cols, "cpu", fmt)
    g = torch.Generator().manual_seed(rows + cols)
    m.data.view(torch.uint8).copy_(torch.randint(0, 127 if fmt == "fp8" else 256, m.data.shape, generator=g))
    m.scales.view(torch.uint8).copy_(torch.randint(100, 150, m.scales.shape, generator=g))
    return m


def e4m3(byte):
    e, f = byte >> 3 & 15, byte & 7
    return (-1) ** (byte >> 7) * (f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10))


def e2m1(code):
    return (-1) ** (code >> 3) * [0, 0.5, 1, 1.5, 2, 3, 4, 6][code & 7]


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("rows,cols", [(0, 32), (0, 1536), (1, 32), (3, 160), (2, 544)])
def test_dequantize(rows, cols, fmt):
    """Value by value from the bytes, also of a matrix without rows."""
    m = random_matrix(rows, cols, fmt)
    got = m.dequantize()
    assert got.shape == (rows, cols) and got.dtype == torch.float32
    data, scales = m.data.view(torch.uint8).tolist(), m.scales.view(torch.uint8).tolist()
    for r in range(rows):
        for c in range(cols):
            v = e4m3(data[r][c]) if fmt == "fp8" else e2m1(data[r][c // 2] >> 4 * (c % 2) & 15)
            b = c // 32
            assert got[r, c].item() == v * 2.0 ** (scales[r][b // 16 * 16 + b % 4 * 4 + b % 16 // 4] - 127)
