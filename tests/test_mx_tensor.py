"""MXTensor and the Python checks of the microscaled (MX) operators where nothing is launched (no GPU)."""
import pytest
import torch

from ditserve_amd import mx, ops


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


@pytest.fixture
def host(monkeypatch):
    """The Python checks on CPU tensors: the device check is left out, and a launch is an error."""
    def check(t, name, dtype=None, dims=None):
        if not isinstance(t, torch.Tensor) or (dtype is not None and t.dtype != dtype) or (dims is not None and t.dim() != dims):
            raise ValueError(name)

    def launched(*args):
        raise AssertionError("launched")
    monkeypatch.setattr(mx, "_check", check)
    monkeypatch.setattr(ops, "_check", check)
    monkeypatch.setattr(mx, "_call", launched)


@pytest.mark.parametrize("out", [[1.0], "out", 3, (torch.zeros(1), torch.zeros(1))])
def test_outputs_that_are_no_tensors_are_refused(host, out):
    x, v = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros(64, dtype=torch.bfloat16)
    q, w, w4 = (mx.MXTensor.empty(n, 64, "cpu", f) for n, f in ((4, "fp8"), (32, "fp8"), (32, "fp4")))
    for call in (lambda: mx.quantize(x, out=out), lambda: mx.norm(x, out=out), lambda: mx.norm(x, x, residual_out=out),
                 lambda: mx.linear(q, w, out=out), lambda: mx.linear(q, w, out=out, out_fmt="fp8"),
                 lambda: mx.matvec(x, w4, out=out), lambda: mx.matvec(v, w4, out=out),
                 lambda: mx.matvec(v, w4, epilogue="res", residual=out),
                 lambda: mx.linear(q, w, epilogue="res", residual=out)):
        with pytest.raises(ValueError):
            call()


def test_outputs_of_the_other_kind_are_refused(host):
    q, w, w4 = (mx.MXTensor.empty(n, 64, "cpu", f) for n, f in ((4, "fp8"), (32, "fp8"), (32, "fp4")))
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    for call in (lambda: mx.linear(q, w, out=mx.MXTensor.empty(4, 32, "cpu")),
                 lambda: mx.linear(q, w, out_fmt="fp8", out=torch.zeros((4, 32), dtype=torch.bfloat16)),
                 lambda: mx.matvec(x, w4, out=mx.MXTensor.empty(4, 32, "cpu")),
                 lambda: mx.matvec(x[0], w4, out=mx.MXTensor.empty(4, 32, "cpu"))):
        with pytest.raises(ValueError):
            call()


def test_outputs_beside_their_operands_in_one_buffer(host):
    """Column ranges of one buffer share an extent but no byte: they are no overlap."""
    wide = torch.zeros((9, 320), dtype=torch.bfloat16)
    left, right, middle = wide[:8, :64], wide[:8, 64:128], wide[:8, 32:96]
    q, w, w4 = (mx.MXTensor.empty(n, 64, "cpu", f) for n, f in ((8, "fp8"), (32, "fp8"), (32, "fp4")))
    for call in (lambda: mx.norm(left, right, residual_out=wide[:8, 128:192]),
                 lambda: mx.norm(left, right, residual_out=wide[1:, 128:192]),
                 lambda: mx.norm(left, left, residual_out=right),
                 lambda: mx.linear(q, w, epilogue="res", residual=wide[1:, :32], out=wide[:8, 32:64]),
                 lambda: mx.linear(q, w, epilogue="res", residual=wide[:8, 32:64], out=wide[1:, :32]),
                 lambda: mx.matvec(left, w4, out=wide[1:, 288:]), lambda: mx.matvec(wide[:8, 256:], w4, out=wide[:8, :32])):
        with pytest.raises(AssertionError, match="launched"):
            call()
    # shared columns overlap, also across the end of a line and with another stride
    flat = wide.view(-1)
    across = flat[288:288 + 8 * 320].view(8, 320)[:, :64]  # columns 288 .. 319 and 0 .. 31 of the next row
    for call in (lambda: mx.norm(left, right, residual_out=middle), lambda: mx.norm(left, right, residual_out=wide[1:, :64]),
                 lambda: mx.matvec(left, w4, out=wide[:8, 56:88]), lambda: mx.matvec(across, w4, out=wide[:8, :32]),
                 lambda: mx.matvec(across, w4, out=wide[:8, 288:]),
                 lambda: mx.matvec(left[:4], w4, out=torch.as_strided(wide, (4, 32), (640, 1), 32))):
        with pytest.raises(ValueError, match="overlaps"):
            call()
