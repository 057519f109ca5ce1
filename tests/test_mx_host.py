"""Refusals of the microscaled (MX) entry points: on the host, before any launch (no GPU)."""
import pytest
import torch

from ditserve_amd import _lib, mx, ops

if not _lib.LIB_PATH.exists():
    pytest.skip("libditk.so not built (run python -m ditserve_amd.build)", allow_module_level=True)

A, B, C, D, E, F, G, H = (0x10000 * i for i in range(1, 9))  # addresses only: nothing is launched


def refused(name, args, word):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == 1
    assert word in lib.ditk_last_error().decode(), lib.ditk_last_error()


QUANT = dict(x=A, ldx=96, data=B, ldd=128, scales=C, lds=16, T=4, K=96, fmt=0, stream=None)
NORM = dict(x=A, ldx=96, res=None, ldr=0, h=None, ldh=0, data=B, ldd=128, scales=C, lds=16, T=4, D=96, cu=None, nseg=0,
            shift=None, scale=None, stride=0, w=None, b=None, eps=1e-6, kind=1, stream=None)
GEMM = dict(A=A, lda=128, As=B, ldas=16, W=C, ldw=128, Ws=D, ldws=16, bias=None, C=E, ldc=64, Cs=None, ldcs=0, M=4, N=64,
            K=96, epi=0, out=0, R=None, ldr=0, gate=None, gs=0, cu=None, nseg=0, stream=None)
MV = dict(x=A, ldx=96, W=B, ldw=64, Ws=C, ldws=16, bias=None, C=E, ldc=64, M=4, N=64, K=96, epi=0, R=None, ldr=0,
          stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(x=None), "rows"), (dict(T=-1), "rows"), (dict(fmt=2), "format"), (dict(K=40), "blocks of 32"),
    (dict(K=0), "blocks"), (dict(ldd=96), "padding"), (dict(ldd=136), "16-byte strides"), (dict(lds=8), "padding"),
    (dict(K=544, ldx=544, ldd=640), "padding"), (dict(x=A + 2), "aligned"), (dict(ldx=92), "aligned"),
    (dict(ldx=88), "aligned"), (dict(data=B + 8), "aligned"), (dict(scales=None), "null")])
def test_quantize_refuses(change, word):
    refused("ditk_mx_quantize", tuple({**QUANT, **change}.values()), word)


@pytest.mark.parametrize("change,word", [
    (dict(x=None), "rows"), (dict(D=6176, ldx=6176, ldd=6272, lds=208), "6144"), (dict(kind=2), "norm"),
    (dict(res=D, ldr=96), "together"), (dict(h=D, ldh=96), "together"), (dict(res=D, h=E, ldr=96, ldh=64), "aligned"),
    (dict(shift=D), "together"), (dict(shift=D, scale=E, stride=96), "modulation"),
    (dict(shift=D, scale=E, stride=98, cu=F, nseg=1), "modulation"), (dict(w=D + 4), "aligned"), (dict(D=100), "blocks")])
def test_norm_refuses(change, word):
    refused("ditk_mx_norm", tuple({**NORM, **change}.values()), word)


@pytest.mark.parametrize("change,word", [
    (dict(W=None), "null"), (dict(A=None), "null"), (dict(M=-1), "shape"), (dict(N=0), "shape"), (dict(K=100), "K=100"),
    (dict(N=60), "N=60"), (dict(lda=96), "padding"), (dict(ldws=0), "padding"), (dict(W=C + 8), "aligned"),
    (dict(out=2), "output"), (dict(epi=4), "epilogue"), (dict(epi=6), "epilogue"), (dict(ldc=60), "ldc"),
    (dict(ldc=56), "ldc"), (dict(ldc=1 << 22), "strides"), (dict(epi=3, R=F, ldr=1 << 22), "strides"), (dict(out=1, epi=3, R=F, ldr=64), "bf16"), (dict(out=1, N=72), "N=72"),
    (dict(out=1, ldc=128), "MX output"), (dict(out=1, Cs=F, ldc=64, ldcs=16), "MX output"), (dict(epi=3), "residual"),
    (dict(epi=3, R=F, ldr=60), "residual"), (dict(epi=2, R=F, ldr=64), "gate"),
    (dict(epi=2, R=F, ldr=64, gate=G, gs=66, cu=H, nseg=1), "gate")])
def test_gemm_refuses(change, word):
    refused("ditk_mx_gemm", tuple({**GEMM, **change}.values()), word)


@pytest.mark.parametrize("change,word", [
    (dict(Ws=None), "null"), (dict(x=None), "null"), (dict(N=0), "shape"), (dict(K=48), "K=48"), (dict(N=4), "N=4"),
    (dict(ldw=48), "padding"), (dict(ldx=88), "padding"), (dict(x=A + 4), "aligned"), (dict(ldc=68), "ldc"),
    (dict(epi=2), "epilogue"), (dict(epi=3), "residual"), (dict(M=65536 * 32), "rows"), (dict(M=2**31 - 1), "rows"),
    (dict(K=81920, ldx=81920, ldw=40960, ldws=2560), "too long")])
def test_matvec_refuses(change, word):
    refused("ditk_mx_matvec", tuple({**MV, **change}.values()), word)


def plan(m, n, k):
    import ctypes
    p = (ctypes.c_int * 3)()
    _lib.call("ditk_mx_gemm_plan", m, n, k, p)
    return tuple(p)


def test_plans():
    """Few rows by single waves, then on small tiles, many on large ones, a short last round on smaller
    ones; both parts of a split have rows, the first one whole tile rows."""
    assert plan(16, 9216, 1536) == (6, 16, 0) and plan(100, 1544, 416) == (7, 100, 0)
    assert plan(130, 96, 128) == (6, 130, 0) and plan(128, 1536, 5120) == (7, 128, 0)
    assert plan(64, 9216, 1536) == (3, 64, 0) and plan(512, 4608, 1536) == (2, 512, 0)
    assert plan(667, 7296, 2432) == (1, 667, 0) and plan(65520, 1536, 8960) == (0, 65520, 0)
    assert plan(2600, 8968, 512) == (0, 1792, 1)
    assert plan(2600, 4096, 384) == (0, 2600, 0) and plan(2600, 4096, 128) == (4, 2600, 0)
    assert plan(700, 4104, 288) == (5, 700, 0)
    heights = (256, 128, 128, 64)
    for m in (1, 63, 64, 65, 127, 500, 1560, 2560, 4097, 20000, 65520):
        for n in (8, 96, 1536, 5120, 13824):
            for k in (416, 1536, 5120, 14336):
                tile, rows, rest = plan(m, n, k)
                assert tile in (0, 1, 2, 3, 6, 7) and 0 <= rest < 4 and 0 < rows <= m
                assert rows == m or rows % heights[tile] == 0
    assert plan(2**31 - 1, 8, 32)[0] not in (6, 7) and plan(8, 2**31 - 8, 32)[0] not in (6, 7)  # their grids
    with pytest.raises(_lib.DitkError):
        plan(0, 64, 64)


def test_no_rows_need_no_pointers():
    lib = _lib.load()
    none = dict(x=None, data=None, scales=None, T=0)
    assert lib.ditk_mx_quantize(*{**QUANT, **none}.values()) == 0
    assert lib.ditk_mx_norm(*{**NORM, **none}.values()) == 0
    assert lib.ditk_mx_gemm(*{**GEMM, **dict(A=None, As=None, C=None, M=0)}.values()) == 0
    assert lib.ditk_mx_matvec(*{**MV, **dict(x=None, C=None, M=0)}.values()) == 0


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


def rows(n, k):
    return torch.zeros((n, k), dtype=torch.bfloat16)


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="cuda"):
        mx.quantize(rows(4, 64))
    with pytest.raises(ValueError, match="cuda"):
        mx.norm(rows(4, 64))
    m = mx.MXTensor.empty(4, 64, "cpu")
    with pytest.raises(ValueError, match="cuda"):
        mx.MXTensor("fp8", m.data, m.scales, 64)


@pytest.mark.parametrize("call", [
    lambda: mx.quantize(rows(4, 40)), lambda: mx.quantize(rows(4, 64).float()), lambda: mx.quantize(rows(4, 64), "int8"),
    lambda: mx.quantize(rows(4, 64)[:, ::2]), lambda: mx.quantize(rows(4, 68)[:, :64]),
    lambda: mx.quantize(rows(4, 64), out=mx.MXTensor.empty(3, 64, "cpu")),
    lambda: mx.quantize(rows(4, 64), out=mx.MXTensor.empty(4, 64, "cpu", "fp4")), lambda: mx.quantize(rows(4, 64), out=rows(4, 64)),
    lambda: mx.MXTensor.empty(4, 48, "cpu"), lambda: mx.MXTensor.empty(4, 64, "cpu", "fp6")])
def test_python_quantize_refuses(host, call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize("kw", [
    dict(residual=rows(3, 64)), dict(residual_out=rows(4, 64)), dict(kind="batch"), dict(shift=torch.zeros(1, 64)),
    dict(shift=torch.zeros(1, 64), scale=torch.zeros(1, 64)), dict(weight=torch.zeros(63)), dict(bias=torch.zeros(64).bfloat16()),
    dict(shift=torch.zeros(1, 64), scale=torch.zeros(1, 64), segments=ops.Segments([0, 3], "cpu")),
    dict(shift=torch.zeros(1, 64), scale=torch.zeros(2, 128)[::2, :64], segments=ops.Segments([0, 4], "cpu")),
    dict(residual=rows(4, 64), residual_out=rows(8, 64)[::2][:, :32])])
def test_python_norm_refuses(host, kw):
    with pytest.raises(ValueError):
        mx.norm(rows(4, 64), **kw)


def test_outputs_over_operands_are_refused(host):
    buf = rows(9, 64)
    with pytest.raises(ValueError, match="overlaps"):
        mx.norm(buf[:8], rows(8, 64), residual_out=buf[1:])
    out = mx.MXTensor.empty(8, 64, "cpu")
    inside = out.data.view(torch.bfloat16)  # [8, 64] values over the output's own bytes
    with pytest.raises(ValueError, match="overlaps"):
        mx.quantize(inside, out=out)
    with pytest.raises(ValueError, match="overlaps"):
        mx.norm(rows(8, 64), inside, out=out)
    with pytest.raises(AssertionError, match="launched"):  # an input in place of the residual's sum
        mx.norm(buf[:8], rows(8, 64), residual_out=buf[:8])
    q, w, w4 = (mx.MXTensor.empty(n, 64, "cpu", f) for n, f in ((8, "fp8"), (32, "fp8"), (32, "fp4")))
    wide = rows(9, 32)
    with pytest.raises(ValueError, match="overlaps"):
        mx.linear(q, w, epilogue="res", residual=wide[:8], out=wide[1:])
    with pytest.raises(AssertionError, match="launched"):
        mx.linear(q, w, epilogue="res", residual=wide[:8], out=wide[:8])
    with pytest.raises(ValueError, match="overlaps"):
        mx.linear(q, w, out_fmt="fp8", out=mx.MXTensor("fp8", *both(q, 32), 32))
    x = rows(8, 64)
    with pytest.raises(ValueError, match="overlaps"):
        mx.matvec(x, w4, out=x[:, :32])


def both(m, cols):
    """The same bytes as an output of `cols` columns."""
    return m.data[:, :128], m.scales[:, :16]


@pytest.mark.parametrize("call", [
    lambda q, w, w4: mx.linear(q, w4), lambda q, w, w4: mx.linear(rows(8, 64), w), lambda q, w, w4: mx.linear(q, w, epilogue="f32"),
    lambda q, w, w4: mx.linear(q, w, epilogue="res"), lambda q, w, w4: mx.linear(q, w, out_fmt="bf16"),
    lambda q, w, w4: mx.linear(q, w, epilogue="res", residual=rows(8, 32), out_fmt="fp8"),
    lambda q, w, w4: mx.linear(q, w[:24], out_fmt="fp8"), lambda q, w, w4: mx.linear(q, w[:28]),
    lambda q, w, w4: mx.linear(q, w[:0]), lambda q, w, w4: mx.linear(q, w, torch.zeros(31)),
    lambda q, w, w4: mx.linear(q, w, out=rows(7, 32)), lambda q, w, w4: mx.linear(q, w, out=rows(8, 36)[:, :32]),
    lambda q, w, w4: mx.linear(q, mx.MXTensor.empty(32, 96, "cpu")),
    lambda q, w, w4: mx.linear(q, w, epilogue="gate_res", residual=rows(8, 32), gate=torch.zeros(1, 32)),
    lambda q, w, w4: mx.linear(q, w, epilogue="gate_res", residual=rows(8, 32), gate=torch.zeros(2, 32),
                               segments=ops.Segments([0, 8], "cpu")),
    lambda q, w, w4: mx.matvec(rows(8, 64), w), lambda q, w, w4: mx.matvec(rows(8, 96), w4),
    lambda q, w, w4: mx.matvec(rows(8, 64), w4, epilogue="gate_res"), lambda q, w, w4: mx.matvec(rows(8, 64).float(), w4),
    lambda q, w, w4: mx.matvec(rows(8, 64).view(2, 4, 64), w4), lambda q, w, w4: mx.matvec(rows(8, 64), w4, epilogue="res"),
    lambda q, w, w4: mx.matvec(rows(8, 64), w4, out=torch.zeros(8, 32)), lambda q, w, w4: q[::2], lambda q, w, w4: q[3]])
def test_python_products_refuse(host, call):
    q, w, w4 = (mx.MXTensor.empty(n, 64, "cpu", f) for n, f in ((8, "fp8"), (32, "fp8"), (32, "fp4")))
    with pytest.raises(ValueError):
        call(q, w, w4)
