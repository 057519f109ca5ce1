"""Which kernel the microscaled (MX) products run on, by size, row stride and output (host only, 256 CUs)."""
import pytest

from ditserve_amd import _lib
from tests.helpers import mx_gemm_plan, mx_matvec_plan

if not _lib.LIB_PATH.exists():
    pytest.skip("libditk.so not built (run python -m ditserve_amd.build)", allow_module_level=True)

WIDE = (1 << 23) + 16  # 256 rows of it pass 2^31 bytes


@pytest.mark.parametrize("shape,want", [
    # few rows or few features by single waves, 16 x 16 outputs (6; 16 x 32 for an MX output) or 32 x 32 (7)
    ((129, 24, 8960), (6, 129, 0)), ((300, 40, 14336), (6, 300, 0)), ((4353, 24, 544), (7, 4353, 0)),
    # tiles wider than the matrix
    ((9000, 120, 1536), (3, 9000, 0)), ((20000, 64, 1536), (2, 20000, 0)), ((40000, 200, 1536), (0, 40000, 0)),
    # split launches
    ((1000, 4616, 1056), (1, 1000, 0)), ((2600, 4104, 640), (0, 2600, 0)), ((2600, 8968, 512), (0, 1792, 1)),
    ((9000, 2440, 3104), (0, 6400, 1)), ((70000, 200, 1536), (0, 65536, 3))])
def test_plans_of_bf16_outputs(shape, want):
    assert mx_gemm_plan(*shape) == want
    p = mx_gemm_plan(*shape, name="ditk_mx_gemm_plan")
    assert p == want


@pytest.mark.parametrize("shape,want", [
    ((1560, 8960, 512), (0, 1560, 0)), ((333, 4640, 1536), (3, 333, 0)), ((700, 7328, 1056), (1, 700, 0)),
    ((100, 1568, 416), (7, 100, 0)), ((4353, 4128, 448), (0, 3840, 2)), ((20000, 96, 672), (2, 20000, 0)),
    ((16, 1536, 1536), (6, 16, 0))])
def test_plans_of_mx_outputs(shape, want):
    assert mx_gemm_plan(*shape, mx_out=True) == want


@pytest.mark.parametrize("mx_out", [False, True])
def test_plans_of_wide_strides(mx_out):
    """Row strides that 32-bit offsets do not reach over 256 rows: 256 x 256 (4) and 64 x 128 (5) with 64-bit
    addresses, but for few rows, whose kernel has 64-bit addresses anyway."""
    for k in (512, 1056, 14336):
        assert mx_gemm_plan(5, 96, k, WIDE, mx_out)[0] in (6, 7)
        assert mx_gemm_plan(1333, 1568, k, WIDE, mx_out) == (5, 1333, 0)
        assert mx_gemm_plan(4200, 2016, k, WIDE, mx_out) == (4, 4200, 0)
        assert mx_gemm_plan(4200, 2016, k, (1 << 23) - 16, mx_out)[0] < 4


def test_plan_refusals():
    for bad in (dict(m=0), dict(n=12), dict(k=40), dict(ld=96), dict(n=24, mx_out=True)):
        with pytest.raises(_lib.DitkError, match="bad arguments"):
            mx_gemm_plan(**{**dict(m=4, n=64, k=128), **bad})


HOST = dict(A=0x10000, lda=128, As=0x20000, ldas=16, W=0x30000, ldw=128, Ws=0x40000, ldws=16, bias=None, C=0x50000,
            ldc=64, Cs=None, ldcs=0, M=4, N=64, K=96, epi=0, out=0, R=None, ldr=0, gate=None, gs=0, cu=None, nseg=0,
            stream=None)  # addresses only


@pytest.mark.parametrize("change,word", [(dict(M=2**31 - 1), "rows"), (dict(M=2**31 - 2**28 + 1), "rows"),
                                         (dict(K=2**31 - 32, lda=1 << 31, ldw=1 << 31, ldas=1 << 26, ldws=1 << 26), "long"),
                                         (dict(K=2**30 + 32, lda=1 << 31, ldw=1 << 31, ldas=1 << 26, ldws=1 << 26), "long")])
def test_product_refuses_sizes_near_2_31(change, word):
    lib = _lib.load()
    assert lib.ditk_mx_gemm(*{**HOST, **change}.values()) == 1
    assert word in lib.ditk_last_error().decode(), lib.ditk_last_error()


@pytest.mark.parametrize("K", [2**31 - 32, 2**30 + 32])
def test_quantize_refuses_rows_near_2_31(K):
    lib = _lib.load()
    assert lib.ditk_mx_quantize(0x10000, 1 << 31, 0x20000, 1 << 31, 0x30000, 1 << 26, 1, K, 0, None) == 1
    assert "too long" in lib.ditk_last_error().decode(), lib.ditk_last_error()


def test_plans_near_2_31():
    """Row, feature and column counts are multiplied and rounded up past 31 bits."""
    for m, n, k in ((2**31 - 1, 8, 512), (2**31 - 1, 264, 32), (8, 2**31 - 8, 512), (2**31 - 1, 2**31 - 8, 1536)):
        assert mx_gemm_plan(m, n, k)[0] not in (6, 7), (m, n, k)
    assert mx_gemm_plan(2**31 - 1, 264, 32) == (4, 2**31 - 1, 0)
    # the longest rows: no fewer steps than those of half the length
    assert mx_gemm_plan(16, 64, 2**31 - 32)[0] == mx_gemm_plan(16, 64, 2**30)[0]


@pytest.mark.parametrize("shape,want", [
    # few rows past the weight: one or two fragments of 16 rows, more rows in more passes
    ((1, 9216, 1536), (0, 1, 1)), ((2, 499712, 1536), (0, 1, 1)), ((17, 264, 2432), (0, 2, 1)), ((100, 72, 1536), (0, 2, 4)),
    ((33, 520, 8960), (0, 1, 5)), ((2, 24, 60000), (0, 1, 2)), ((1, 24, 65408), (0, 1, 1)),
    # tiles of 64 features, 1 to 4 fragments
    ((11, 10008, 13856), (1, 1, 1)), ((25, 9000, 8928), (1, 2, 1)), ((48, 9000, 8960), (1, 3, 1)),
    ((64, 9224, 5120), (1, 4, 1)), ((64, 16000, 480), (1, 4, 1)),
    # and of 128
    ((3, 27016, 5120), (2, 1, 1)), ((2, 33800, 4640), (2, 1, 1)), ((30, 17000, 1568), (2, 2, 1)),
    ((17, 33016, 1056), (2, 2, 1)), ((40, 33000, 2432), (2, 3, 1)), ((100, 16648, 1056), (2, 4, 2))])
def test_plans_of_matvec(shape, want):
    assert mx_matvec_plan(*shape) == want
    # what one row of a few features runs on, which others are compared with bitwise
    assert mx_matvec_plan(1, 1000, shape[2])[0] == 0


def test_matvec_plan_refusals():
    for bad in ((0, 64, 128), (1, 12, 128), (1, 64, 40), (1, 64, 65440), (1, 64, 2**31 - 32), (65536 * 32, 64, 128)):
        with pytest.raises(_lib.DitkError):
            mx_matvec_plan(*bad)
