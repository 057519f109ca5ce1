"""Which kernel the microscaled (MX) products run on, by size, row stride and output (host only, 256 CUs)."""
import pytest

from ditserve_amd import _lib
from tests.helpers import mx_gemm_plan

if not _lib.LIB_PATH.exists():
    pytest.skip("libditk.so not built (run python -m ditserve_amd.build)", allow_module_level=True)

WIDE = (1 << 23) + 16  # 256 rows of it pass 2^31 bytes


@pytest.mark.parametrize("shape,want", [
    # few rows or few features by single waves, 16 x 16 outputs (6; 16 x 32 for an MX output) or 32 x 32 (7)
    ((129, 24, 8960), (6, 129, 0)), ((300, 40, 14336), (6, 300, 0)), ((4353, 24, 544), (7, 4353, 0)),
    # tiles wider than the matrix
    ((9000, 120, 1536), (3, 9000, 0)), ((20000, 64, 1536), (2, 20000, 0)), ((40000, 200, 1536), (0, 40000, 0)),
    # split launches
    ((1000, 4616, 1056), (1, 1000, 0)), ((2600, 4104, 640), (0, 2600, 0)), ((4600, 5128, 416), (0, 3072, 1)),
    ((9000, 2440, 3104), (0, 6400, 1)), ((70000, 200, 1536), (0, 65536, 3))])
def test_plans_of_bf16_outputs(shape, want):
    assert mx_gemm_plan(*shape) == want
    p = mx_gemm_plan(*shape, name="ditk_mx_gemm_plan")
    assert p == want


@pytest.mark.parametrize("shape,want", [
    ((1560, 8960, 512), (0, 1560, 0)), ((333, 4640, 1536), (3, 333, 0)), ((700, 7328, 1056), (1, 700, 0)),
    ((100, 1568, 416), (7, 100, 0)), ((4600, 5152, 448), (0, 3072, 1)), ((20000, 96, 672), (2, 20000, 0)),
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
