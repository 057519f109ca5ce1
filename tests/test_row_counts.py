"""Row counts that a launch of the row kernels cannot hold are refused on the host (addresses only, no GPU)."""
import pytest

from ditserve_amd import _lib

if not _lib.LIB_PATH.exists():
    pytest.skip("libditk.so not built (run python -m ditserve_amd.build)", allow_module_level=True)

A, B, C, D, E = (0x10000 * i for i in range(1, 6))
ROWS = [(1 << 26) - 3, 1 << 26, 2**31 - 1]  # 2^24 workgroups of 256 threads, a wave a row


def refused(name, *args):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == 1
    assert "too many rows" in lib.ditk_last_error().decode(), lib.ditk_last_error()


@pytest.mark.parametrize("T", ROWS)
def test_adaln(T):
    refused("ditk_adaln", A, 64, B, 64, T, 64, None, 0, None, None, 0, None, None, 1e-6, 1, None)
    jobs = (_lib.AdalnJob * 2)(*(_lib.AdalnJob(x=A, ldx=64, y=B, ldy=64, T=t, D=64, norm_kind=1, eps=1e-6)
                                 for t in (T - 5, 5)))
    refused("ditk_adaln_multi", jobs, 2, None)


@pytest.mark.parametrize("T", ROWS)
def test_qk_norm(T):
    refused("ditk_qk_norm_rope", A, 64, B, 64, T, 64, 64, C, D, 1e-6, 1, None, None, 0, None, None, 0, 0, 0, None)
    jobs = (_lib.QkNormJob * 1)(_lib.QkNormJob(q=A, ldq=64, k=B, ldk=64, q_out=A, ldqo=64, k_out=B, ldko=64, wq=C, wk=D,
                                               T=T, D=64, head_dim=64, per_head=1, eps=1e-6))
    refused("ditk_qk_norm_multi", jobs, 1, None)


@pytest.mark.parametrize("total", [1 << 26, 2**31 - 1])
def test_joint_copy(total):
    refused("ditk_joint_copy", A, 64, B, 64, C, 64, D, E, 1, total, 64, 0, None)
