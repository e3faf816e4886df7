"""CPU: a grouped product without groups still needs its one bound; without it the call is refused before anything is launched."""
import pytest

from dance_amd import _lib

P = 4096  # some non-null address: no call below may get as far as using it
INVALID = -1


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("trans_b", [0, 1])
@pytest.mark.parametrize("zero", [0, 1])
@pytest.mark.parametrize("W", [None, P])
def test_no_groups_and_no_bounds(dtype, trans_b, zero, W):
    lib = _lib.load()
    rc = lib.dh_gemm_grouped(8, 4, 4, 0, trans_b, dtype, P, 4, W, 4, 0, None, None, 0, 0, P, 4, dtype, zero, None)
    assert rc == INVALID and b"dh_gemm_grouped" in lib.dh_last_error_string()
    assert lib.dh_gemm_grouped(0, 4, 4, 0, trans_b, dtype, None, 4, W, 4, 0, None, None, 0, 0, None, 4, dtype, zero, None) == 0  # no rows either
