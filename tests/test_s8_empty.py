"""The 8-bit entry points take empty batches without their pointers (no GPU needed)."""
import ctypes

import pytest

from xe2x2_b200 import _lib as L


def _f(addr=0x10000):
    return ctypes.c_void_p(addr)


@pytest.mark.parametrize("a_rows", [0, 8])
@pytest.mark.parametrize("dtype", [L.W4_BF16, L.W4_E4M3])
def test_a_grouped_batch_without_rows(a_rows, dtype):
    """No row is gathered from eight tokens: an empty index has no address."""
    call = L.lib().w4_s8_gemm_grouped
    assert call(_f(), _f(), a_rows, _f(), _f(), None, _f(), None, 4, None, dtype, None, 0, 64, 64, None, 0,
                None) == L.W4_OK
    assert call(_f(), _f(), -1, _f(), _f(), None, _f(), None, 4, None, dtype, None, 0, 64, 64, None, 0,
                None) == L.W4_ERR_INVALID
