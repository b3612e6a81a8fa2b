"""The 8-bit integer and mixture-of-experts entry points refuse bad arguments on the host, before
anything is launched (no GPU needed)."""
import ctypes

import pytest
import torch

from xe2x2_b200 import _lib as L
from xe2x2_b200 import ops


def _f(addr=0x10000):
    return ctypes.c_void_p(addr)


def test_quant_s8_refusals():
    call = L.lib().w4_quant_s8
    ok = [_f(), L.W4_BF16, L.W4_FN_NONE, _f(), _f(), 4, 64, None]

    def rc(**kw):
        args = list(ok)
        for i, v in kw.items():
            args[int(i[1:])] = v
        return call(*args)

    assert rc(_0=None) == L.W4_ERR_INVALID and b"null" in L.lib().w4_last_error()
    assert rc(_1=L.W4_E4M3) == L.W4_ERR_INVALID
    assert rc(_2=3) == L.W4_ERR_INVALID
    assert rc(_0=_f(0x10008)) == L.W4_ERR_INVALID and b"aligned" in L.lib().w4_last_error()
    assert rc(_3=_f(0x10008)) == L.W4_ERR_INVALID
    assert rc(_5=-1) == L.W4_ERR_INVALID
    assert rc(_6=0) == L.W4_ERR_INVALID
    assert rc(_6=24) == L.W4_ERR_UNSUPPORTED
    assert rc(_0=None, _3=None, _4=None, _5=0) == L.W4_OK  # no rows: nothing to do


def test_quant_s8_wrapper_refusals():
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.quant_s8(x)
    with pytest.raises(ValueError, match="act"):
        ops.quant_s8(x, "gelu")
    with pytest.raises(ValueError, match="2-D"):
        ops.quant_s8(torch.zeros(64))
