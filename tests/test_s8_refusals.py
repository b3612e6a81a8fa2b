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
    assert rc(_6=24) == L.W4_ERR_UNSUPPORTED and rc(_5=2**30 + 1) == L.W4_ERR_UNSUPPORTED
    assert rc(_0=None, _3=None, _4=None, _5=0) == L.W4_OK  # no rows: nothing to do


def test_quant_s8_wrapper_refusals():
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.quant_s8(x)
    with pytest.raises(ValueError, match="act"):
        ops.quant_s8(x, "gelu")
    with pytest.raises(ValueError, match="2-D"):
        ops.quant_s8(torch.zeros(64))


def _with(call, ok):
    def rc(**kw):
        args = list(ok)
        for i, v in kw.items():
            args[int(i[1:])] = v
        return call(*args)
    return rc


def test_moe_route_refusals():
    lib = L.lib()
    #       logits dtype  bias  T   E  k  score  G  tg gs  ren scale  ids  w    off   rows  slots ws   bytes   stream
    ok = [_f(), L.W4_BF16, None, 300, 64, 6, 0, 1, 1, 0, 1, 1.0, _f(), _f(), _f(), _f(), _f(), _f(), 1 << 20, None]
    rc = _with(lib.w4_moe_route, ok)
    for i in (0, 12, 13):
        assert rc(**{f"_{i}": None}) == L.W4_ERR_INVALID
    for i in (14, 15, 16):  # the plan's tensors come together
        assert rc(**{f"_{i}": None}) == L.W4_ERR_INVALID and b"together" in lib.w4_last_error()
    assert rc(_1=L.W4_E4M3) == L.W4_ERR_INVALID
    assert rc(_3=-1) == L.W4_ERR_INVALID
    assert rc(_4=0) == L.W4_ERR_INVALID
    assert rc(_4=513) == L.W4_ERR_UNSUPPORTED
    assert rc(_5=0) == L.W4_ERR_INVALID
    assert rc(_5=33) == L.W4_ERR_UNSUPPORTED
    assert rc(_4=4, _5=6) == L.W4_ERR_INVALID            # more than there are
    assert rc(_6=2) == L.W4_ERR_INVALID and rc(_9=2) == L.W4_ERR_INVALID
    assert rc(_7=5) == L.W4_ERR_INVALID                  # does not divide 64
    assert rc(_7=8, _8=9) == L.W4_ERR_INVALID and rc(_7=8, _8=0) == L.W4_ERR_INVALID
    assert rc(_7=16, _8=1, _5=6) == L.W4_ERR_INVALID     # 4 experts to choose 6 from
    assert rc(_4=32, _7=32, _8=8, _9=1) == L.W4_ERR_INVALID  # top 2 of groups of one
    assert rc(_7=64, _8=64) == L.W4_ERR_UNSUPPORTED
    assert rc(_3=2**30) == L.W4_ERR_UNSUPPORTED          # T * top_k past 2^31
    assert rc(_3=2**31 - 1, _5=1) == L.W4_ERR_UNSUPPORTED
    assert rc(_17=None) == L.W4_ERR_INVALID and b"workspace" in lib.w4_last_error()
    assert rc(_18=16) == L.W4_ERR_INVALID
    assert rc(_0=_f(0x10001)) == L.W4_ERR_INVALID
    assert lib.w4_moe_route_workspace_bytes(8, 64) == 0 and lib.w4_moe_route_workspace_bytes(0, 64) == 0
    assert lib.w4_moe_route_workspace_bytes(8192, 256) >= 8192 // 1024 * 256 * 2


def test_moe_combine_refusals():
    lib = L.lib()
    ok = [_f(), L.W4_BF16, 48, _f(), _f(), None, _f(0x90000), L.W4_BF16, 8, 6, 64, None]
    rc = _with(lib.w4_moe_combine, ok)
    for i in (0, 3, 4, 6):
        assert rc(**{f"_{i}": None}) == L.W4_ERR_INVALID
    assert rc(_1=L.W4_S8) == L.W4_ERR_INVALID and rc(_7=L.W4_E4M3) == L.W4_ERR_INVALID
    assert rc(_2=-1) == L.W4_ERR_INVALID and rc(_8=-1) == L.W4_ERR_INVALID and rc(_10=0) == L.W4_ERR_INVALID
    assert rc(_9=0) == L.W4_ERR_INVALID and rc(_9=33) == L.W4_ERR_UNSUPPORTED
    assert rc(_10=2**22 + 1) == L.W4_ERR_UNSUPPORTED
    assert rc(_6=_f()) == L.W4_ERR_INVALID               # out is y
    assert rc(_8=0) == L.W4_OK


def test_moe_wrapper_refusals():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.moe_route(x, 2)
    with pytest.raises(ValueError, match="score"):
        ops.moe_route(x, 2, score="tanh")
    with pytest.raises(ValueError, match="group_score"):
        ops.moe_route(x, 2, group_score="sum")
    with pytest.raises(ValueError, match="2-D"):
        ops.moe_route(x[0], 2)
    with pytest.raises(ValueError, match="CUDA"):
        ops.moe_combine(x, torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2))


def test_s8_gemm_refusals():
    lib = L.lib()
    #       a     as    w     ws    bias  c     dtype      rs    M  N   K   ws    bytes stream
    ok = [_f(), _f(), _f(), _f(), None, _f(), L.W4_BF16, None, 4, 64, 64, None, 0, None]
    rc = _with(lib.w4_s8_gemm, ok)
    for i in (0, 1, 2, 3, 5):
        assert rc(**{f"_{i}": None}) == L.W4_ERR_INVALID
    for i in (0, 2):
        assert rc(**{f"_{i}": _f(0x10008)}) == L.W4_ERR_INVALID and b"aligned" in lib.w4_last_error()
    assert rc(_6=L.W4_S8) == L.W4_ERR_INVALID
    assert rc(_8=-1) == L.W4_ERR_INVALID and rc(_9=0) == L.W4_ERR_INVALID and rc(_10=0) == L.W4_ERR_INVALID
    assert rc(_8=2**31 - 1) == L.W4_ERR_UNSUPPORTED and rc(_9=2**31 - 1) == L.W4_ERR_UNSUPPORTED
    assert rc(_10=72) == L.W4_ERR_UNSUPPORTED and rc(_10=131072) == L.W4_ERR_UNSUPPORTED
    assert rc(_6=L.W4_E4M3) == L.W4_ERR_INVALID and b"row_scale" in lib.w4_last_error()
    assert rc(_6=L.W4_E4M3, _7=_f()) == L.W4_ERR_INVALID and b"workspace" in lib.w4_last_error()
    assert rc(_8=0, _0=None) == L.W4_OK
    assert lib.w4_s8_gemm_workspace_bytes(4, 64, 64, L.W4_BF16) == 0
    assert lib.w4_s8_gemm_workspace_bytes(4, 64, 64, L.W4_E4M3) == 1024


def test_s8_gemm_grouped_refusals():
    lib = L.lib()
    #       a     as  a_rows w    ws    bias  off   rows E  c     dtype      rs   R  N   K   ws    bytes stream
    ok = [_f(), _f(), 8, _f(), _f(), None, _f(), None, 4, _f(), L.W4_BF16, None, 8, 64, 64, None, 0, None]
    rc = _with(lib.w4_s8_gemm_grouped, ok)
    for i in (0, 1, 3, 4, 6, 9):
        assert rc(**{f"_{i}": None}) == L.W4_ERR_INVALID
    assert rc(_2=7) == L.W4_ERR_INVALID and b"a_rows" in lib.w4_last_error()
    assert rc(_2=0, _7=_f()) == L.W4_ERR_INVALID
    assert rc(_8=0) == L.W4_ERR_INVALID and rc(_8=513) == L.W4_ERR_UNSUPPORTED
    assert rc(_12=-1) == L.W4_ERR_INVALID and rc(_14=24) == L.W4_ERR_UNSUPPORTED
    assert rc(_10=L.W4_E4M3) == L.W4_ERR_INVALID
    assert rc(_0=_f(0x10004)) == L.W4_ERR_INVALID and rc(_6=_f(0x10002)) == L.W4_ERR_INVALID
    assert rc(_12=0, _2=0) == L.W4_OK


def test_s8_wrapper_refusals():
    a, s = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4)
    w, ws = torch.zeros(8, 64, dtype=torch.int8), torch.zeros(8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.s8_gemm(a, s, w, ws)
    with pytest.raises(ValueError):
        ops.s8_gemm(a, s, w[0], ws)
    with pytest.raises(ValueError):
        ops.s8_gemm_grouped(a, s, w, ws, torch.zeros(2, dtype=torch.int32))


def test_sizes_past_32_bits_are_refused_before_the_call():
    """A size of 2^32 + 64 would arrive as 64."""
    big = 2**32 + 64

    def meta(*shape, dtype=torch.int8):
        return torch.empty(shape, dtype=dtype, device="meta")

    s1 = meta(1, dtype=torch.float32)
    off = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.quant_s8(meta(1, big, dtype=torch.float16)),
                 lambda: ops.quant_s8(meta(big, 16, dtype=torch.float16)),
                 lambda: ops.s8_gemm(meta(big, 16), s1, meta(1, 16), s1),
                 lambda: ops.s8_gemm(meta(1, 16), s1, meta(big, 16), s1),
                 lambda: ops.s8_gemm_grouped(meta(big, 16), s1, meta(1, 1, 16), s1, off),
                 lambda: ops.moe_route(meta(big, 1, dtype=torch.float16), 1),
                 lambda: ops.moe_route(meta(1, 64, dtype=torch.float16), 1, n_group=2**32 + 1),
                 lambda: ops.moe_combine(meta(1, big), meta(1, 1), meta(1, 1))):
        with pytest.raises(ValueError, match="2\\^31"):
            call()
