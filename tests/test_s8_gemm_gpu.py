"""w4_s8_gemm and w4_s8_gemm_grouped against the exact integer sums, scaled in 64 bits."""
import numpy as np
import pytest
import torch

import oracle as O
from tests._util import np_
from xe2x2_b200 import _lib as L
from xe2x2_b200 import ops

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _s8(shape, g):
    return torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int32).to(torch.int8)


def _scales(shape, g):
    return (0.5 + torch.rand(shape, generator=g, device="cuda")) * 1e-3


def _check(out, acc, a_scale, w_scale, bias):
    """acc: exact sums (f64).  The kernel rounds the sum to f32, the product with the token's scale, the
    fused multiply-add with the channel's scale and the bias, and the store."""
    p = acc * a_scale.double()[:, None] * w_scale.double()
    y = p if bias is None else p + bias.double()
    half = 0.0 if out.dtype == torch.float32 else torch.finfo(out.dtype).eps / 2
    tol = 2.01 * 2.0 ** -24 * p.abs() + (2.0 ** -24 + 1.01 * half) * y.abs()
    tol += 2.0 ** -25 if out.dtype == torch.float16 else 1e-38
    d = (out.double() - y).abs()
    assert bool((d <= tol).all()), float((d / tol.clamp(min=1e-300)).max())


DENSE = [(1, 1, 16), (1, 128, 128), (2, 3, 32), (3, 130, 48), (16, 256, 2688), (17, 64, 1856), (33, 300, 144),
         (64, 512, 512), (65, 1000, 272), (100, 256, 1024), (128, 127, 640), (129, 129, 1040), (200, 333, 4096),
         (300, 2688, 1856), (1000, 384, 512), (257, 4224, 256), (5, 5120, 17408), (1, 5120, 5120), (2, 17408, 5120),
         (700, 5120, 640), (2050, 1856, 2688), (3, 257, 4096), (40, 131, 8192), (150, 259, 4096), (250, 130, 2064)]


@pytest.mark.parametrize("out", list(DTYPES))
@pytest.mark.parametrize("M,N,K", DENSE)
def test_gemm(cuda, M, N, K, out):
    g = _gen(M + 3 * N + K)
    a, w = _s8((M, K), g), _s8((N, K), g)
    sa, sw = _scales(M, g), _scales(N, g)
    bias = torch.randn(N, generator=g, device=cuda) if (M + N) % 2 else None
    acc = a.double() @ w.double().t()
    _check(ops.s8_gemm(a, sa, w, sw, bias, DTYPES[out]), acc, sa, sw, bias)
    assert L.lib().w4_check_device_status() == L.W4_OK


def test_largest_sums_are_exact(cuda):
    """-128 * -128 over the longest K: the sum is the largest that s32 is asked to hold."""
    K = 131056
    one = torch.ones(2, device=cuda)
    a = torch.full((2, K), -128, dtype=torch.int8, device=cuda)
    w = torch.full((2, K), -128, dtype=torch.int8, device=cuda)
    w[1] = 127
    y = ops.s8_gemm(a, one, w, one, out_dtype=torch.float32)
    assert y.double().tolist() == [[float(np.float32(16384 * K)), float(np.float32(-16256 * K))]] * 2


@pytest.mark.parametrize("M,N,K", [(1, 5120, 4096), (40, 640, 2048), (300, 1000, 1024)])
def test_equal_calls_give_equal_bits_and_rows_do_not_mix(cuda, M, N, K):
    g = _gen(5)
    a, w, sa, sw = _s8((M, K), g), _s8((N, K), g), _scales(M, g), _scales(N, g)
    y = ops.s8_gemm(a, sa, w, sw, out_dtype=torch.float32)
    assert torch.equal(y, ops.s8_gemm(a, sa, w, sw, out_dtype=torch.float32))
    # each row by itself (another tile, another split): the integer sums are exact, so the same bits
    i = M // 2
    assert torch.equal(y[i:i + 1], ops.s8_gemm(a[i:i + 1].clone(), sa[i:i + 1].clone(), w, sw, out_dtype=torch.float32))


def test_rows_with_nan_scales_stay_their_own(cuda):
    x = torch.randn(20, 256, device=cuda)
    x[3, 5] = float("inf")
    g = _gen(6)
    w, sw = _s8((96, 256), g), _scales(96, g)
    q, s = ops.quant_s8(x)
    y = ops.s8_gemm(q, s, w, sw, out_dtype=torch.float32)
    assert torch.isnan(y[3]).all() and torch.isfinite(y[[0, 1, 2] + list(range(4, 20))]).all()


@pytest.mark.parametrize("M", [1, 16, 40, 300])
def test_fp8_output_is_the_row_scaled_cast(cuda, M):
    g = _gen(M)
    N, K = 330, 512
    a, w, sa, sw = _s8((M, K), g), _s8((N, K), g), _scales(M, g), _scales(N, g)
    y = ops.s8_gemm(a, sa, w, sw, out_dtype=torch.float32)
    q, s = ops.s8_gemm(a, sa, w, sw, out_dtype=torch.float8_e4m3fn)
    q_ref, s_ref = O.rowscale_fp8(np_(y))
    assert np.array_equal(np_(q.view(torch.uint8)), q_ref) and np.array_equal(np_(s), s_ref)


def test_out_argument_no_rows_and_streams(cuda):
    g = _gen(9)
    a, w, sa, sw = _s8((30, 512), g), _s8((200, 512), g), _scales(30, g), _scales(200, g)
    want = ops.s8_gemm(a, sa, w, sw)
    buf = torch.full((32, 200), 7.0, dtype=torch.bfloat16, device=cuda)
    assert ops.s8_gemm(a, sa, w, sw, out=buf[:30]).data_ptr() == buf.data_ptr()
    assert torch.equal(buf[:30], want) and (buf[30:] == 7).all()
    assert ops.s8_gemm(a[:0], sa[:0], w, sw).shape == (0, 200)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        q = (a.int() // 2).to(torch.int8)  # written by the kernel just before
        y = ops.s8_gemm(q, sa, w, sw)
    side.synchronize()
    assert torch.equal(y, ops.s8_gemm((a.int() // 2).to(torch.int8), sa, w, sw))


# ------------------------------------------------------------------------------------- grouped
COUNTS = {
    "decode": [3, 0, 1, 7, 2, 16, 5, 1],
    "ragged": [20, 1, 0, 33, 9, 2, 17, 4],
    "heavy": [150, 3, 0, 600, 17, 1, 0, 9],
    "one": [0, 0, 20, 0, 0, 0, 0, 0],
    "last": [0, 0, 0, 0, 0, 0, 0, 129],
    "none": [0] * 8,
    "single": [5],
    "many": [(e * 7) % 5 for e in range(300)],
}


def _grouped(cnt, N, K, seed, gather, tail=0):
    g = _gen(seed)
    E, off = len(cnt), [0] + list(np.cumsum(cnt))
    R = off[-1] + tail
    T = max(1, R // 2) if gather else R
    a, sa = _s8((T, K), g), _scales(T, g)
    w, sw = _s8((E, N, K), g), _scales((E, N), g)
    bias = torch.randn(E, N, generator=g, device="cuda")
    rows = torch.randint(0, T, (R,), generator=g, device="cuda", dtype=torch.int32) if gather else None
    return a, sa, w, sw, bias, torch.tensor(off, dtype=torch.int32, device="cuda"), rows, off, R


def _check_grouped(out, a, sa, w, sw, bias, rows, off):
    for e in range(len(off) - 1):
        i, j = off[e], off[e + 1]
        if i == j:
            continue
        src = torch.arange(i, j, device="cuda") if rows is None else rows[i:j].long()
        acc = a[src].double() @ w[e].double().t()
        _check(out[i:j], acc, sa[src], sw[e], None if bias is None else bias[e])


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("counts", list(COUNTS))
@pytest.mark.parametrize("N,K", [(1856, 2688), (300, 48), (129, 1040)])
def test_grouped(cuda, counts, N, K, gather):
    cnt = COUNTS[counts]
    a, sa, w, sw, bias, offsets, rows, off, R = _grouped(cnt, N, K, len(cnt) + N, gather)
    if R == 0:
        out = ops.s8_gemm_grouped(a[:0], sa[:0], w, sw, offsets)
        assert out.shape == (0, N)
        return
    for dt, b in ((torch.float32, None), (torch.bfloat16, bias)):
        out = ops.s8_gemm_grouped(a, sa, w, sw, offsets, rows, b, dt)
        _check_grouped(out, a, sa, w, sw, b, rows, off)
    assert L.lib().w4_check_device_status() == L.W4_OK


@pytest.mark.parametrize("gather", [False, True])
def test_grouped_leaves_rows_behind_the_last_expert(cuda, gather):
    a, sa, w, sw, _, offsets, rows, off, R = _grouped([3, 0, 40, 9], 200, 256, 3, gather, tail=30)
    if gather:
        rows[off[-1]:] = -1  # as the router leaves them
    buf = torch.full((R, 200), 7.0, device=cuda)
    out = ops.s8_gemm_grouped(a, sa, w, sw, offsets, rows, out=buf, out_dtype=torch.float32)
    _check_grouped(out, a, sa, w, sw, None, rows, off)
    assert (out[off[-1]:] == 7).all()
    q, s = ops.s8_gemm_grouped(a, sa, w, sw, offsets, rows, out_dtype=torch.float8_e4m3fn)
    q_ref, s_ref = O.rowscale_fp8(np_(out[:off[-1]]))
    assert np.array_equal(np_(q.view(torch.uint8))[:off[-1]], q_ref) and np.array_equal(np_(s)[:off[-1]], s_ref)
    q2 = torch.full((R, 200), 1.0, device=cuda).to(torch.float8_e4m3fn)
    ops.s8_gemm_grouped(a, sa, w, sw, offsets, rows, out=q2)
    assert (q2[off[-1]:].float() == 1).all()
    none = torch.zeros_like(offsets)  # no expert has rows
    buf.fill_(5.0)
    ops.s8_gemm_grouped(a, sa, w, sw, none, rows, out=buf)
    assert (buf == 5).all()


def test_grouped_rows_outside_the_tokens_are_zeros(cuda):
    a, sa, w, sw, bias, offsets, rows, off, R = _grouped([9, 30, 2], 140, 272, 4, True)
    rows[5], rows[20] = -1, a.shape[0]
    out = ops.s8_gemm_grouped(a, sa, w, sw, offsets, rows, bias, torch.float32)
    assert torch.equal(out[5], bias[0]) and torch.equal(out[20], bias[1])
    keep = [i for i in range(R) if i not in (5, 20)]
    rows2 = rows.clone()
    rows2[5] = rows2[20] = 0
    assert torch.equal(out[keep], ops.s8_gemm_grouped(a, sa, w, sw, offsets, rows2, bias, torch.float32)[keep])


def test_grouped_offsets_out_of_range_are_clamped(cuda):
    """Offsets that the device memory holds wrongly never reach outside the buffers."""
    a, sa, w, sw, _, offsets, _, off, R = _grouped([5, 20, 3, 8], 130, 128, 5, False)
    buf = torch.full((R + 4, 130), 7.0, device=cuda)
    bad = torch.tensor([0, -50, 1 << 30, 3, -(1 << 31)], dtype=torch.int32, device=cuda)
    out = ops.s8_gemm_grouped(a, sa, w, sw, bad, out=buf[:R])
    _check_grouped(out, a, sa, w, sw, None, None, [0, 0, R, R, R])  # expert 1 gets every row
    assert (buf[R:] == 7).all()


def test_grouped_equals_plain_calls_bit_for_bit(cuda):
    a, sa, w, sw, _, offsets, _, off, _ = _grouped([70, 1, 300, 12], 500, 768, 6, False)
    y = ops.s8_gemm_grouped(a, sa, w, sw, offsets, out_dtype=torch.float32)
    for e in range(4):
        i, j = off[e], off[e + 1]
        assert torch.equal(y[i:j], ops.s8_gemm(a[i:j].clone(), sa[i:j].clone(), w[e], sw[e], out_dtype=torch.float32))
