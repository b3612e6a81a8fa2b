"""w4_quant_s8 / ops.quant_s8 against the definition in 64 bits."""
import numpy as np
import pytest
import torch

from tests._util import np_
from xe2x2_b200 import ops

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# relative error of y with SwiGLU: the exponential 2^-22 and its argument's rounding, |g| 2^-24 (gates
# below 8 in size here), the sum 2^-24, the reciprocal 2^-23, two products 2^-24 each; the scale's
# division rounds once more
Y_REL = {None: 0.0, "relu2": 2.0 ** -24, "silu_mul": 2.0 ** -22 + 8 * 2.0 ** -24 + 3 * 2.0 ** -24 + 2.0 ** -23}


def _y64(x, act):
    x = np_(x.double())
    if act == "silu_mul":
        k = x.shape[1] // 2
        return x[:, :k] / (1 + np.exp(-x[:, :k])) * x[:, k:]
    return np.maximum(x, 0) ** 2 if act == "relu2" else x


def _check(x, act):
    y = _y64(x, act)
    q, s = ops.quant_s8(x, act)
    q, s = np_(q).astype(np.float64), np_(s).astype(np.float64)
    amax = np.abs(y).max(1)
    want = np.where(amax > 0, amax / 127, 1.0)
    assert np.all(np.abs(s - want) <= want * (Y_REL[act] + 2.0 ** -24))
    # q is the nearest whole number to y / s, whose rounding errors are below 127 * 2 * (its relative
    # error): half a step and that much
    slack = 127 * 2 * (Y_REL[act] + 2.0 ** -23)
    assert np.all(np.abs(q - y / s[:, None]) <= 0.5 + slack)
    assert np.abs(q).max() <= 127


@pytest.mark.parametrize("act", [None, "silu_mul", "relu2"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("M,K", [(1, 16), (3, 48), (5, 2688), (2, 17408), (300, 1856), (1, 40000), (7, 8208)])
def test_matches_the_definition(cuda, M, K, dtype, act):
    g = torch.Generator(device=cuda).manual_seed(M * 7 + K)
    x = torch.randn(M, K * (2 if act == "silu_mul" else 1), generator=g, device=cuda).to(DTYPES[dtype])
    _check(x, act)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_plain_codes_equal_f32_arithmetic(cuda, dtype):
    """Without an activation every step is one IEEE operation: codes and scales bit for bit."""
    g = torch.Generator(device=cuda).manual_seed(5)
    x = torch.randn(40, 2688, generator=g, device=cuda).to(DTYPES[dtype])
    x[3] = 0
    x[4, 1:] = 0
    x[5, 7] = x[5].abs().amax() * 64  # an outlier channel
    q, s = ops.quant_s8(x)
    xf = np_(x.float())
    amax = np.abs(xf).max(1)
    want = np.where(amax > 0, amax / np.float32(127), np.float32(1)).astype(np.float32)
    assert np.array_equal(np_(s), want)
    assert np.array_equal(np_(q), np.clip(np.rint(xf / want[:, None]), -127, 127).astype(np.int8))


def test_far_gates_and_type_limits(cuda):
    """Gates far below zero give zero, not NaN; the lowest finite values of a type are values."""
    for dt in DTYPES.values():
        x = torch.zeros(4, 64, dtype=dt, device=cuda)
        x[0, :32], x[0, 32:] = -100.0, 3.0          # exp(100) overflows f32
        x[0, 1], x[0, 33] = 2.0, 1.0
        x[1, :32], x[1, 32:] = torch.finfo(dt).min, 1.0
        x[2, :32], x[2, 32:] = 30.0, 0.5
        q, s = ops.quant_s8(x, "silu_mul")
        assert q[0, 1] == 127 and int(q[0].abs().sum()) == 127
        assert not q[1].any() and float(s[1]) == 1.0
        assert torch.all(q[2] == 127)
        assert not q[3].any() and float(s[3]) == 1.0


def test_rows_with_nan_or_infinity(cuda):
    x = torch.randn(5, 256, device=cuda)
    x[1, 17] = float("nan")
    x[2, 255] = float("-inf")
    x[3, 0], x[3, 1] = float("inf"), float("nan")
    q, s = ops.quant_s8(x)
    assert torch.isnan(s[1]) and torch.isinf(s[2]) and torch.isnan(s[3])
    assert not q[1:4].any()
    q0, s0 = ops.quant_s8(x[[0, 4]].contiguous())
    assert torch.equal(q[[0, 4]], q0) and torch.equal(s[[0, 4]], s0)


@pytest.mark.parametrize("size", [1e-45, 1e-41, 1e-38, 3e-36, 1e-29, 1e-20, 3e38])
def test_tiny_and_huge_rows_equal_f32_arithmetic(cuda, size):
    """Scales down to the smallest subnormals (a scale that rounds to 0 becomes 1) and near the largest."""
    g = torch.Generator(device=cuda).manual_seed(3)
    x = (torch.rand(8, 512, generator=g, device=cuda) * 2 - 1) * size
    x[:, ::7] *= 0.5
    q, s = ops.quant_s8(x)
    xf = np_(x)
    amax = np.abs(xf).max(1)
    want = (amax / np.float32(127)).astype(np.float32)
    want = np.where(want > 0, want, np.float32(1)).astype(np.float32)
    assert np.array_equal(np_(s), want)
    ref = np.clip(np.rint((xf / want[:, None]).astype(np.float32)), -127, 127)
    assert np.array_equal(np_(q).astype(np.float32), ref)


def test_scales_of_a_few_units_clamp_the_codes(cuda):
    """A scale of k units in the last place of the subnormals is off by up to half a unit, so max / scale
    passes 127 (190 at k = 1): such codes are 127."""
    k = np.arange(1, 160)[:, None]
    units = np.concatenate([127 * k + 63, -(127 * k + 60), 64 * k, 127 * k, np.repeat(k, 12, 1)], 1).astype(np.uint32)
    sign = np.zeros_like(units)
    units[:, 1], sign[:, 1] = 127 * k[:, 0] + 60, 1
    xf = np.ascontiguousarray(units | sign << np.uint32(31)).view(np.float32)
    q, s = ops.quant_s8(torch.from_numpy(xf).to(cuda))
    want = (np.abs(xf).max(1) / np.float32(127)).astype(np.float32)
    assert np.array_equal(np_(s), want)
    assert np.array_equal(np_(q), np.clip(np.rint((xf / want[:, None]).astype(np.float32)), -127, 127).astype(np.int8))


def test_halves_of_the_maximum_round_to_even(cuda):
    """x = max / 2 is a tie in real arithmetic (63.5): decided as y / s rounds in f32."""
    for dt in DTYPES.values():
        a = torch.linspace(0.5, 8.0, 64, device=cuda).to(dt)
        x = (a[:, None].float() * torch.tensor([1.0, 0.5, -0.5, 0.25, 1 / 3] + [0.0] * 11, device=cuda)).to(dt)
        q, s = ops.quant_s8(x)
        xf = np_(x.float())
        want = (np.abs(xf).max(1) / np.float32(127)).astype(np.float32)
        assert np.array_equal(np_(q), np.rint((xf / want[:, None]).astype(np.float32)).astype(np.int8))


def test_no_rows_and_other_stream(cuda):
    q, s = ops.quant_s8(torch.empty(0, 64, dtype=torch.bfloat16, device=cuda), "silu_mul")
    assert q.shape == (0, 32) and s.shape == (0,)
    side = torch.cuda.Stream()
    x = torch.randn(64, 2048, device=cuda)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        y = x * 2
        q, s = ops.quant_s8(y)
    side.synchronize()
    q0, s0 = ops.quant_s8(x * 2)
    assert torch.equal(q, q0) and torch.equal(s, s0)
