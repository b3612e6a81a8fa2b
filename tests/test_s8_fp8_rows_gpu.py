"""The fp8 form of the grouped s8 GEMM casts the rows that the product wrote and no others; calls
with no rows."""
import numpy as np
import pytest
import torch

import oracle as O
from tests._util import np_
from xe2x2_b200 import ops

pytestmark = pytest.mark.gpu


def _setup(E=4, R=60, N=130, K=128):
    g = torch.Generator(device="cuda").manual_seed(3)
    s8 = lambda *shape: torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8)  # noqa: E731
    return (s8(R, K), torch.rand(R, generator=g, device="cuda"), s8(E, N, K),
            torch.rand(E, N, generator=g, device="cuda") * 1e-3)


# offsets, and the first row and the one behind the last that some expert has once they are made ascending
@pytest.mark.parametrize("offsets,first,end", [
    ([0, 10, 10, 45, 60], 0, 60),
    ([7, 10, 10, 45, 50], 7, 50),       # one shard's part of a longer batch
    ([0, 30, 12, 40, 25], 0, 40),       # out of order: expert 1 has none, expert 3 none
    ([-5, 20, 1 << 30, 3, -9], 0, 60),
    ([50, 20, 10, 5, 1], 50, 50),       # nothing left
    ([0, 0, 0, 0, 0], 0, 0),
])
@pytest.mark.parametrize("gather", [False, True])
def test_fp8_rows_are_those_of_the_product(cuda, offsets, first, end, gather):
    a, sa, w, sw = _setup()
    R, N = a.shape[0], w.shape[1]
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda)
    rows = torch.arange(R - 1, -1, -1, dtype=torch.int32, device=cuda) if gather else None
    y = torch.full((R, N), 5.0, device=cuda)
    ops.s8_gemm_grouped(a, sa, w, sw, off, rows, out=y)
    assert (y[:first] == 5).all() and (y[end:] == 5).all()
    q = torch.full((R, N), 2.0, device=cuda).to(torch.float8_e4m3fn)
    _, s = ops.s8_gemm_grouped(a, sa, w, sw, off, rows, out=q)
    assert (q[:first].float() == 2).all() and (q[end:].float() == 2).all()
    if end > first:
        q_ref, s_ref = O.rowscale_fp8(np_(y[first:end]))
        assert np.array_equal(np_(q.view(torch.uint8))[first:end], q_ref)
        assert np.array_equal(np_(s)[first:end], s_ref)


def test_no_rows_are_gathered_from_some_tokens(cuda):
    a, sa, w, sw = _setup()
    off = torch.zeros(5, dtype=torch.int32, device=cuda)
    none = torch.empty(0, dtype=torch.int32, device=cuda)
    assert ops.s8_gemm_grouped(a, sa, w, sw, off, none).shape == (0, 130)
    q, s = ops.s8_gemm_grouped(a, sa, w, sw, off, none, out_dtype=torch.float8_e4m3fn)
    assert q.shape == (0, 130) and s.shape == (0,)


def test_a_layer_without_tokens(cuda):
    _, _, w, sw = _setup(4, 1, 256, 128)
    wo, so = w.transpose(1, 2).contiguous()[:, :, :128].contiguous(), torch.ones(4, 128, device=cuda)
    lay = ops.S8Experts(w, sw, wo, so, top_k=2)
    assert lay(torch.empty(0, 128, device=cuda), torch.empty(0, 4, device=cuda)).shape == (0, 128)
    assert ops.S8Linear(w[0], sw[0])(torch.empty(0, 128, device=cuda)).shape == (0, 256)
