"""Gathered token rows in tiles of two CTAs: one CTA's threads copy rows that the other one's MMAs read.
Every call gives the bits of the call on rows that were gathered beforehand, with other tokens in
the same buffers from call to call, so that a stage read too early would show."""
import numpy as np
import pytest
import torch

from xe2x2_b200 import _lib as L
from xe2x2_b200 import ops

pytestmark = pytest.mark.gpu


def _s8(shape, g):
    return torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8)


# more than 128 rows for an expert on average over two, and more than 128 channels: tiles of pairs
@pytest.mark.parametrize("counts,N,K", [
    ([300, 256, 1, 340], 400, 2688),      # a tail of a row: all of it in the first CTA
    ([257, 0, 512, 288], 129, 16),        # one block of k, odd channels; tails of 1 and 32 rows
    ([1000, 7, 33, 130], 512, 1040),      # k ends inside a block
    ([700], 1856, 640),
    ([513, 255, 129, 300, 271, 64, 500, 90], 300, 2064),
])
def test_gathered_pairs_equal_copied_rows(cuda, counts, N, K):
    g = torch.Generator(device="cuda").manual_seed(N + K)
    E, off = len(counts), [0] + list(np.cumsum(counts))
    R, T = int(off[-1]), 600
    assert 2 * R // E > 128
    w = _s8((E, N, K), g)
    sw = torch.rand(E, N, generator=g, device=cuda) * 1e-3
    offsets = torch.tensor(off, dtype=torch.int32, device=cuda)
    a = torch.empty(T, K, dtype=torch.int8, device=cuda)
    rows = torch.empty(R, dtype=torch.int32, device=cuda)
    for turn in range(12):
        a.copy_(_s8((T, K), g))
        sa = torch.rand(T, generator=g, device=cuda)
        rows.copy_(torch.randint(0, T, (R,), generator=g, device=cuda, dtype=torch.int32))
        y = [ops.s8_gemm_grouped(a, sa, w, sw, offsets, rows, out_dtype=torch.float32) for _ in range(3)]
        src = rows.long()
        copied = ops.s8_gemm_grouped(a[src], sa[src], w, sw, offsets, out_dtype=torch.float32)
        assert all(torch.equal(v, copied) for v in y), turn
    e = int(np.argmax(counts))
    i, j = off[e], off[e + 1]
    acc = a[src[i:j]].double() @ w[e].double().t() * sa[src[i:j]].double()[:, None] * sw[e].double()
    # the sum, the product with the token's scale and the one with the channel's round once each
    assert bool(((copied[i:j].double() - acc).abs() <= 3.01 * 2.0 ** -24 * acc.abs() + 1e-38).all())
    assert L.lib().w4_check_device_status() == L.W4_OK
