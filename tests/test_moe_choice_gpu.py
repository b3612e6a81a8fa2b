"""Choices of w4_moe_route that 32 bits cannot make alone: signed zeros, group sums that cancel, ties at
the last rank, scores far below the largest.  Every id against the definition in 64 bits."""
import pytest
import torch

from xe2x2_b200 import ops

pytestmark = pytest.mark.gpu


def _ids64(x, k, bias=None, score="softmax", G=1, tg=1, group_score="max"):
    T, E = x.shape
    xd = x.double()
    p = torch.softmax(xd, 1) if score == "softmax" else torch.sigmoid(xd)
    key = xd if bias is None else p + bias.double()
    if G > 1:
        val = p if bias is None and group_score == "top2" else key
        best = val.view(T, G, E // G).sort(dim=2, descending=True).values
        total = best[:, :, 0] + (best[:, :, 1] if group_score == "top2" else 0)
        kept = total.sort(dim=1, descending=True, stable=True).indices[:, :tg]
        on = torch.zeros(T, G, dtype=torch.bool, device=x.device).scatter_(1, kept, True)
        key = key.masked_fill(~on.repeat_interleave(E // G, 1), -float("inf"))
    return key.sort(dim=1, descending=True, stable=True).indices[:, :k]


def _check(x, k, bias=None, score="softmax", G=1, tg=1, group_score="max"):
    want = _ids64(x, k, bias, score, G, tg, group_score)
    got = ops.moe_route(x, k, bias, score, n_group=G, topk_group=tg, group_score=group_score).ids.long()
    wrong = (got != want).any(1)
    assert not wrong.any(), (int(wrong.sum()), got[wrong][0].tolist(), want[wrong][0].tolist())


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------------------- signed zeros
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_minus_zero_ties_with_zero_under_tied_groups(cuda, score):
    x = torch.tensor([[-0.0, 0.0, -0.0, 0.0]], device=cuda)
    assert ops.moe_route(x, 1, score=score, n_group=2, topk_group=1, group_score="top2").ids.tolist() == [[0]]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_choices_among_mixed_zeros(cuda, dtype, score):
    """No logit above zero, a third of them -0: the choice reaches 0 and -0."""
    x = (torch.randint(-2, 1, (300, 64), generator=_gen(1), device=cuda) * 0.5).to(dtype)
    x[:, ::3] = -0.0
    zero = torch.zeros(64, device=cuda)
    for b in (None, zero):
        _check(x, 8, b, score)
        for gs in ("max", "top2"):
            _check(x, 8, b, score, 8, 3, gs)
            _check(x, 8, b, score, 4, 1, gs)


# ---------------------------------------------------------------------------- group sums that cancel
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("size", [64.0, 4096.0])
def test_groups_whose_two_best_cancel(cuda, size, score):
    """Biases near +size and -size on a group's two best: the sums are of the scores' size, their 32-bit
    errors of the biases'."""
    T, E, G = 50_000, 64, 8
    x = torch.randn(T, E, generator=_gen(2), device=cuda)
    bias = torch.full((E,), -3 * size, device=cuda)
    bias[1::8], bias[4::8] = size, -size
    for tg in (1, 3):
        _check(x, tg, bias, score, G, tg, "top2")


# ---------------------------------------------------------------------------- ties at the last rank
def test_a_tie_at_the_last_rank_does_not_hide_a_larger_score(cuda):
    """In 32 bits all three have the score 1; the two at 20 tie in any precision, the one at 21 is larger."""
    x = torch.full((1, 40), -3.0, device=cuda)
    x[0, 4] = x[0, 9] = 20.0
    x[0, 30] = 21.0
    zero = torch.zeros(40, device=cuda)
    assert ops.moe_route(x, 1, zero, "sigmoid").ids.tolist() == [[30]]
    x[0, 1] = 22.0
    assert ops.moe_route(x, 2, zero, "sigmoid").ids.tolist() == [[1, 30]]


@pytest.mark.parametrize("E", [48, 256, 480])
@pytest.mark.parametrize("k", [1, 2, 6, 31, 32])
def test_logits_on_a_grid_with_equal_scores_in_32_bits(cuda, E, k):
    x = 18 + torch.randint(0, 24, (400, E), generator=_gen(E + k), device=cuda) * 0.5
    zero = torch.zeros(E, device=cuda)
    _check(x, k, zero, "sigmoid")                       # within 2^-24 of 1, up to 1 - 6e-14
    _check(x.bfloat16(), k, zero, "sigmoid")
    half = torch.full((E,), 0.5, device=cuda)
    low = -38 + torch.randint(0, 30, (400, E), generator=_gen(k), device=cuda) * 0.5
    _check(low, k, half, "sigmoid")                     # lost in the sum with the bias
    low[:, 7] = 0.0
    _check(low, k, half, "softmax")
    if k <= 12:
        _check(x, k, zero, "sigmoid", 4, 2, "top2")
        _check(low, k, half, "softmax", 4, 2, "max")


# ---------------------------------------------------------------------------- scores far below the largest
@pytest.mark.parametrize("gap", [15.0, 30.0, 60.0, 82.0])
def test_softmax_scores_far_below_the_largest(cuda, gap):
    """One expert holds all of the sum; the others' scores, and biases of their size, lie as close as the
    rounding of exp's argument (gap * 2^-24 each time it is rounded)."""
    T, E, k = 40_000, 64, 8
    g = _gen(int(gap))
    x = -gap + 1.7 + 1e-3 * torch.rand(T, E, generator=g, device=cuda)
    x[:, 11] = 1.7 + torch.rand(T, generator=g, device=cuda)
    bias = torch.exp(torch.tensor(-gap, device=cuda)) * 5e-4 * torch.rand(E, generator=g, device=cuda)
    _check(x, k, bias, "softmax")
    _check(x, k, bias, "softmax", 4, 4, "max")
