"""w4_moe_route and w4_moe_combine against their definitions in 64 bits, token by token."""
import numpy as np
import pytest
import torch

from tests._util import np_
from xe2x2_b200 import ops

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
FMAX = float(np.finfo(np.float32).max)


def _route64(logits, bias, k, score, renorm, scaling, n_group, topk_group, group_score):
    x = np_(logits.double())
    T, E = x.shape
    ids, w = np.full((T, k), -1, np.int32), np.zeros((T, k))
    for t in range(T):
        row = np.where(np.isnan(x[t]), -np.inf, x[t])
        live = [e for e in range(E) if row[e] > -np.inf]
        p = np.zeros(E)
        c = np.minimum(row, FMAX)
        if live:
            if score == "softmax":
                p = np.exp(c - c[live].max())
                p /= p.sum()
            else:
                with np.errstate(over="ignore"):
                    p = 1 / (1 + np.exp(-c))
        key = row if bias is None else p + bias
        live = [e for e in live if key[e] > -np.inf]
        if n_group > 1:
            size = E // n_group
            val = p if bias is None and group_score == "top2" else key
            tot = []
            for g in range(n_group):
                best = sorted((val[e] for e in live if e // size == g), reverse=True)
                tot.append(sum(best[:2 if group_score == "top2" else 1]) if best else -np.inf)
            kept = sorted(range(n_group), key=lambda g: (-tot[g], g))[:topk_group]
            live = [e for e in live if e // size in kept]
        got = sorted(live, key=lambda e: (-key[e], e))[:k]
        v = p[got]
        if renorm:
            v = v / v.sum() if v.sum() > 0 else v * 0
        ids[t, :len(got)], w[t, :len(got)] = got, v * scaling
        if np.isnan(x[t]).any():
            w[t] = np.nan
    return ids, w


def _check_plan(r, ids, E):
    T, k = ids.shape
    taken = sorted((e, t, j) for t in range(T) for j, e in enumerate(ids[t]) if e >= 0)
    rows, slots = np.full(T * k, -1), np.full((T, k), -1)
    for i, (_, t, j) in enumerate(taken):
        rows[i], slots[t, j] = t, i
    counts = np.bincount(ids[ids >= 0].ravel(), minlength=E)
    assert np.array_equal(np_(r.offsets), np.concatenate([[0], np.cumsum(counts)]))
    assert np.array_equal(np_(r.rows), rows)
    assert np.array_equal(np_(r.slots), slots)


def _check(logits, k, bias=None, score="softmax", renormalize=True, scaling=1.0, n_group=1, topk_group=1,
           group_score="max"):
    b = None if bias is None else np_(bias.double())
    ids, w = _route64(logits, b, k, score, renormalize, scaling, n_group, topk_group, group_score)
    r = ops.moe_route(logits, k, bias, score, renormalize, scaling, n_group, topk_group, group_score)
    assert np.array_equal(np_(r.ids), ids)
    # In 32 bits: expf within 1 ulp (2^-23) of its argument, which rounds by at most |x| 2^-24 (x the
    # logit under the softmax's largest; logits here are below 32 in size where a weight counts), 1 + e and
    # the quotient (2^-24 each); the same again in the sum, plus its additions (5), and the last quotient,
    # the scaling and the store.  Without renormalising the softmax's sum has E terms of its own, with the
    # base-2 exponential (2^-22).
    E = logits.shape[1]
    rel = 2 * (2 * 32 * 2.0 ** -24 if score == "softmax" else 0) + 16 * 2.0 ** -24
    if not renormalize and score == "softmax":
        rel += 2.0 ** -22 + E * 2.0 ** -24
    got = np_(r.weights).astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(w))
    fine = ~np.isnan(w)
    assert np.all(np.abs(got - w)[fine] <= rel * np.abs(w[fine]) + 1e-38)
    _check_plan(r, ids, E)
    return r


def _logits(T, E, dtype, seed, cuda, sigma=1.5):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return (sigma * torch.randn(T, E, generator=g, device=cuda)).to(DTYPES[dtype])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (3, 33, 6), (64, 64, 6), (65, 60, 4), (200, 128, 8),
                                   (17, 512, 32), (700, 257, 3), (333, 32, 32)])
def test_softmax_and_sigmoid(cuda, T, E, k, dtype):
    x = _logits(T, E, dtype, T + E, cuda)
    _check(x, k)
    _check(x, k, score="sigmoid", scaling=2.5)
    _check(x, k, renormalize=False)
    bias = 0.2 * torch.randn(E, device=cuda, generator=torch.Generator(device=cuda).manual_seed(E))
    _check(x, k, bias, score="sigmoid")
    _check(x, k, bias, score="softmax", renormalize=False, scaling=0.5)


@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,G,tg", [(5, 64, 6, 8, 3), (300, 256, 8, 8, 4), (40, 60, 4, 3, 1), (33, 96, 8, 32, 9),
                                        (9, 512, 8, 2, 1), (21, 320, 8, 10, 10)])
def test_groups(cuda, T, E, k, G, tg, score, group_score):
    x = _logits(T, E, "f32", 3 * T + E, cuda)
    bias = 0.1 * torch.randn(E, device=cuda, generator=torch.Generator(device=cuda).manual_seed(E))
    for b in (None, bias):
        _check(x, k, b, score, n_group=G, topk_group=tg, group_score=group_score)
        _check(x.bfloat16(), k, b, score, False, 1.5, G, tg, group_score)


def test_ties_go_to_the_lower_index(cuda):
    """bf16 logits from a few values: many exact ties, across lanes and inside one; -0 ties with 0."""
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randint(-2, 3, (200, 256), generator=g, device=cuda).to(torch.bfloat16) * 0.5
    x[:, ::3] = -0.0
    zero = torch.zeros(256, device=cuda)
    for b in (None, zero):
        _check(x, 8, b)
        _check(x, 8, b, score="sigmoid", n_group=8, topk_group=3, group_score="top2")
    assert np.array_equal(np_(ops.moe_route(torch.zeros(2, 100, device=cuda), 5).ids), [[0, 1, 2, 3, 4]] * 2)


def test_near_ties_are_decided_in_64_bits(cuda):
    """Biases that bring two scores to within 1e-12 of each other, either way round."""
    T, E = 64, 64
    x = torch.full((T, E), -3.0, device=cuda)
    x[:, 10], x[:, 50] = 0.25, 0.75
    p10, p50 = 1 / (1 + np.exp(-0.25)), 1 / (1 + np.exp(-0.75))
    base = np.float32(p50 - p10)
    bias = torch.zeros(E, device=cuda)
    for step in (-1, 0, 1):
        bias[10] = float(np.nextafter(base, np.float32(step * 9)) if step else base)
        _check(x, 2, bias, score="sigmoid")
        _check(x, 1, bias, score="sigmoid", n_group=4, topk_group=1, group_score="top2")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_masked_experts_and_rows(cuda, score, with_bias):
    x = _logits(90, 40, "f32", 4, cuda)
    inf = float("inf")
    x[3] = -inf                       # a padded token
    x[:, 17] = -inf                   # an expert switched off
    x[5, 3:] = -inf                   # fewer experts than top_k
    x[6] = torch.finfo(torch.float32).min   # lowest values: all alike
    x[7, :39] = torch.finfo(torch.float32).min
    x[8, 4] = inf
    x[9, 4], x[9, 8] = inf, inf
    x[10, 0] = float("nan")
    x[11] = float("nan")
    x[12] = 1e30
    x[13] = -200.0
    x[70:] = -inf
    bias = 0.1 * torch.randn(40, device=cuda, generator=torch.Generator(device=cuda).manual_seed(2))
    bias[20], bias[21] = -inf, inf
    b = bias if with_bias else None
    for kw in (dict(), dict(n_group=8, topk_group=4), dict(n_group=8, topk_group=2, group_score="top2")):
        k = 6
        _check(x, k, b, score, **kw)
        _check(x, k, b, score, renormalize=False, **kw)
    r = ops.moe_route(x, 6, b, score)
    assert not (r.ids[70:] >= 0).any() and not r.weights[70:].any()
    assert torch.isnan(r.weights[10:12]).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_lowest_value_of_a_type_as_mask(cuda, dtype):
    x = _logits(40, 64, dtype, 8, cuda)
    x[:, 32:] = torch.finfo(DTYPES[dtype]).min
    r = _check(x, 8)
    assert (r.ids < 32).all()
    x[4] = torch.finfo(DTYPES[dtype]).min  # nothing but masked ones: values like any other
    r = _check(x, 8)
    assert r.ids[4].tolist() == list(range(8))


def test_no_tokens_and_many(cuda):
    r = ops.moe_route(torch.empty(0, 16, device=cuda), 2)
    assert r.ids.shape == (0, 2) and r.offsets.tolist() == [0] * 17
    # chunks at their largest, and a last one with a single token
    x = _logits(148 * 64 + 1, 16, "bf16", 6, cuda)
    _check(x, 2)


def test_many_tokens_in_capped_chunks(cuda):
    """More tokens than 1024 for each SM: counts still add up (checked with torch's sort)."""
    x = _logits(170001, 32, "bf16", 7, cuda)
    r = ops.moe_route(x, 4)
    ids = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(r.ids.long(), ids)
    order = torch.sort(ids.reshape(-1), stable=True).indices
    assert torch.equal(r.rows.long(), order // 4)
    back = torch.empty_like(order)
    back[order] = torch.arange(order.numel(), device=cuda)
    assert torch.equal(r.slots.long().reshape(-1), back)
    assert torch.equal(r.offsets[1:].long(), torch.cumsum(torch.bincount(ids.reshape(-1), minlength=32), 0))


def test_route_without_a_plan(cuda):
    """The C entry point takes ids and weights alone."""
    import ctypes
    from xe2x2_b200 import _lib as L
    x = _logits(500, 64, "f32", 9, cuda)
    r = ops.moe_route(x, 4)
    ids, w = torch.empty_like(r.ids), torch.empty_like(r.weights)
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    L.call("w4_moe_route", p(x), L.W4_F32, None, 500, 64, 4, L.W4_SCORE_SOFTMAX, 1, 1, L.W4_GROUP_MAX, 1, 1.0, p(ids),
           p(w), None, None, None, None, 0, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert torch.equal(ids, r.ids) and torch.equal(w, r.weights)


@pytest.mark.parametrize("T", [7, 900])
def test_route_replayed_from_a_graph(cuda, T):
    x = _logits(T, 128, "f32", 10, cuda)
    bias = torch.zeros(128, device=cuda)
    ops.moe_route(x, 8, bias, "sigmoid")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = ops.moe_route(x, 8, bias, "sigmoid")
    for seed in (11, 12):
        x.copy_(_logits(T, 128, "f32", seed, cuda))
        want = ops.moe_route(x, 8, bias, "sigmoid")
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(r, want))


# ------------------------------------------------------------------------------------- combine
@pytest.mark.parametrize("ydt", list(DTYPES))
@pytest.mark.parametrize("odt", list(DTYPES))
@pytest.mark.parametrize("T,k,H,with_add", [(1, 1, 1, False), (1, 6, 2688, True), (5, 8, 333, True), (64, 2, 4096, False),
                                            (3, 32, 72, True), (130, 3, 1032, False)])
def test_combine(cuda, T, k, H, with_add, ydt, odt):
    g = torch.Generator(device=cuda).manual_seed(T + H)
    R = T * k + 3
    y = torch.randn(R, H, generator=g, device=cuda).to(DTYPES[ydt])
    slots = torch.randperm(R, generator=g, device=cuda)[:T * k].view(T, k).to(torch.int32)
    w = torch.rand(T, k, generator=g, device=cuda)
    if T > 1:
        slots[1, 0], slots[0, k - 1] = -1, R + 5  # no such row
    if T > 2:
        slots[2] = -1
    add = torch.randn(T, H, generator=g, device=cuda).to(DTYPES[odt]) if with_add else None
    out = ops.moe_combine(y, slots, w, add, DTYPES[odt])
    yd, wd, sd = np_(y.double()), np_(w.double()), np_(slots)
    ref, mag = np.zeros((T, H)), np.zeros((T, H))
    if with_add:
        ref, mag = np_(add.double()).copy(), np.abs(np_(add.double()))
    for t in range(T):
        for j in range(k):
            if 0 <= sd[t, j] < R:
                ref[t] += wd[t, j] * yd[sd[t, j]]
                mag[t] += wd[t, j] * np.abs(yd[sd[t, j]])
    # k fused multiply-adds round once each on sums below mag; the store rounds by half a step
    tol = k * 2.0 ** -24 * mag * 1.01 + torch.finfo(DTYPES[odt]).eps / 2 * np.abs(ref) * 1.01 + 1e-7
    assert np.all(np.abs(np_(out.double()) - ref) <= tol)


def test_combine_ignores_what_no_slot_names(cuda):
    """Rows that nothing points at (behind the last expert's) may hold anything."""
    y = torch.randn(10, 64, device=cuda)
    y[7:] = float("nan")
    slots = torch.tensor([[0, 6], [-1, 3]], dtype=torch.int32, device=cuda)
    w = torch.tensor([[0.5, 0.5], [0.0, 1.0]], device=cuda)
    out = ops.moe_combine(y, slots, w)
    assert torch.equal(out[1], y[3]) and torch.isfinite(out).all()
    w[1, 0] = float("nan")  # a token whose logits were NaN stays visible
    assert torch.isnan(ops.moe_combine(y, slots, w)[1]).all()
    assert ops.moe_combine(y, slots[:0], w[:0]).shape == (0, 64)


# ------------------------------------------------------------------------------------- many tokens
@pytest.mark.parametrize("score,G,tg,group_score", [("sigmoid", 1, 1, "max"), ("sigmoid", 8, 4, "top2"),
                                                    ("softmax", 1, 1, "max"), ("softmax", 8, 3, "max"),
                                                    ("softmax", 4, 2, "top2")])
@pytest.mark.parametrize("E", [256, 96])
def test_every_choice_of_many_tokens_is_the_64_bit_one(cuda, E, score, G, tg, group_score):
    """Among 200,000 tokens hundreds have neighbours that 32 bits cannot tell apart."""
    T, k = 200_000, 8
    x = _logits(T, E, "f32", E + G, cuda)
    bias = 0.1 * torch.randn(E, device=cuda, generator=torch.Generator(device=cuda).manual_seed(7))
    r = ops.moe_route(x, k, bias, score, n_group=G, topk_group=tg, group_score=group_score)
    xd = x.double()
    p = torch.softmax(xd, 1) if score == "softmax" else torch.sigmoid(xd)
    key = p + bias.double()
    if G > 1:
        best = key.view(T, G, E // G).topk(2, dim=2).values
        tot = best[:, :, 0] + (best[:, :, 1] if group_score == "top2" else 0)
        kept = torch.zeros(T, G, dtype=torch.bool, device=cuda).scatter_(1, tot.topk(tg, dim=1).indices, True)
        key = key.masked_fill(~kept.repeat_interleave(E // G, 1), -float("inf"))
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(r.ids.long(), ids)
    w = p.gather(1, ids)
    w = w / w.sum(1, keepdim=True)
    assert float(((r.weights.double() - w) / w).abs().max()) < 1e-5


def test_threads_with_calls_of_different_sizes(cuda):
    """Calls that take much and little shared memory, from threads at once, do not refuse each other."""
    from concurrent.futures import ThreadPoolExecutor

    g = torch.Generator(device=cuda).manual_seed(8)
    big = torch.randn(40000, 480, generator=g, device=cuda)     # 32 groups of 15: masks and scratch
    small = torch.randn(3000, 480, generator=g, device=cuda)
    calls = [(big, 8), (small, 8), (small, 4), (big, 2)]
    torch.cuda.synchronize()

    def run(logits, k):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            for _ in range(50):
                r = ops.moe_route(logits, k, score="sigmoid", n_group=32, topk_group=5, group_score="top2")
        side.synchronize()
        return r

    want = [run(*c) for c in calls]
    with ThreadPoolExecutor(4) as pool:
        got = list(pool.map(lambda c: run(*c), calls))
    for r, w in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(r, w))
