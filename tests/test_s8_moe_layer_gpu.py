"""The 8-bit MoE layer as it is used: router -> quantiser -> experts' products -> combine in one
object (ops.S8Experts), eagerly, on another stream and replayed from a CUDA graph; the router
feeding the 4-bit grouped GEMMs; the RMSNorm producer feeding the s8 GEMM."""
import numpy as np
import pytest
import torch

from tests._util import np_
from xe2x2_b200 import _lib as L
from xe2x2_b200 import ops, synth

pytestmark = pytest.mark.gpu


def _weights(shape, g):
    w = torch.randn(shape, generator=g, device="cuda") / shape[-1] ** 0.5
    s = w.abs().amax(-1) / 127
    return torch.round(w / s[..., None]).to(torch.int8), s


def _layer(E, H, I, act, k, seed, **route):
    g = torch.Generator(device="cuda").manual_seed(seed)
    F = 2 * I if act == "silu_mul" else I
    return ops.S8Experts(*_weights((E, F, H), g), *_weights((E, H, I), g), top_k=k, act=act, **route)


def _float_layer(lay, x, logits, add):
    """The same layer on unquantised activations, in 64 bits, token by token."""
    r = ops.moe_route(logits, lay.top_k, **lay.route)
    ids, w = np_(r.ids), np_(r.weights.double())
    out = np.zeros(x.shape) if add is None else np_(add.double()).copy()
    for t in range(x.shape[0]):
        for j, e in enumerate(ids[t]):
            if e < 0:
                continue
            h = (lay.w_in[e].double() @ x[t].double()) * lay.in_scale[e].double()
            if lay.act == "silu_mul":
                gate, up = h.chunk(2)
                h = torch.nn.functional.silu(gate) * up
            else:
                h = h.clamp(min=0) ** 2
            out[t] += w[t, j] * np_((lay.w_out[e].double() @ h) * lay.out_scale[e].double())
    return out


@pytest.mark.parametrize("act", ["silu_mul", "relu2"])
@pytest.mark.parametrize("T", [1, 5, 70])
def test_layer_is_near_the_unquantised_one(cuda, T, act):
    """An 8-bit step is amax / 127, so a row's error is amax / (127 sqrt(12)) a value: about 0.8 % of
    the rms for the states (amax about 3.5 rms) and about 2.5 % for the activated ones (heavy tails,
    amax up to 11 rms); with the slope of the activation at most 2 that adds up to 4 %, and 5 % is
    allowed."""
    lay = _layer(16, 512, 384, act, 4, 3, score="sigmoid", scaling=1.5)
    g = torch.Generator(device=cuda).manual_seed(T)
    x = torch.randn(T, 512, generator=g, device=cuda).bfloat16()
    logits = torch.randn(T, 16, generator=g, device=cuda)
    add = torch.randn(T, 512, generator=g, device=cuda).bfloat16()
    if T > 4:
        logits[3] = -float("inf")  # padding
    got = np_(lay(x, logits, add).double())
    ref = _float_layer(lay, x, logits, add)
    base = np_(add.double())
    err = np.linalg.norm(got - ref) / np.linalg.norm(ref - base)
    assert err < 0.05, err
    if T > 4:
        assert np.array_equal(got[3], base[3])
    assert L.lib().w4_check_device_status() == L.W4_OK


def test_layer_equals_its_steps_and_token_order_does_not_matter(cuda):
    lay = _layer(32, 256, 128, "silu_mul", 6, 4, score="sigmoid", n_group=4, topk_group=2, group_score="top2")
    g = torch.Generator(device=cuda).manual_seed(9)
    x = torch.randn(90, 256, generator=g, device=cuda).half()
    logits = torch.randn(90, 32, generator=g, device=cuda).half()
    y = lay(x, logits)
    r = ops.moe_route(logits, 6, score="sigmoid", n_group=4, topk_group=2, group_score="top2")
    q, s = ops.quant_s8(x)
    h = ops.s8_gemm_grouped(q, s, lay.w_in, lay.in_scale, r.offsets, r.rows, out_dtype=torch.float16)
    q, s = ops.quant_s8(h, "silu_mul")
    z = ops.s8_gemm_grouped(q, s, lay.w_out, lay.out_scale, r.offsets, out_dtype=torch.float16)
    assert torch.equal(y, ops.moe_combine(z, r.slots, r.weights))
    # every token's own arithmetic is the same wherever it stands in whatever batch
    p = torch.randperm(90, generator=g, device=cuda)
    assert torch.equal(lay(x[p], logits[p]), y[p])
    assert torch.equal(lay(x[:1], logits[:1]), y[:1])


@pytest.mark.parametrize("T", [4, 200])
def test_layer_in_a_graph_beside_an_eager_one(cuda, T):
    """Two captured layers (one stream each) replayed at once beside eager calls: no scratch is shared."""
    lay = [_layer(16, 256, 128, "silu_mul", 4, 5 + i, score="sigmoid") for i in range(2)]
    bias = torch.zeros(16, device=cuda)
    for la in lay:
        la.route["bias"] = bias
    x = [torch.empty(T, 256, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    lg = [torch.empty(T, 16, device=cuda) for _ in range(2)]

    def fill(seed):
        g = torch.Generator(device=cuda).manual_seed(seed)
        for i in range(2):
            x[i].copy_(torch.randn(T, 256, generator=g, device=cuda))
            lg[i].copy_(torch.randn(T, 16, generator=g, device=cuda))

    fill(0)
    for i in range(2):
        lay[i](x[i], lg[i])
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(lay[i](x[i], lg[i]))
        graphs.append(gr)
    for seed in (1, 2, 3):
        fill(seed)
        want = [lay[i](x[i], lg[i]) for i in range(2)]
        torch.cuda.synchronize()
        for _ in range(4):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
            eager = lay[0](x[0], lg[0])
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0])
        for i in range(2):
            assert torch.equal(outs[i], want[i])


def test_router_feeds_the_4_bit_grouped_gemms(cuda):
    """offsets.tolist() and rows are what the GPTQ grouped GEMM takes."""
    E, H, N, T, k = 8, 256, 128, 20, 2
    ws = [synth.gptq_weights(H, N, 128, asym=True, seed=e, device="cuda")[:3] for e in range(E)]
    qw, qz, sc = (torch.stack([w[i] for w in ws]).contiguous() for i in range(3))
    x = synth.activations(T, H, torch.bfloat16, seed=3, device="cuda")
    r = ops.moe_route(torch.randn(T, E, device="cuda"), k)
    y = ops.gptq_gemm_grouped(x[r.rows.long()], qw, qz, sc, r.offsets.tolist(), 128, 1, torch.float32)
    out = ops.moe_combine(y, r.slots, r.weights)
    ref = torch.zeros(T, N, dtype=torch.float64, device="cuda")
    for t in range(T):
        for j in range(k):
            e = int(r.ids[t, j])
            one = ops.gptq_gemm(x[t:t + 1], qw[e], qz[e], sc[e], 128, 1, out_dtype=torch.float32)
            ref[t] += float(r.weights[t, j]) * one[0].double()
    assert float((out.double() - ref).norm() / ref.norm()) < 1e-4  # f32 sums in another order


def test_s8_linear_behind_the_norm_and_by_itself(cuda):
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn(40, 512, generator=g, device=cuda).half()
    w, ws = _weights((300, 512), g)
    q, s = ops.rmsnorm_quant_s8(x)
    y = ops.s8_gemm(q, s, w, ws, out_dtype=torch.float32)
    ref = (q.double() * s.double()[:, None]) @ (w.double() * ws.double()[:, None]).t()
    assert float((y.double() - ref).abs().max() / ref.abs().max()) < 1e-6
    lin = ops.S8Linear(w, ws, torch.ones(300, device=cuda))
    q, s = ops.quant_s8(x)
    assert torch.equal(lin(x), ops.s8_gemm(q, s, w, ws, torch.ones(300, device=cuda), torch.float16))
    assert lin(x, torch.float32).dtype == torch.float32
