"""The 8-bit operators where indices pass 32 bits, on two streams at once, under every launch overlap
mode, and refused views."""
import pytest
import torch

from xe2x2_b200 import _lib as L
from xe2x2_b200 import ops

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _s8(shape, g):
    return torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8)


def _free():
    torch.cuda.empty_cache()


def test_gemm_output_past_2_31_elements(cuda):
    g = _gen(1)
    M, N, K = 70001, 32768, 48
    a, w = _s8((M, K), g), _s8((N, K), g)
    sa, sw = torch.rand(M, generator=g, device=cuda), torch.rand(N, generator=g, device=cuda)
    y = ops.s8_gemm(a, sa, w, sw)
    assert y.numel() > 2 ** 31
    for i in (0, 1, 65535, 65536, M - 1):
        ref = (a[i].double() @ w.double().t()) * sa[i].double() * sw.double()
        assert float((y[i].double() - ref).abs().max() / ref.abs().max()) < 2 ** -8
    del y
    _free()


def test_quant_and_combine_past_2_31_elements(cuda):
    g = _gen(2)
    M, K = 140003, 16384
    x = torch.empty(M, K, dtype=torch.bfloat16, device=cuda).normal_(generator=g)
    assert x.numel() > 2 ** 31
    q, s = ops.quant_s8(x)
    for i in (0, 131072, M - 1):
        q1, s1 = ops.quant_s8(x[i:i + 1].clone())
        assert torch.equal(q[i], q1[0]) and torch.equal(s[i], s1[0])
    slots = torch.tensor([[0, M - 1], [131072, -1]], dtype=torch.int32, device=cuda)
    wt = torch.tensor([[0.25, 0.5], [1.0, 0.0]], device=cuda)
    out = ops.moe_combine(x, slots, wt, out_dtype=torch.float32)
    assert torch.equal(out[1], x[131072].float())
    assert torch.equal(out[0], 0.25 * x[0].float() + 0.5 * x[M - 1].float())
    del x, q, out
    _free()


def test_grouped_weights_and_tokens_past_2_31_bytes(cuda):
    """Experts and gathered rows whose byte offsets pass 2^31."""
    g = _gen(3)
    E, N, K = 4, 40000, 16384          # 2.6 GB of weights
    w = _s8((E, N, K), g)
    sw = torch.rand(E, N, generator=g, device=cuda)
    T = 140003                          # 2.3 GB of tokens
    a = _s8((T, K), g)
    sa = torch.rand(T, generator=g, device=cuda)
    rows = torch.tensor([5, T - 1, 0, 131073, T - 2], dtype=torch.int32, device=cuda)
    offsets = torch.tensor([0, 1, 1, 2, 5], dtype=torch.int32, device=cuda)
    y = ops.s8_gemm_grouped(a, sa, w, sw, offsets, rows, out_dtype=torch.float32)
    for r, e in ((0, 0), (1, 2), (2, 3), (3, 3), (4, 3)):
        t = int(rows[r])
        acc = (w[e].double() @ a[t].double()) * sa[t].double() * sw[e].double()
        assert float((y[r].double() - acc).abs().max() / acc.abs().max()) < 1e-6
    assert L.lib().w4_check_device_status() == L.W4_OK
    del w, a
    _free()


@pytest.mark.parametrize("M,N,K", [(1, 640, 4096), (200, 512, 4096), (700, 512, 1024)])
def test_two_streams_at_once(cuda, M, N, K):
    """Calls that overlap on the GPU share nothing: the fp8 form's scratch is the call's own too."""
    g = _gen(4)
    a = [_s8((M, K), g) for _ in range(2)]
    w = [_s8((N, K), g) for _ in range(2)]
    sa, sw = torch.rand(M, generator=g, device=cuda), torch.rand(N, generator=g, device=cuda)
    want = [ops.s8_gemm(a[i], sa, w[i], sw, out_dtype=torch.float8_e4m3fn) for i in range(2)]
    torch.cuda.synchronize()
    st = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(st[i]):
                got[i].append(ops.s8_gemm(a[i], sa, w[i], sw, out_dtype=torch.float8_e4m3fn))
    torch.cuda.synchronize()
    for i in range(2):
        for q, s in got[i]:
            assert torch.equal(q.view(torch.uint8), want[i][0].view(torch.uint8)) and torch.equal(s, want[i][1])


def test_chains_are_ordered_under_every_overlap_mode(cuda):
    """Each kernel reads what the one launched just before it wrote; the modes give the same bits."""
    g = _gen(5)
    E, H, I, T = 8, 256, 128, 24
    wi, wo = _s8((E, 2 * I, H), g), _s8((E, H, I), g)
    si = torch.rand(E, 2 * I, generator=g, device=cuda) * 1e-3
    so = torch.rand(E, H, generator=g, device=cuda) * 1e-3
    lay = ops.S8Experts(wi, si, wo, so, top_k=2)
    router = torch.randn(H, E, generator=g, device=cuda).bfloat16()
    x0 = torch.randn(T, H, generator=g, device=cuda).bfloat16()
    old, outs = L.lib().w4_get_launch_overlap(), []
    try:
        for mode in (L.W4_OVERLAP_OFF, L.W4_OVERLAP_DEPENDENT, L.W4_OVERLAP_STATIC_WEIGHTS):
            L.call("w4_set_launch_overlap", mode)
            x = x0
            for _ in range(6):
                x = lay(x, x @ router, x)
                x = x / x.float().abs().amax().to(x.dtype)
            outs.append(x)
    finally:
        L.call("w4_set_launch_overlap", old)
    assert torch.isfinite(outs[0]).all()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_views_that_are_refused(cuda):
    g = _gen(6)
    a, w = _s8((8, 64), g), _s8((32, 64), g)
    sa, sw = torch.ones(8, device=cuda), torch.ones(32, device=cuda)
    with pytest.raises(ValueError, match="contiguous"):
        ops.s8_gemm(_s8((64, 8), g).t(), sa, w, sw)
    with pytest.raises(ValueError, match="contiguous"):
        ops.quant_s8(torch.randn(8, 128, device=cuda)[:, :64])
    with pytest.raises(ValueError, match="float32"):
        ops.s8_gemm(a, sa.half(), w, sw)
    with pytest.raises(ValueError, match=r"\[8\]"):
        ops.s8_gemm(a, sa[:7], w, sw)
    with pytest.raises(ValueError, match="out"):
        ops.s8_gemm(a, sa, w, sw, out=torch.empty(8, 31, device=cuda))
    off = torch.empty(8 * 64 + 8, dtype=torch.int8, device=cuda)[8:].view(8, 64)  # 8 bytes off
    with pytest.raises(L.W4Error, match="aligned"):
        ops.s8_gemm(off, sa, w, sw)
    with pytest.raises(L.W4Error, match="multiple of 16"):
        ops.s8_gemm(a[:, :24].contiguous(), sa, w[:, :24].contiguous(), sw)
    with pytest.raises(ValueError, match="int32"):
        ops.s8_gemm_grouped(a, sa, w.view(1, 32, 64), sw.view(1, 32), torch.tensor([0, 8], device=cuda))
    with pytest.raises(ValueError, match="cpu|CUDA"):
        ops.s8_gemm(a, sa, w, sw.cpu())
    with pytest.raises(ValueError, match="int32"):
        ops.moe_combine(torch.randn(4, 8, device=cuda), torch.zeros(2, 2, device=cuda), torch.ones(2, 2, device=cuda))


def test_results_land_at_unaligned_outputs(cuda):
    """Outputs that cannot be stored in pairs or fours: odd N, views that start in the middle."""
    g = _gen(7)
    for N in (63, 66, 129):
        a, w = _s8((40, 96), g), _s8((N, 96), g)
        sa, sw = torch.rand(40, generator=g, device=cuda), torch.rand(N, generator=g, device=cuda)
        want = ops.s8_gemm(a, sa, w, sw, out_dtype=torch.float16)
        for skip in (1, 2, 3):
            buf = torch.zeros(40 * N + 8, dtype=torch.float16, device=cuda)
            out = buf[skip:skip + 40 * N].view(40, N)
            ops.s8_gemm(a, sa, w, sw, out=out)
            assert torch.equal(out, want) and not buf[:skip].any() and not buf[skip + 40 * N:].any()
