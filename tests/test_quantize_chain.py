"""The row passes as producers of the fused products, run back to back with new inputs and no pause between calls.

Every step's results are compared with the formula on the codes, scales and residual stream that this step produced, so a
product that read what an earlier step had left anywhere shows up.  u = 2^-24.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
STEPS = 12


def steps_of(cuda, x, others, call, outputs):
    """call() for STEPS inputs without a pause, then for the same inputs with one; the outputs of each, cloned."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    fresh = [[torch.randn(t.shape, device=cuda, generator=gen).to(t.dtype) for t in (x, *others)] for _ in range(STEPS)]

    def all_of(wait):
        got = []
        for new in fresh:
            for t, v in zip((x, *others), new):
                t.copy_(v)
            call()
            got.append([t.clone() for t in outputs])
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return got

    eager = all_of(False)
    for one, other in zip(eager, all_of(True)):
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(one, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for new, want in zip(fresh, eager):
        for t, v in zip((x, *others), new):
            t.copy_(v)
        graph.replay()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(outputs, want))
    return eager


@pytest.mark.parametrize("M,H,N", [(1, 4096, 1024), (48, 1024, 2048), (300, 512, 1040)])
@pytest.mark.parametrize("dtype_d", [torch.bfloat16, torch.float32])
def test_int8_norm_into_the_int8_product(capi, cuda, M, H, N, dtype_d):
    """The product's integer sum is exact; its conversion and two products round once each, then the result."""
    gen = torch.Generator(device="cuda").manual_seed(M + H + N)
    x, res = torch.empty(M, H, device=cuda, dtype=torch.bfloat16), torch.empty(M, H, device=cuda, dtype=torch.bfloat16)
    w = torch.randn(H, device=cuda, generator=gen).to(torch.bfloat16)
    W = torch.randint(-127, 128, (H, N), device=cuda, dtype=torch.int8, generator=gen)
    col = torch.rand(N, device=cuda, generator=gen) / 127
    q, scale = torch.empty(M, H, device=cuda, dtype=torch.int8), torch.empty(M, device=cuda)
    h, D = torch.empty_like(x), torch.empty(M, N, device=cuda, dtype=dtype_d)
    plan = capi.GemmPlan(q, W, D, row_scale=scale, col_scale=col)

    def call():
        capi.rms_norm_quantize(q, scale, x, w, res, h)
        plan.run()

    for qs, ss, hs, Ds in steps_of(cuda, x, [res], call, [q, scale, h, D]):
        want = (qs.double() @ W.double()) * ss.double()[:, None] * col.double()
        tol = 4 * U + (2.0 ** -8 if dtype_d == torch.bfloat16 else 0.0)
        assert bool(((Ds.double() - want).abs() <= tol * want.abs()).all())
    assert plan.device_status() == 0


@pytest.mark.parametrize("M,H,K", [(1, 4096, 256), (70, 1024, 512), (513, 2048, 320)])
@pytest.mark.parametrize("by_tma", [True, False])
def test_norm_residual_stream_into_a_product(capi, cuda, M, H, K, by_tma):
    """The stream that the norm wrote is added by the next product's epilogue, by TMA or by plain loads.  A running sum
    of K products and the stream: K + 1 truncations of 2 u of the sum of magnitudes, then one rounding to bf16."""
    gen = torch.Generator(device="cuda").manual_seed(M + H + K)
    x, res = torch.empty(M, H, device=cuda, dtype=torch.bfloat16), torch.empty(M, H, device=cuda, dtype=torch.bfloat16)
    a = torch.randn(M, K, device=cuda, generator=gen).to(torch.bfloat16)
    b = torch.randn(K, H, device=cuda, generator=gen).mul_(K ** -0.5).to(torch.bfloat16)
    q = torch.empty(M, H, device=cuda, dtype=torch.int8).view(torch.float8_e4m3fn)
    scale = torch.empty(H // 128, M, device=cuda).t()
    h, D = torch.empty_like(x), torch.empty(M, H, device=cuda, dtype=torch.bfloat16)
    plan = capi.GemmPlan(a, b, D, residual=h, flags=0 if by_tma else capi.FLAG_NO_RESIDUAL_TMA | capi.FLAG_NO_TAIL_STAGING)

    def call():
        capi.rms_norm_quantize(q, scale, x, None, res, h)
        plan.run()

    product, magnitudes = a.double() @ b.double(), a.double().abs() @ b.double().abs()
    for hs, Ds in steps_of(cuda, x, [res], call, [h, D]):
        want = product + hs.double()
        slack = (K + 1) * 2 * U * (magnitudes + hs.double().abs())
        assert bool(((Ds.double() - want).abs() <= slack + 2.0 ** -8 * (want.abs() + slack)).all())
    assert plan.device_status() == 0


@pytest.mark.parametrize("M,K,N", [(1, 1003, 256), (130, 1003, 264), (33, 129, 72)])
def test_a_row_pass_of_odd_width_feeds_a_product(capi, cuda, M, K, N):
    """Rows on 16-byte boundaries (a pitch that is a multiple of 16 codes), as the products' operands need them; with the
    width as the pitch the pass still writes them and the product refuses them.  128 truncations of 2 u within a block,
    one rounding per block, four for the factors; the last block is short."""
    gen = torch.Generator(device="cuda").manual_seed(K + N)
    e4m3, blocks = torch.float8_e4m3fn, -(-K // 128)
    x = torch.randn(M, 2 * K, device=cuda, generator=gen).to(torch.bfloat16)
    q = torch.empty(M, -(-K // 16) * 16, device=cuda, dtype=torch.int8).view(e4m3)[:, :K]
    scale = torch.empty(blocks, M, device=cuda).t()
    B = torch.randn(K, -(-N // 16) * 16, device=cuda, generator=gen).mul_(90).to(e4m3)[:, :N]
    sb = torch.rand(blocks, -(-N // 128), device=cuda, generator=gen) / 64
    D = torch.empty(M, N, device=cuda)
    plan = capi.GroupedGemmPlan(q, B, D, scale_a=scale, scale_b=sb)

    def wide(t, dim, n):
        return t.double().repeat_interleave(128, dim).narrow(dim, 0, n)

    for producer in (lambda: capi.rms_norm_quantize(q, scale, x[:, :K]), lambda: capi.act_mul_quantize(q, scale, x)):
        producer()
        plan.run()
        a, b = q.double() * wide(scale, 1, K), B.double() * wide(wide(sb, 0, K), 1, N)
        slack = (min(K, 128) * 2 + blocks + 4 + 148) * U * (a.abs() @ b.abs())
        assert bool(((D.double() - a @ b).abs() <= slack).all())
    tight = torch.empty(M, K, device=cuda, dtype=torch.int8).view(e4m3)
    capi.rms_norm_quantize(tight, scale, x[:, :K])
    capi.rms_norm_quantize(q, scale, x[:, :K])
    assert torch.equal(tight.double(), q.double())
    if M > 1:
        with pytest.raises(capi.XfError, match="16 bytes"):
            capi.GroupedGemmPlan(tight, B, D, scale_a=scale, scale_b=sb)
