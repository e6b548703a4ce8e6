"""Ranks without tokens and steps whose tokens find no expert: the products and the MoE layer on zero rows."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')
BF = torch.bfloat16


@needs_cuda
def test_products_of_zero_rows():
    from deepep_trn_b200.ops import gemm
    z = lambda *s, dtype=BF: torch.zeros(*s, device='cuda', dtype=dtype)  # noqa: E731
    offs = torch.zeros(4, dtype=torch.int64, device='cuda')
    for kn in (False, True):
        B = z(3, 128, 256) if kn else z(3, 256, 128)
        assert gemm.grouped_gemm(z(0, 128), B, offs, b_layout='kn' if kn else 'nk').shape == (0, 256)
    assert [t.shape for t in gemm.grouped_gemm(z(0, 128), z(3, 256, 128), offs, epilogue='swiglu')] == [(0, 128), (0, 256)]
    q, s = gemm.quantize_fp8_blocks(z(3, 256, 128))
    assert gemm.grouped_gemm_fp8(z(0, 128).to(torch.float8_e4m3fn), z(0, 1, dtype=torch.float32), q, s, offs).shape == (0, 256)
    for dtype in (BF, torch.float32):
        out = torch.full((3, 128, 256), 7.0, device='cuda', dtype=dtype)
        gemm.grouped_gemm_wgrad(z(0, 128), z(0, 256), offs, out=out)
        assert (out == 0).all()
        out.fill_(7)
        gemm.grouped_gemm_wgrad(z(128, 0), z(256, 0), offs, out=out, layout='mk')
        assert (out == 0).all()
    gemm.check()


def _layer(**kw):
    import torch.distributed as dist
    from deepep_trn_b200 import Buffer
    from deepep_trn_b200.models.moe import MoELayer
    from test_moe_weights import _init_single
    _init_single()
    buf = Buffer(dist.group.WORLD, backend='nvlink', num_max_tokens_per_rank=64)
    return buf, MoELayer(buf, 512, 256, 16, 4, device='cuda', init_std=0.05, **kw)


@needs_cuda
@pytest.mark.parametrize('kw,T', [(dict(), 0), (dict(fp8_block=True), 0), (dict(gate=dict(scoring='sigmoid')), 0),
                                  (dict(gate=dict(scoring='sigmoid')), 8),
                                  (dict(gate=dict(scoring='softmax', renormalize=False), fp8_block=True), 0),
                                  (dict(gate=dict(scoring='softmax', renormalize=False), fp8_block=True), 8)])
def test_layer_without_work(kw, T):
    buf, layer = _layer(**kw)
    if T:
        layer.router_bias.fill_(-math.inf)      # closes every expert
    x = torch.randn(T, 512, device='cuda').to(BF).requires_grad_()
    y = layer(x)
    assert y.shape == (T, 512) and (y == 0).all()
    y.backward(torch.ones_like(y))
    torch.cuda.synchronize()
    for g in (x.grad, layer.router.grad, layer.w1.grad, layer.w2.grad):
        assert (g == 0).all()
    if kw.get('fp8_block'):
        out = layer.forward_low_latency(x.detach(), 64)
        assert out.shape == (T, 512) and (out == 0).all()
    # the next step is an ordinary one
    layer.router_bias.zero_()
    x = torch.randn(32, 512, device='cuda').to(BF)
    assert layer(x).abs().amax() > 0
    buf.check()
    buf.destroy()


@needs_cuda
def test_power_of_two_fp8_layer_without_tokens():
    buf, layer = _layer(fp8_experts=True)
    with torch.no_grad():
        assert layer(torch.zeros(0, 512, device='cuda', dtype=BF)).shape == (0, 512)
        assert layer(torch.randn(8, 512, device='cuda').to(BF)).abs().amax() > 0
    buf.check()
    buf.destroy()
