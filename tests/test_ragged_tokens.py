"""The MoE layer's backward at token counts that are no multiple of anything, with few experts."""
import pytest
import torch

pytestmark = pytest.mark.gpu
needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')


@needs_cuda
@pytest.mark.parametrize('T', [1, 5, 60, 63])
@pytest.mark.parametrize('kw', [dict(), dict(fp8_block=True, gate=dict(scoring='sigmoid', num_groups=4, topk_groups=2))])
def test_router_gradient_of_ragged_tokens(T, kw):
    # the same tokens and eight-fold padding with rows whose gradient is zero give the same router gradient: the
    # added products are zeros
    from test_zero_tokens import _layer
    buf, layer = _layer(**kw)
    x = torch.randn(64, 512, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).cuda()
    dy = torch.randn(64, 512, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    dy[T:] = 0
    want = torch.autograd.grad(layer(x), layer.router, dy)[0]
    got = torch.autograd.grad(layer(x[:T]), layer.router, dy[:T])[0]
    assert want.abs().amax() > 0 and torch.equal(got, want)
    buf.check()
    buf.destroy()
