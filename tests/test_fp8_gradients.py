"""e4m3 gradients of any size: the quantiser's floor, and the backward of fp8_block layers."""
import pytest
import torch

from deepep_trn_b200.ops.quant import GRAD_AMAX_FLOOR, quantize_fp8
from deepep_trn_b200.utils.codec import dequantize_fp8_1x128, quantize_fp8_1x128

needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')
SIZES = [1.0, 1e-4, 1e-8, 1e-10, 1e-20, 1e-30]


def _rows(size, seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(50, 512, generator=g)
    x[3] = 0
    x[7, 130:200] = 0
    return (x * size).to(dtype)


@pytest.mark.parametrize('size', SIZES)
def test_small_rows_keep_their_values(size):
    x = _rows(size)
    q, s = quantize_fp8(x, amax_floor=GRAD_AMAX_FLOOR)
    # half a step of e4m3: 2^-4 of the value, 2^-10 of the scale below the normal range; the scaled value
    # and the scale carry a rounding each (2^-22 together, with room)
    err = (dequantize_fp8_1x128(q, s).double() - x.double()).abs()
    bound = x.double().abs() * (2.0 ** -4 + 2.0 ** -22) + s.double().repeat_interleave(128, -1) * 2.0 ** -10
    assert (err <= bound).all()
    assert (q[3].float() == 0).all() and (s > 0).all() and torch.isfinite(s).all()
    block = x.float().abs().unflatten(1, (4, 128)).amax(-1)
    assert torch.equal(s[block > 0], torch.div(block, torch.full_like(block, 448.0))[block > 0])


def test_floor_of_activations_is_unchanged():
    x = _rows(1e-8)
    q, s = quantize_fp8(x)
    assert torch.equal(s, torch.full_like(s, 1e-4) / torch.full_like(s, 448.0))
    for bad in (0.0, 2.0 ** -117, 1e3, float('nan')):
        with pytest.raises(RuntimeError):
            quantize_fp8(x, amax_floor=bad)


@pytest.mark.gpu
@needs_cuda
@pytest.mark.parametrize('size', SIZES)
@pytest.mark.parametrize('round_scale', [False, True])
@pytest.mark.parametrize('floor', [GRAD_AMAX_FLOOR, 1e-4, 2.0])
def test_floor_on_cuda_matches_definition(size, round_scale, floor):
    for dtype in (torch.bfloat16, torch.float16):
        x = _rows(size, 1, dtype)
        q, s = quantize_fp8(x.cuda(), round_scale, floor)
        rq, rs = quantize_fp8_1x128(x, round_scale, floor)
        assert torch.equal(s.cpu(), rs) and torch.equal(q.cpu().view(torch.uint8), rq.view(torch.uint8))
    for bad in (0.0, 2.0 ** -117, 1e3, float('nan')):
        with pytest.raises(RuntimeError):
            quantize_fp8(x.cuda(), round_scale, bad)


@pytest.mark.gpu
@needs_cuda
@pytest.mark.parametrize('gate', [None, dict(scoring='sigmoid', num_groups=4, topk_groups=2, scale=2.5)])
def test_gradients_scale_with_the_loss(gate):
    # The backward is linear and a power of two goes through every rounding unchanged (nothing comes near
    # the subnormal numbers at 2^-33 of these values), so the gradients have to scale to the last bit.
    import torch.distributed as dist
    from deepep_trn_b200 import Buffer
    from deepep_trn_b200.models.moe import MoELayer
    from test_moe_weights import _init_single
    _init_single()
    buf = Buffer(dist.group.WORLD, backend='nvlink', num_max_tokens_per_rank=128)
    layer = MoELayer(buf, 512, 256, 16, 4, device='cuda', init_std=0.05, gate=gate, fp8_block=True)
    g = torch.Generator(device='cuda').manual_seed(5)
    x = (torch.randn(128, 512, generator=g, device='cuda') * 0.5).to(torch.bfloat16).requires_grad_()
    dy = torch.randn(128, 512, generator=g, device='cuda').to(torch.bfloat16)
    leaves = (x, layer.router, layer.w1, layer.w2)
    for factor in (2.0 ** -10, 2.0 ** -33):
        want = torch.autograd.grad(layer(x), leaves, dy)
        got = torch.autograd.grad(layer(x), leaves, dy * factor)
        for name, a, b in zip(('dx', 'dWr', 'dW1', 'dW2'), got, want):
            assert b.abs().max() > 0 and torch.equal(a.float() / factor, b.float()), name
    buf.check()
    buf.destroy()
