"""The quantised expert weights of a layer follow its weights, however those are written."""
import os
import socket

import pytest
import torch

from deepep_trn_b200.models.moe import MoELayer
from deepep_trn_b200.ops.gemm import quantize_fp8_weight
from deepep_trn_b200.utils.codec import quantize_fp8_128x128

needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')


class Group:
    group_size, rank = 1, 0


def _write(layer, how):
    """Doubles W1 and negates W2 as an optimizer with fp32 masters, an optimizer or a checkpoint does."""
    w1, w2 = 2 * layer.w1.detach(), -layer.w2.detach()
    if how == 'data':
        layer.w1.data.copy_(w1)
        layer.w2.data.copy_(w2)
    elif how == 'no_grad':
        with torch.no_grad():
            layer.w1.copy_(w1)
            layer.w2.copy_(w2)
    else:
        layer.load_state_dict(dict(layer.state_dict(), w1=w1, w2=w2))


def _equal(wq, layer):
    want = (*quantize_fp8_128x128(layer.w1.detach().cpu()), *quantize_fp8_128x128(layer.w2.detach().cpu()))
    return all(torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8)) for a, b in zip(wq, want))


@pytest.mark.parametrize('how', ['data', 'no_grad', 'load'])
def test_training_quantises_the_weights_of_the_step(how):
    layer = MoELayer(Group(), 256, 128, 4, 2, fp8_block=True)
    first = layer._block_weights(True)
    assert _equal(first, layer)
    _write(layer, how)
    assert _equal(layer._block_weights(True), layer)
    assert not _equal(first, layer)     # the first step's weights stay what its backward needs


def _init_single():
    import torch.distributed as dist
    if dist.is_initialized():
        return
    os.environ['MASTER_ADDR'] = '127.0.0.1'
    with socket.socket() as s:
        s.bind(('127.0.0.1', 0))
        os.environ['MASTER_PORT'] = str(s.getsockname()[1])
    torch.cuda.set_device(0)
    dist.init_process_group('nccl', rank=0, world_size=1, device_id=torch.device('cuda', 0))


def _buffer():
    import torch.distributed as dist
    from deepep_trn_b200 import Buffer
    _init_single()
    return Buffer(dist.group.WORLD, backend='nvlink', num_max_tokens_per_rank=64)


def _layer(buf, **kw):
    return MoELayer(buf, 512, 256, 16, 4, device='cuda', init_std=0.05, **kw)


def _x(T=64, seed=3):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return (torch.randn(T, 512, generator=g, device='cuda') * 0.5).to(torch.bfloat16)


@pytest.mark.gpu
@needs_cuda
@pytest.mark.parametrize('how', ['data', 'no_grad', 'load'])
@pytest.mark.parametrize('kw', [dict(fp8_block=True), dict(fp8_experts=True)])
def test_training_and_evaluation_follow_the_weights(how, kw):
    # train, evaluate, update, train, evaluate: as a layer that is made with the new weights
    buf = _buffer()
    layer, x = _layer(buf, **kw), _x()
    old = layer(x).detach()
    with torch.no_grad():
        layer(x)
    _write(layer, how)
    fresh = _layer(buf, **kw)
    fresh.load_state_dict(layer.state_dict())
    y = layer(x).detach()
    assert torch.equal(y, fresh(x).detach()) and not torch.equal(y, old)
    with torch.no_grad():
        assert torch.equal(layer(x), fresh(x))
    buf.check()
    buf.destroy()
