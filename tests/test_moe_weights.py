"""The quantised expert weights of a layer follow its weights, however those are written."""
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
    # by address, not through the environment: other tests start children that would take the port from it
    with socket.socket() as s:
        s.bind(('127.0.0.1', 0))
        port = s.getsockname()[1]
    torch.cuda.set_device(0)
    dist.init_process_group('nccl', init_method=f'tcp://127.0.0.1:{port}', rank=0, world_size=1,
                            device_id=torch.device('cuda', 0))


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


# ------------------------------------------------------------------------------- the kept copy
def _ptrs(wq):
    return [t.data_ptr() for t in wq]


@pytest.mark.parametrize('how', ['data', 'no_grad', 'load'])
def test_quantize_weights_renews_its_copy_in_place(how):
    layer = MoELayer(Group(), 256, 128, 4, 2, fp8_block=True)
    layer.quantize_weights()
    kept = layer._block_weights(False)
    assert _equal(kept, layer) and _ptrs(layer._block_weights(False)) == _ptrs(kept)
    _write(layer, how)
    if how != 'data':                       # a write that can be seen is
        assert _equal(layer._block_weights(False), layer)
    layer.quantize_weights()
    assert _ptrs(layer._block_weights(False)) == _ptrs(kept) and _equal(kept, layer)


def test_copy_is_left_aside():
    layer = MoELayer(Group(), 256, 128, 4, 2, fp8_block=True)
    assert _equal(layer._block_weights(False), layer)      # none was asked for
    layer.quantize_weights()
    kept = layer._block_weights(False)
    with pytest.raises((AttributeError, RuntimeError)):
        layer(torch.zeros(4, 256, dtype=torch.bfloat16))   # a call with gradients (on the CPU it gets no further)
    _write(layer, 'data')
    assert _equal(layer._block_weights(False), layer) and not _equal(kept, layer)
    layer.quantize_weights()
    with torch.inference_mode():
        assert _ptrs(layer._block_weights(False)) == _ptrs(kept)
        made_inside = MoELayer(Group(), 256, 128, 4, 2, fp8_block=True)
        made_inside.quantize_weights()
        assert _equal(made_inside._block_weights(False), made_inside)
    layer.w2 = torch.nn.Parameter(torch.cat([layer.w2.detach()] * 2, 1))   # of another shape
    layer.quantize_weights()
    assert _equal(layer._block_weights(False), layer)
    with pytest.raises(ValueError):
        MoELayer(Group(), 256, 128, 4, 2).quantize_weights()


def test_quantiser_into_given_tensors():
    w = torch.randn(2, 200, 264)
    q, sc = quantize_fp8_weight(w)
    out = torch.zeros_like(q), torch.zeros_like(sc)
    got = quantize_fp8_weight(w, out=out)
    assert got[0] is out[0] and got[1] is out[1]
    assert torch.equal(out[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(out[1], sc)
    from deepep_trn_b200.ops import available
    if not available():
        return
    for bad in ((q[:1], sc), (q, sc[:, :1]), (q.view(torch.uint8), sc), (q, sc.double()),
                (q.transpose(1, 2).contiguous().transpose(1, 2), sc), (None, sc)):
        with pytest.raises(RuntimeError):
            quantize_fp8_weight(w, out=bad)


@pytest.mark.gpu
@needs_cuda
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('N,K,offset', [(200, 264, 0), (200, 264, 3), (130, 77, 1)])
def test_quantiser_into_given_tensors_on_cuda(dtype, N, K, offset):
    w = torch.randn(2, N, K, generator=torch.Generator().manual_seed(N)).to(dtype).cuda()
    q, sc = quantize_fp8_weight(w)
    store = torch.full((q.numel() + 64,), 0x55, dtype=torch.uint8, device='cuda')
    out = store[offset:offset + q.numel()].view(q.shape).view(q.dtype), torch.zeros_like(sc)
    quantize_fp8_weight(w, out=out)
    assert torch.equal(out[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(out[1], sc)
    assert (store[:offset] == 0x55).all() and (store[offset + q.numel():] == 0x55).all()
    with pytest.raises(RuntimeError):
        quantize_fp8_weight(w, out=(out[0].cpu(), out[1]))


def _captured(layer, x):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        layer.forward_low_latency(x, 64)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.forward_low_latency(x, 64)
    return graph, out


@pytest.mark.gpu
@needs_cuda
@pytest.mark.parametrize('how', ['data', 'no_grad'])
@pytest.mark.parametrize('keep', [True, False])
def test_captured_generation_step_follows_the_weights(how, keep):
    buf = _buffer()
    layer, x = _layer(buf, fp8_block=True), _x()
    if keep:
        layer.quantize_weights()
    graph, out = _captured(layer, x)
    graph.replay()
    torch.cuda.synchronize()
    old = out.clone()
    assert torch.equal(old, layer.forward_low_latency(x, 64))
    layer(x).sum().backward()               # a training step between the replays
    _write(layer, how)
    if keep:
        layer.quantize_weights()
    fresh = _layer(buf, fp8_block=True)
    fresh.load_state_dict(layer.state_dict())
    want = fresh.forward_low_latency(x, 64)
    hold = [torch.full_like(layer.w1, 9.0) for _ in range(4)]   # what the allocator had to give is written over
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and not torch.equal(out, old)
    assert torch.equal(layer.forward_low_latency(x, 64), want)
    del hold, graph
    buf.check()
    buf.destroy()


@pytest.mark.gpu
@needs_cuda
def test_quantize_weights_is_refused_in_a_capture():
    layer = MoELayer(Group(), 256, 128, 4, 2, device='cuda', fp8_block=True)
    layer.quantize_weights()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layer.w1 + 1
        with pytest.raises(RuntimeError):
            layer.quantize_weights()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, layer.w1 + 1) and _equal(layer._block_weights(False), layer)
