"""The expert-parallel layer with the grouped gate and fp8 block-scaled experts on one B200, forward,
backward and the low-latency step, against a torch definition that quantises where the layer does."""
import math
import os
import socket

import pytest
import torch

pytestmark = pytest.mark.gpu
needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')

GATE = dict(scoring='sigmoid', num_groups=4, topk_groups=2, group_score='top2', renormalize=True, scale=2.5)


def _rel(a, b):
    a, b = a.float(), b.float()
    return ((a - b).norm() / b.norm().clamp_min(1e-12)).item()


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


def _through(value, quantised):
    """The quantised values, with the gradient of the values."""
    return value + (quantised - value).detach()


def _rows(x):
    from deepep_trn_b200.utils.codec import dequantize_fp8_1x128, quantize_fp8_1x128
    return _through(x, dequantize_fp8_1x128(*quantize_fp8_1x128(x.detach())))


def _weights(w):
    from deepep_trn_b200.utils.codec import dequantize_fp8_128x128, quantize_fp8_128x128
    return _through(w, dequantize_fp8_128x128(*quantize_fp8_128x128(w.detach())))


def _definition(x, Wr, W1, W2, k, bias, gate, quant):
    """fp32 layer on one rank; with `quant` x, h and the weights are rounded to e4m3 as the layer does."""
    from deepep_trn_b200.ops.gemm import deinterleave
    from deepep_trn_b200.utils.testing import router_gate_reference
    logits = x @ Wr.t()
    idx, _ = router_gate_reference(logits.detach(), k, bias=bias, **gate)
    has = idx >= 0
    s = torch.sigmoid(logits) if gate['scoring'] == 'sigmoid' else torch.softmax(logits, 1)
    w = torch.where(has, s.gather(1, idx.clamp_min(0)), torch.zeros((), device=x.device))
    if gate['renormalize']:
        w = w / w.sum(1, keepdim=True).clamp_min(1e-20)
    w = w * gate['scale']
    xq, w1, w2 = (_rows(x), _weights(W1), _weights(W2)) if quant else (x, W1, W2)
    out = torch.zeros_like(x)
    for e in range(W1.shape[0]):
        hit = idx == e
        tok = hit.any(1).nonzero().flatten()
        if tok.numel() == 0:
            continue
        g, u = deinterleave(xq[tok] @ w1[e].t())
        h = torch.nn.functional.silu(g) * u
        we = (w[tok] * hit[tok]).sum(1, keepdim=True)
        out = out.index_add(0, tok, we * ((_rows(h) if quant else h) @ w2[e].t()))
    return out, idx


def _layer(buf, H, I, E, K, **kw):
    from deepep_trn_b200.models.moe import MoELayer
    layer = MoELayer(buf, H, I, E, K, device='cuda', init_std=0.05, **kw)
    g = torch.Generator(device='cuda').manual_seed(11)
    layer.router_bias.copy_(torch.randn(E, generator=g, device='cuda') * 0.05)
    return layer


def _check(fp8_block, gate, close_experts=0):
    import torch.distributed as dist
    from deepep_trn_b200 import Buffer
    _init_single()
    buf = Buffer(dist.group.WORLD, backend='nvlink', num_max_tokens_per_rank=512)
    T, H, I, E, K = 384, 512, 256, 16, 4
    layer = _layer(buf, H, I, E, K, gate=gate, fp8_block=fp8_block)
    if close_experts:
        layer.router_bias[close_experts:] = -math.inf
    g = torch.Generator(device='cuda').manual_seed(5)
    x = (torch.randn(T, H, generator=g, device='cuda') * 0.5).to(torch.bfloat16).requires_grad_()
    dy = torch.randn(T, H, generator=g, device='cuda').to(torch.bfloat16)
    y = layer(x)
    y.backward(dy)
    torch.cuda.synchronize()
    r = [t.detach().float().requires_grad_() for t in (x, layer.router, layer.w1, layer.w2)]
    yr, idx = _definition(*r, K, layer.router_bias, gate, fp8_block)
    yr.backward(dy.float())
    if close_experts and close_experts < K:
        assert (idx[:, close_experts:] == -1).all()
    # Forward: bf16 activations between the products (each 2^-9 rms relative) and fp32 sums; the e4m3
    # roundings are the definition's own but for ties moved by those sums. A token whose logits, summed in
    # another order, tie within 1e-6 may pick another expert: none at this size.
    assert _rel(y, yr) < 1e-2, _rel(y, yr)
    # Backward: e4m3 of d_o and of dpre (rms 2.6 % of a value each, not in the definition) reach dx through
    # both, dW1 through the first; dW2 and the router see bf16 only.
    names = ['dx', 'dWr', 'dW1', 'dW2']
    tol = dict(dx=6e-2, dWr=3e-2, dW1=5e-2, dW2=2e-2) if fp8_block else dict(dx=2e-2, dWr=3e-2, dW1=2e-2, dW2=2e-2)
    for n, got, ref in zip(names, (x, layer.router, layer.w1, layer.w2), r):
        assert _rel(got.grad, ref.grad) < tol[n], (n, _rel(got.grad, ref.grad))
    with torch.no_grad():
        assert torch.equal(layer(x), y)      # inference runs the same products
    buf.check()
    buf.destroy()


@needs_cuda
@pytest.mark.parametrize('fp8_block', [True, False])
@pytest.mark.parametrize('gate', [GATE, dict(scoring='softmax', renormalize=False, scale=4.0)])
def test_layer_with_gate(fp8_block, gate):
    _check(fp8_block, gate)


@needs_cuda
def test_layer_with_fewer_experts_than_choices():
    # three experts left for four choices: the last id is -1, which dispatch skips, in both directions
    _check(True, dict(scoring='sigmoid', renormalize=True, scale=1.0), close_experts=3)


@needs_cuda
def test_low_latency_step_matches_definition_and_replays():
    import torch.distributed as dist
    from deepep_trn_b200 import Buffer
    _init_single()
    buf = Buffer(dist.group.WORLD, backend='nvlink', num_max_tokens_per_rank=64)
    H, I, E, K, M = 512, 256, 16, 4, 64
    layer = _layer(buf, H, I, E, K, gate=GATE, fp8_block=True)
    g = torch.Generator(device='cuda').manual_seed(6)
    for T in (1, 7, 64):
        x = (torch.randn(T, H, generator=g, device='cuda') * 0.5).to(torch.bfloat16)
        y = layer.forward_low_latency(x, M)
        yr, _ = _definition(x.float(), layer.router.float(), layer.w1.float(), layer.w2.float(), K, layer.router_bias,
                            GATE, True)
        assert _rel(y, yr) < 1e-2, (T, _rel(y, yr))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        layer.forward_low_latency(x, M)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.forward_low_latency(x, M)
    x.copy_(x.roll(3, 0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, y.roll(3, 0))
    with pytest.raises(ValueError):
        _layer(buf, H, I, E, K).forward_low_latency(x, M)
    buf.check()
    buf.destroy()


@needs_cuda
def test_custom_ops():
    import deepep_trn_b200.ops.library  # noqa: F401
    ops = torch.ops.b200ep
    torch.manual_seed(6)
    logits = torch.randn(64, 32, device='cuda')
    torch.library.opcheck(ops.router_gate, (logits, 4, 'sigmoid', None, 4, 2))
    idx, w = ops.router_gate(logits, 4)
    torch.library.opcheck(ops.router_gate_bwd, (logits, idx, w))
    q, s = ops.quantize_fp8_weight(torch.randn(2, 256, 512, device='cuda'))
    x, xs = ops.quantize_fp8(torch.randn(100, 512, device='cuda').bfloat16())
    offs = torch.tensor([0, 40, 100], device='cuda')
    h, hs, pre = ops.grouped_gemm_fp8_swiglu(x, xs, q, s, offs)
    out = ops.grouped_gemm_fp8_block(x, xs, q, s, offs)
    assert torch.equal(out, pre) and h.shape == (100, 128) and hs.shape == (100, 1)


def test_layer_refusals():
    from deepep_trn_b200.models.moe import MoELayer

    class Group:
        group_size, rank = 1, 0

    with pytest.raises(ValueError):
        MoELayer(Group(), 128, 128, 8, 2, fp8_experts=True, fp8_block=True)
    with pytest.raises(ValueError):
        MoELayer(Group(), 128, 128, 8, 2, fp8_experts=True, gate=GATE)
