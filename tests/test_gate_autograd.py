"""The expert gate under autograd: the weights of CUDA logits carry the gradient that router_gate_bwd gives."""
import math

import pytest
import torch

from deepep_trn_b200.ops.moe_ops import router_gate, router_gate_bwd
from deepep_trn_b200.utils.testing import router_gate_bwd_reference

needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')
KW = dict(num_groups=4, topk_groups=2)


def _logits(dev, dtype=torch.float32):
    x = torch.randn(60, 64, generator=torch.Generator().manual_seed(1))
    x[3] = -math.inf
    x[5, 10:] = -math.inf
    return x.to(dtype).to(dev).requires_grad_()


def _dw():
    return torch.randn(60, 6, generator=torch.Generator().manual_seed(2))


@pytest.mark.parametrize('scoring', ['sigmoid', 'softmax'])
def test_gradient_on_cpu(scoring):
    x = _logits('cpu')
    idx, w = router_gate(x, 6, scoring, **KW, scale=2.5)
    assert not idx.requires_grad
    w.backward(_dw())
    ref = router_gate_bwd_reference(x.detach(), idx, _dw(), scoring, True, 2.5)
    assert torch.equal(x.grad, ref) and torch.isfinite(ref).all()
    # rows without masked experts can be differentiated as they are defined: the same formulas in fp64 in
    # another order, rounded to fp32 once, so one step apart
    y = x.detach().double().requires_grad_()
    s = torch.sigmoid(y) if scoring == 'sigmoid' else torch.softmax(y, 1)
    w = s.gather(1, idx.clamp_min(0))
    (2.5 * w / w.sum(1, keepdim=True) * _dw()).sum().backward()
    whole = torch.isfinite(x.detach()).all(1)
    assert whole.sum() == 58
    assert ((x.grad - y.grad).abs() <= 2.0 ** -23 * y.grad.abs() + 1e-12)[whole].all()


@pytest.mark.gpu
@needs_cuda
@pytest.mark.parametrize('scoring', ['sigmoid', 'softmax'])
@pytest.mark.parametrize('renorm', [True, False])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_gradient_on_cuda(scoring, renorm, dtype):
    x, dw = _logits('cuda', dtype), _dw().cuda()
    bias = torch.randn(64, device='cuda')
    args = dict(scoring=scoring, renormalize=renorm, scale=2.5)
    idx, w = router_gate(x, 6, bias=bias, **KW, **args)
    plain_idx, plain_w = router_gate(x.detach(), 6, bias=bias, **KW, **args)
    assert w.requires_grad and not idx.requires_grad and not plain_w.requires_grad
    assert torch.equal(idx, plain_idx) and torch.equal(w, plain_w)
    w.backward(dw)
    assert x.grad.dtype == dtype and torch.equal(x.grad, router_gate_bwd(x.detach(), idx, dw, **args))
    # a broadcast gradient, and a leaf behind another operation
    g, = torch.autograd.grad(router_gate(x * 1.0, 6, bias=bias, **KW, **args)[1].sum(), x)
    assert torch.equal(g, router_gate_bwd(x.detach(), idx, torch.ones_like(dw), **args))
    with torch.no_grad():
        assert not router_gate(x, 6, bias=bias, **KW, **args)[1].requires_grad
    g, = torch.autograd.grad(router_gate(x, 6, bias=bias, **KW, **args)[1].square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()          # once only


@pytest.mark.gpu
@needs_cuda
def test_gradient_in_a_graph_and_on_a_stream():
    x, dw = _logits('cuda'), _dw().cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want, = torch.autograd.grad(router_gate(x, 6, **KW)[1], x, dw)
    torch.cuda.current_stream().wait_stream(s)
    static = x.detach().clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(router_gate(static, 6, **KW)[1], static, dw)
    with torch.no_grad():
        static.copy_(x.roll(1, 0))
    graph.replay()
    torch.cuda.synchronize()
    idx, _ = router_gate(static.detach(), 6, **KW)
    assert torch.equal(got, router_gate_bwd(static.detach(), idx, dw))
    assert torch.equal(want, router_gate_bwd(x.detach(), router_gate(x.detach(), 6, **KW)[0], dw))
