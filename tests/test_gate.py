"""The expert gate (router_gate and its gradient): the torch definition on the CPU, and the kernels
against it in fp64, where its selection has to be the same to the last id."""
import math

import pytest
import torch

from deepep_trn_b200.ops.moe_ops import router_gate, router_gate_bwd
from deepep_trn_b200.utils.testing import router_gate_bwd_reference, router_gate_reference

needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')
INF = math.inf


def _logits(T, E, seed, dtype=torch.float32, masked=0.0, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, E, generator=g) * spread
    if masked:
        x = x.masked_fill(torch.rand(T, E, generator=g) < masked, -INF)
        x = x.masked_fill(torch.rand(T, 1, generator=g) < 0.1, -INF)   # rows with nothing left
    return x.to(dtype)


# ------------------------------------------------------------------------------- definition (CPU)
def test_gate_by_hand():
    x = torch.tensor([[2.0, 1.0, 0.0, 3.0, -1.0, 0.5]])
    idx, w = router_gate(x, 2, renormalize=False)
    assert idx.tolist() == [[3, 0]]
    assert torch.allclose(w, torch.sigmoid(torch.tensor([[3.0, 2.0]])))
    # the bias moves the choice, not the weight
    b = torch.tensor([0, 0, 0, 0, 5.0, 0])
    idx, w = router_gate(x, 2, bias=b, renormalize=False)
    assert idx.tolist() == [[4, 3]] and torch.allclose(w, torch.sigmoid(torch.tensor([[-1.0, 3.0]])))
    # groups {0,1}, {2,3}, {4,5}: by their largest {2,3} wins, by the sum of two {0,1}
    assert router_gate(x, 1, num_groups=3, topk_groups=1, group_score='max')[0].item() == 3
    assert router_gate(x, 1, num_groups=3, topk_groups=1, group_score='top2')[0].item() == 0
    idx, w = router_gate(x, 2, scoring='softmax', scale=3.0)
    assert torch.allclose(w, 3 * torch.softmax(torch.tensor([[3.0, 2.0]]), 1))
    idx, w = router_gate(x, 2, scoring='softmax', renormalize=False)
    assert torch.allclose(w, torch.softmax(x, 1)[:, [3, 0]])


def test_gate_unavailable_experts():
    x = torch.tensor([[-INF, math.nan, 0.5, -INF], [-INF] * 4, [INF, 1.0, INF, 0.0]])
    for scoring in ('sigmoid', 'softmax'):
        idx, w = router_gate(x, 2, scoring=scoring)
        assert idx.tolist() == [[2, -1], [-1, -1], [0, 2]]
        assert torch.equal(w, torch.tensor([[1.0, 0.0], [0.0, 0.0], [0.5, 0.5]]))
        d = router_gate_bwd(x, idx, torch.ones(3, 2), scoring=scoring, renormalize=False)
        assert torch.isfinite(d).all() and (d[1] == 0).all()
    # ties go to the lower id; a bias of -inf closes an expert
    assert router_gate(torch.zeros(1, 6), 3, renormalize=False)[0].tolist() == [[0, 1, 2]]
    assert router_gate(torch.zeros(1, 3), 2, bias=torch.tensor([-INF, 0.0, 0.0]))[0].tolist() == [[1, 2]]


@pytest.mark.parametrize('scoring', ['sigmoid', 'softmax'])
@pytest.mark.parametrize('renorm', [True, False])
def test_gate_gradient_against_differences(scoring, renorm):
    # central differences of the fp64 weights: error h^2/6 * |f'''|, and |f'''| < 1 for products of
    # sigmoids and softmaxes, so h = 1e-4 leaves 2e-9 per weight (and 1e-16 / h = 1e-12 of rounding).
    # Logits 0.15 apart keep the selection fixed.
    T, E, K, scale, h = 3, 12, 4, 1.5, 1e-4
    g = torch.Generator().manual_seed(1)
    x = torch.stack([torch.randperm(E, generator=g) for _ in range(T)]).double() * 0.15
    idx, _ = router_gate(x.float(), K, scoring, renormalize=renorm, scale=scale)
    dw = torch.randn(T, K, generator=g)

    def weights(x):
        s = torch.sigmoid(x) if scoring == 'sigmoid' else torch.softmax(x, 1)
        w = s.gather(1, idx)
        return scale * (w / w.sum(1, keepdim=True) if renorm else w)

    num = torch.zeros(T, E, dtype=torch.float64)
    for e in range(E):
        d = torch.zeros(T, E, dtype=torch.float64)
        d[:, e] = h
        num[:, e] = ((weights(x + d) - weights(x - d)) / (2 * h) * dw).sum(1)
    got = router_gate_bwd_reference(x, idx, dw, scoring, renorm, scale)
    tol = 4 * scale * dw.abs().sum(1).max().item() * h * h
    assert (got - num).abs().max().item() < tol + 1e-10
    assert torch.allclose(router_gate_bwd(x.float(), idx, dw, scoring, renorm, scale), num.float(), atol=1e-6)


def _refusals(dev):
    x = torch.zeros(4, 12, device=dev)
    cases = [
        (ValueError, lambda: router_gate(x, 2, scoring='relu')),
        (ValueError, lambda: router_gate(x, 2, group_score='sum')),
        (ValueError, lambda: router_gate_bwd(x, x[:, :2].long(), x[:, :2], scoring='none')),
        (RuntimeError, lambda: router_gate(x, 0)),
        (RuntimeError, lambda: router_gate(x, 13)),
        (RuntimeError, lambda: router_gate(torch.zeros(4, 64, device=dev), 33)),
        (RuntimeError, lambda: router_gate(x, 2, num_groups=5)),
        (RuntimeError, lambda: router_gate(x, 2, num_groups=4, topk_groups=5)),
        (RuntimeError, lambda: router_gate(x, 4, num_groups=4, topk_groups=1)),
        (RuntimeError, lambda: router_gate(x, 2, num_groups=0)),
        (RuntimeError, lambda: router_gate(torch.zeros(2, 1025, device=dev), 2)),
        (RuntimeError, lambda: router_gate(x.double(), 2)),
        (RuntimeError, lambda: router_gate(x[0], 2)),
        (RuntimeError, lambda: router_gate(x.t(), 2)),
        (RuntimeError, lambda: router_gate(x, 2, bias=torch.zeros(11, device=dev))),
        (RuntimeError, lambda: router_gate(x, 2, bias=torch.zeros(12, device=dev, dtype=torch.bfloat16))),
        (RuntimeError, lambda: router_gate_bwd(x, torch.zeros(3, 2, device=dev, dtype=torch.long), x[:, :2])),
        (RuntimeError, lambda: router_gate_bwd(x, torch.zeros(4, 2, device=dev, dtype=torch.int32), x[:, :2])),
        (RuntimeError, lambda: router_gate_bwd(x, torch.zeros(4, 2, device=dev, dtype=torch.long), x[:, :3])),
    ]
    for err, call in cases:
        with pytest.raises(err):
            call()


def test_gate_refusals():
    from deepep_trn_b200.ops import available
    if not available():
        pytest.skip('the extension is not built')
    _refusals('cpu')


# --------------------------------------------------------------------------------------- kernels
def _close_w(got, ref, scale):
    # Kernel weights: an exponential of a rounded difference (|x| <= 24 here: 24 * 2^-24 of the
    # value, plus 2 units = 2^-22), a sum of at most 32 terms in a tree (5 * 2^-24), two
    # divisions and the scale (3 * 2^-24): below 40 * 2^-24 relative.
    bound = 40 * 2.0 ** -24 * ref.abs() + 1e-37 * scale
    assert ((got - ref).abs() <= bound).all(), ((got - ref).abs() / bound).max()


def _check(x, k, train=True, **kw):
    kw_b = {n: kw[n] for n in ('scoring', 'renormalize', 'scale') if n in kw}
    bias = kw.pop('bias', None)
    idx, w = router_gate(x.cuda(), k, bias=None if bias is None else bias.cuda(), **kw)
    ridx, rw = router_gate_reference(x, k, bias=bias, **kw)
    assert torch.equal(idx.cpu(), ridx)
    _close_w(w.cpu(), rw, kw.get('scale', 1.0))
    if not train:
        return
    g = torch.Generator().manual_seed(7)
    dw = torch.randn(*idx.shape, generator=g)
    d = router_gate_bwd(x.cuda(), idx, dw.cuda(), **kw_b)
    ref = router_gate_bwd_reference(x.double(), ridx, dw, **kw_b)
    # each gradient is p * (dw - sum p dw): the errors of p and of the sum (48 * 2^-24 together with
    # 1 - s) apply to |dw| + sum p |dw| <= 2 max|dw|, with p <= 1; then one rounding to the type
    top = 2 * dw.abs().amax(1, keepdim=True).double() * kw.get('scale', 1.0)
    bound = 96 * 2.0 ** -24 * top + torch.finfo(x.dtype).eps / 2 * ref.abs() + torch.finfo(x.dtype).tiny
    assert d.dtype == x.dtype
    assert ((d.cpu().double() - ref).abs() <= bound).all()


@pytest.mark.gpu
@needs_cuda
@pytest.mark.parametrize('scoring', ['sigmoid', 'softmax'])
@pytest.mark.parametrize('renorm', [True, False])
@pytest.mark.parametrize('E,K,n,g', [(256, 8, 8, 4), (160, 6, 8, 3), (8, 2, 1, 1), (1, 1, 1, 1), (33, 5, 3, 2),
                                     (512, 16, 16, 5), (1024, 32, 32, 7), (384, 8, 1, 1), (96, 32, 2, 2), (64, 4, 32, 2),
                                     (24, 3, 24, 5)])
@pytest.mark.parametrize('group_score,with_bias', [('top2', True), ('max', True), ('top2', False), ('max', False)])
def test_gate_matches_definition(scoring, renorm, E, K, n, g, group_score, with_bias):
    x = _logits(203, E, E + K, masked=0.2 if E > 8 else 0.0)
    bias = torch.randn(E, generator=torch.Generator().manual_seed(3)) * 0.1 if with_bias else None
    _check(x, K, scoring=scoring, bias=bias, num_groups=n, topk_groups=g, group_score=group_score, renormalize=renorm,
           scale=2.5)


@pytest.mark.gpu
@needs_cuda
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('scoring', ['sigmoid', 'softmax'])
def test_gate_16_bit_logits_with_many_ties(dtype, scoring):
    # 16-bit logits on a coarse grid: most rows have equal logits at the border
    x = (_logits(400, 128, 5) * 4).round().div(4).to(dtype)
    for n, g in ((1, 1), (4, 2)):
        for group_score in ('top2', 'max'):
            _check(x, 8, scoring=scoring, num_groups=n, topk_groups=g, group_score=group_score)
            _check(x, 8, scoring=scoring, num_groups=n, topk_groups=g, group_score=group_score, renormalize=False,
                   bias=torch.zeros(128))


@pytest.mark.gpu
@needs_cuda
def test_gate_near_ties_are_decided_as_in_fp64():
    # scores of trained gates saturate: logits near 15 differ by 2^-20 of each other, their
    # sigmoids by less than a 32-bit rounding
    g = torch.Generator().manual_seed(2)
    x = 15 + torch.randint(0, 64, (500, 96), generator=g).float() * 2.0 ** -16
    _check(x, 8, bias=torch.zeros(96), train=False)
    _check(x, 8, num_groups=6, topk_groups=3, train=False)
    bias = torch.randint(0, 3, (96,), generator=g).float() * 1e-7
    _check(x, 8, bias=bias, train=False)
    _check(x, 8, bias=bias * 1e4, num_groups=6, topk_groups=3, train=False)
    y = _logits(500, 96, 9, spread=1e-5)
    _check(y, 8, scoring='softmax', bias=bias, train=False)


@pytest.mark.gpu
@needs_cuda
def test_gate_edge_rows():
    x = _logits(64, 40, 11, masked=0.6)
    x[0] = -INF
    x[1] = math.nan
    x[2, 3] = INF
    x[3] = -200.0            # every sigmoid underflows in fp32: the weights are still a distribution
    x[4] = torch.finfo(torch.float32).min
    x[5, ::2] = -0.0
    x[5, 1::2] = 0.0
    x[6] = 80.0
    bias = torch.randn(40, generator=torch.Generator().manual_seed(1))
    bias[7], bias[9] = -INF, INF
    for scoring in ('sigmoid', 'softmax'):
        for renorm in (True, False):
            for b in (None, bias):
                _check(x, 6, scoring=scoring, renormalize=renorm, bias=b, num_groups=4, topk_groups=2)
                _check(x, 6, scoring=scoring, renormalize=renorm, bias=b)


@pytest.mark.gpu
@needs_cuda
def test_gate_strides_sizes_streams_and_graphs():
    base = torch.randn(70, 300, generator=torch.Generator().manual_seed(4)).cuda()
    x = base[3:68, 17:17 + 96]                       # unaligned rows, a stride of its own
    idx, w = router_gate(x, 4, num_groups=4, topk_groups=2)
    ridx, rw = router_gate_reference(x.cpu(), 4, num_groups=4, topk_groups=2)
    assert torch.equal(idx.cpu(), ridx)
    for T in (0, 1, 2, 5):
        idx, w = router_gate(base[:T], 8)
        assert idx.shape == (T, 8) and torch.equal(idx.cpu(), router_gate_reference(base[:T].cpu(), 8)[0])
        assert router_gate_bwd(base[:T], idx, w).shape == (T, 300)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        idx_s, w_s = router_gate(x, 4, num_groups=4, topk_groups=2)
    s.synchronize()
    assert torch.equal(idx_s.cpu(), ridx)
    static = x.contiguous()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gi, gw = router_gate(static, 4, num_groups=4, topk_groups=2)
        gd = router_gate_bwd(static, gi, gw)
    static.copy_(static.roll(1, 0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(gi.cpu(), ridx.roll(1, 0))
    assert torch.equal(gd, router_gate_bwd(static, gi, gw))


@pytest.mark.gpu
@needs_cuda
def test_gate_gradient_of_given_ids():
    # ids from elsewhere: the same id twice adds up, ids out of range count for nothing
    x = _logits(50, 48, 21)
    g = torch.Generator().manual_seed(5)
    idx = torch.randint(-2, 52, (50, 6), generator=g)
    idx[:, 1] = idx[:, 0]
    dw = torch.randn(50, 6, generator=g)
    for scoring in ('sigmoid', 'softmax'):
        got = router_gate_bwd(x.cuda(), idx.cuda(), dw.cuda(), scoring, False, 1.5)
        ref = router_gate_bwd_reference(x.double(), idx, dw, scoring, False, 1.5)
        assert torch.allclose(got.cpu().double(), ref, atol=96 * 2.0 ** -24 * 2 * 6 * dw.abs().max().item() * 1.5)


@pytest.mark.gpu
@needs_cuda
def test_gate_refusals_on_cuda():
    _refusals('cuda')
    x = torch.zeros(4, 12, device='cuda')
    with pytest.raises(RuntimeError):
        router_gate(x, 2, bias=torch.zeros(12))
    with pytest.raises(RuntimeError):
        router_gate_bwd(x, torch.zeros(4, 2, dtype=torch.long), x[:, :2])
