"""The expert gate's selection where 32 bits cannot tell: group sums that cancel, biases of the type's lowest
value, experts at the same score. Ids have to equal those of the definition in fp64."""
import math

import pytest
import torch

from deepep_trn_b200.ops.moe_ops import router_gate
from deepep_trn_b200.utils.testing import router_gate_reference

pytestmark = pytest.mark.gpu
needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')


def _same_ids(x, k, **kw):
    bias = kw.pop('bias')
    idx, _ = router_gate(x.cuda(), k, bias=bias.cuda(), **kw)
    ref, _ = router_gate_reference(x, k, bias=bias, **kw)
    wrong = (idx.cpu() != ref).any(1)
    assert not wrong.any(), (int(wrong.sum()), wrong.nonzero()[:4].flatten().tolist())


@needs_cuda
@pytest.mark.parametrize('scoring', ['sigmoid', 'softmax'])
@pytest.mark.parametrize('size', [1e2, 1e4, 1e6])
def test_group_sums_that_cancel(scoring, size):
    # A bias of +size and -size in each group of two: the sums are of order 1, their summands rounded to the
    # spacing of fp32 at `size`. Of 2 million rows at 1e4 about 160 come out as certain and wrong where the
    # bound goes with the sum (counted with ideal fp32 scores).
    x = torch.randn(2_000_000, 4, generator=torch.Generator().manual_seed(1))
    bias = torch.tensor([size, -size, size, -size])
    _same_ids(x, 2, scoring=scoring, bias=bias, num_groups=2, topk_groups=1)


@needs_cuda
@pytest.mark.parametrize('E,n,g', [(256, 8, 4), (160, 8, 3), (96, 32, 7), (48, 4, 1)])
def test_group_sums_that_cancel_in_wide_rows(E, n, g):
    # groups in whole lanes and groups through shared memory
    x = torch.randn(100000, E, generator=torch.Generator().manual_seed(E))
    bias = torch.full((E,), -1e4)
    bias[::E // n] = 1e4
    _same_ids(x, 2, scoring='sigmoid', bias=bias, num_groups=n, topk_groups=g)


@needs_cuda
@pytest.mark.parametrize('scoring', ['sigmoid', 'softmax'])
@pytest.mark.parametrize('group_score', ['top2', 'max'])
@pytest.mark.parametrize('E,n', [(16, 4), (256, 8), (160, 8), (6, 3)])
def test_biases_of_the_lowest_value(scoring, group_score, E, n):
    # closed by the lowest value an expert comes last, but is available: two of them add up to less than fp32
    # holds, and their group still comes before one that has nothing left
    low = torch.finfo(torch.float32).min
    x = torch.randn(3000, E, generator=torch.Generator().manual_seed(E))
    gs = E // n
    bias = torch.zeros(E)
    bias[gs:2 * gs] = low
    bias[2 * gs:3 * gs] = -math.inf
    if n > 3:
        bias[3 * gs:4 * gs] = low
    for g, k in ((1, 1), (2, gs + 1), (n, min(32, 2 * gs))):
        _same_ids(x, min(k, 32, g * gs), scoring=scoring, bias=bias, num_groups=n, topk_groups=g,
                  group_score=group_score)
    bias[:gs] = low
    _same_ids(x, min(gs, 32), scoring=scoring, bias=bias, num_groups=n, topk_groups=2, group_score=group_score)
    bias = torch.full((E,), low)
    bias[::gs] = 0.25      # one open expert a group
    _same_ids(x, 2, scoring=scoring, bias=bias, num_groups=n, topk_groups=2, group_score=group_score)
    high = torch.finfo(torch.float32).max
    bias[1::gs] = high
    bias[::gs] = high
    _same_ids(x, 2, scoring=scoring, bias=bias, num_groups=n, topk_groups=2, group_score=group_score)
