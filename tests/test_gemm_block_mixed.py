"""Slabs of which some have few and some many rows: both kernels of the fp8 block GEMM work on one call, each on
its groups. The form is asked for, so that a change of the estimates cannot leave these cases without it."""
import pytest
import torch

from deepep_trn_b200.ops.gemm import check, fp8_block_plan, grouped_gemm_fp8_block
from test_gemm_block import _check, _expected, _masked_case, _rows, _weight

pytestmark = pytest.mark.gpu
needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')

# at the border of few rows (48), at tiles of many (128), empty, over-full and negative counts
WIDE = ([55, 37, 2, 124, 33, 88, 113, 4, 82, 54, 62, 66, 126], 128, 3584, 6656, 0)
BORDER = ([48, 49, 0, 128, 47, 200, 113, -1, 82, 54, 62, 66, 1], 128, 3584, 6656, 0)
NARROW = ([57, 84, 18, 31, 61, 45, 68, 89, 59, 99], 128, 2304, 4480, 8)     # few SMs: several rounds of either kernel


def _assert_mixed(counts, cap, N, K, num_sms):
    p = fp8_block_plan(len(counts), cap, N, K, True, num_sms, counts)
    assert p['form'] == 'both: mixed', p


@needs_cuda
@pytest.mark.parametrize('case,epilogue,kn', [(WIDE, 'bf16', False), (WIDE, 'swiglu', False), (WIDE, 'f32', True),
                                              (BORDER, 'f32', False), (BORDER, 'swiglu', False), (BORDER, 'bf16', True),
                                              (NARROW, 'swiglu', False), (NARROW, 'bf16', True)])
def test_each_kernel_takes_its_groups(case, epilogue, kn):
    counts, cap, N, K, num_sms = case
    _assert_mixed(*case)
    _masked_case(counts, cap, N, K, epilogue, 'cuda', kn=kn, seed=N + len(epilogue), num_sms=num_sms)
    check()


@needs_cuda
@pytest.mark.parametrize('case', [WIDE, NARROW])
def test_mixed_calls_side_by_side_and_in_graphs(case):
    counts, cap, N, K, num_sms = case
    _assert_mixed(*case)
    g = torch.Generator().manual_seed(12)
    q, sc = (t.cuda() for t in _rows((len(counts), cap), K, g))
    B, sb = (t.cuda() for t in _weight(len(counts), N, K, g))
    cnt = torch.tensor(counts, dtype=torch.int32).cuda()

    def call():
        out = torch.full((len(counts), cap, N), 7.0, dtype=torch.bfloat16, device='cuda')
        return grouped_gemm_fp8_block(q, sc, B, sb, counts=cnt, out=out, num_sms=num_sms)

    ref = call()
    for e, n in enumerate(counts):
        assert (ref[e, n:] == 7).all()
        if e % 4 == 0:
            _check(ref[e, :n], *_expected(q[e:e + 1].cpu(), sc[e:e + 1].cpu(), B[e:e + 1].cpu(), sb[e:e + 1].cpu(),
                                          (0, slice(0, n)), 0, False), K)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for i in range(9):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs)
    graphs, held = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(call())
            held.append(call())
        graphs.append(graph)
    cnt.copy_(torch.tensor(counts[::-1], dtype=torch.int32))     # the device decides at each replay
    for graph, s in zip(graphs, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    want = call()
    assert all(torch.equal(h, want) for h in held)
    check()
