"""Calls of the fp8 block GEMM that give up: they return, say so, and leave nothing behind for the next call."""
import pytest
import torch

from deepep_trn_b200.ops import gemm
from test_gemm_block import _masked_case, _rows, _segment_case, _segments, _weight

pytestmark = pytest.mark.gpu
needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')


@needs_cuda
@pytest.mark.parametrize('epilogue', ['bf16', 'swiglu'])
@pytest.mark.parametrize('counts,N,K', [
    ([1], 512, 256),                 # one tile, fewer K blocks than stages: all copies leave before anything runs out
    ([3], 2048, 2320),               # clusters divide K
    ([300, 31], 512, 400),           # groups with many rows, few K blocks
    ([700, 0, 1300], 1024, 2048),    # several tiles a CTA
])
def test_segments_without_a_budget(counts, N, K, epilogue):
    g = torch.Generator().manual_seed(N + K)
    q, sc = _rows((sum(counts) + 2,), K, g)
    B, sb = _weight(len(counts), N, K, g)
    args = [t.cuda() for t in (q, sc, B, sb, _segments(counts, 1))]
    out = torch.full((sum(counts) + 2, N), 7.0, dtype=torch.bfloat16, device='cuda')
    gemm.check()
    for _ in range(3):
        gemm.grouped_gemm_fp8_block(*args, out=out, epilogue=epilogue, save_preact=True, timeout_s=0)
        with pytest.raises(RuntimeError, match='timed-out'):
            gemm.check()
        assert (out[0] == 7).all() and (out[-1] == 7).all()
    gemm.check()                     # the word is cleared by the report
    _segment_case(counts, N, K, epilogue, False, 'cuda', head=1, tail=1, seed=N)
    gemm.check()


@needs_cuda
@pytest.mark.parametrize('timeout_s', [0, -1.0, float('nan')])
def test_slabs_without_a_budget(timeout_s):
    # slabs of a decoding step that both kernels are launched for, on two streams
    counts = [55, 37, 2, 124, 33, 88, 113, 4, 82, 54, 62, 66, 126]
    g = torch.Generator().manual_seed(3)
    q, sc = (t.cuda() for t in _rows((13, 128), 1664, g))
    B, sb = (t.cuda() for t in _weight(13, 1024, 1664, g))
    cnt = torch.tensor(counts, dtype=torch.int32).cuda()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            gemm.grouped_gemm_fp8_block(q, sc, B, sb, counts=cnt, timeout_s=timeout_s)
    with pytest.raises(RuntimeError, match='timed-out'):
        torch.cuda.synchronize()
        gemm.check()
    _masked_case(counts, 128, 1024, 1664, 'bf16', 'cuda', seed=3)
    gemm.check()
