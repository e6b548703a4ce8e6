"""What a call of the fp8 block GEMM launches: forms, clusters and grids, and the SMs that it may hold."""
import pytest
import torch

from deepep_trn_b200.ops import available
from deepep_trn_b200.ops.gemm import fp8_block_plan

needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')
needs_ext = pytest.mark.skipif(not available(), reason='the extension is not built')
B200 = (148, 74, 36, 16)     # SMs, resident clusters of 2, 4 and 8 CTAs (as many as divide the SMs, or fewer)


@needs_ext
@pytest.mark.parametrize('num_sms', [0, 1, 8, 17, 100, 147, 148, 500])
@pytest.mark.parametrize('G,rows,N,K', [(32, 1024, 4096, 7168), (13, 128, 3584, 6656), (10, 128, 2304, 4480),
                                        (1, 1, 128, 16), (256, 64, 7168, 2048)])
@pytest.mark.parametrize('masked', [True, False])
def test_kernels_hold_no_more_sms_than_granted(num_sms, G, rows, N, K, masked):
    p = fp8_block_plan(G, rows, N, K, masked, num_sms, device=B200)
    granted = min(num_sms, 148) if num_sms > 0 else 148
    assert max(p['few_ctas'], p['many_ctas']) <= granted
    assert p['few_ctas'] % p['split'] == 0
    # side by side only where nothing is kept back
    assert p['overlap'] == (p['form'] == 'both' and granted == 148)
    if p['form'] == 'both':
        assert masked and p['few_ctas'] > 0 and p['many_ctas'] > 0


@needs_ext
def test_both_kernels_are_launched_for_decoding_slabs():
    assert fp8_block_plan(32, 1024, 4096, 7168, True, 0, device=B200)['form'] == 'both'
    assert fp8_block_plan(10, 128, 2304, 4480, True, 8, device=B200)['form'] == 'both'
    for bad in ((0, 1, 8, 16), (1, 0, 8, 16)):
        with pytest.raises(RuntimeError):
            fp8_block_plan(*bad, True, 0, device=B200)
    with pytest.raises(RuntimeError):
        fp8_block_plan(1, 1, 8, 16, True, 0, device=(148,))


@pytest.mark.gpu
@needs_cuda
@pytest.mark.parametrize('num_sms', [0, 8, 40])
def test_granted_sms_on_cuda(num_sms):
    from test_gemm_block import _masked_case
    counts = [57, 84, 18, 31, 61, 45, 68, 89, 59, 99]
    p = fp8_block_plan(10, 128, 2304, 4480, True, num_sms, counts)
    print(p)
    assert p['overlap'] == (num_sms == 0 and p['form'].startswith('both'))
    _masked_case(counts, 128, 2304, 4480, 'bf16', 'cuda', seed=1, num_sms=num_sms)
