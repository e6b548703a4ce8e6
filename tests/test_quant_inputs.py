"""Inputs of the row quantiser: types, and tensors that start anywhere."""
import pytest
import torch

from deepep_trn_b200.ops.quant import dequantize_fp8, quantize_fp8
from deepep_trn_b200.utils.codec import dequantize_fp8_1x128, quantize_fp8_1x128

pytestmark = pytest.mark.gpu
needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')


@needs_cuda
@pytest.mark.parametrize('dtype', [torch.float32, torch.float64, torch.uint8, torch.int16])
def test_other_types_are_refused(dtype):
    with pytest.raises(RuntimeError):
        quantize_fp8(torch.ones(4, 128, device='cuda').to(dtype))


@needs_cuda
@pytest.mark.parametrize('offset', [0, 1, 3, 4])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_tensors_that_start_anywhere(offset, dtype):
    store = torch.randn(9 * 256 + 8, generator=torch.Generator().manual_seed(offset)).to(dtype).cuda()
    x = store[offset:offset + 9 * 256].view(9, 256)
    q, s = quantize_fp8(x)
    rq, rs = quantize_fp8_1x128(x.cpu())
    assert torch.equal(s.cpu(), rs) and torch.equal(q.cpu().view(torch.uint8), rq.view(torch.uint8))
    bytes_ = torch.zeros(9 * 256 + 8, dtype=torch.uint8, device='cuda')
    moved = bytes_[offset:offset + 9 * 256].view(9, 256)
    moved.copy_(q.view(torch.uint8))
    out = dequantize_fp8(moved.view(torch.float8_e4m3fn), s)
    assert torch.equal(out.cpu(), dequantize_fp8_1x128(rq, rs).to(torch.bfloat16))
