"""Calls of the bf16 and power-of-two fp8 grouped GEMMs that give up: they return, say so, and leave nothing
behind for the next call."""
import pytest
import torch

from deepep_trn_b200.ops import gemm

pytestmark = pytest.mark.gpu
needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')


@needs_cuda
@pytest.mark.parametrize('K', [128, 2048])     # fewer K blocks than stages: all copies leave before anything runs out
@pytest.mark.parametrize('op', ['nk', 'kn', 'swiglu', 'fp8', 'wgrad', 'wgrad_mk'])
def test_call_without_a_budget(op, K):
    torch.manual_seed(0)
    N, offs = 512, torch.tensor([0, 128, 128, 640], device='cuda')
    A = (torch.randn(640, K, device='cuda') * 0.5).to(torch.bfloat16)
    B = (torch.randn(3, *((K, N) if op == 'kn' else (N, K)), device='cuda') * 0.05).to(torch.bfloat16)
    D = torch.randn(640, N, device='cuda').to(torch.bfloat16)
    if op == 'fp8':
        a, b = gemm.quantize_fp8_blocks(A), gemm.quantize_fp8_blocks(B)
        call = lambda t: gemm.grouped_gemm_fp8(a[0], a[1], b[0], b[1], offs, timeout_s=t)  # noqa: E731
    elif op == 'wgrad':
        call = lambda t: gemm.grouped_gemm_wgrad(A, D, offs, timeout_s=t)  # noqa: E731
    elif op == 'wgrad_mk':
        At, Dt = A.t().contiguous(), D.t().contiguous()
        call = lambda t: gemm.grouped_gemm_wgrad(At, Dt, offs, timeout_s=t, layout='mk')  # noqa: E731
    elif op == 'swiglu':
        call = lambda t: gemm.grouped_gemm(A, B, offs, epilogue='swiglu', timeout_s=t)[1]  # noqa: E731
    else:
        call = lambda t: gemm.grouped_gemm(A, B, offs, b_layout=op, timeout_s=t)  # noqa: E731
    want = call(10.0)
    gemm.check()
    for _ in range(3):
        call(0)
        with pytest.raises(RuntimeError, match='timed-out'):
            gemm.check()
    gemm.check()
    assert torch.equal(call(10.0), want)
    gemm.check()
