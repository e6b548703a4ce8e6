"""The first product of a process inside of a capture: its error word belongs to the process, not to the graph."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')
CHILD = """
import torch
from deepep_trn_b200.ops import gemm
A = torch.randn(256, 512, device='cuda').bfloat16()
B = torch.randn(2, 256, 512, device='cuda').bfloat16()
offs = torch.tensor([0, 128, 256], device='cuda')
pool = torch.cuda.graph_pool_handle()
first = torch.cuda.CUDAGraph()
with torch.cuda.graph(first, pool=pool):
    for _ in range(64):             # the pool's free memory is full of ones, word after word
        held = torch.full((1,), -1, dtype=torch.int32, device='cuda')
    held = [torch.full((1,), -1, dtype=torch.int32, device='cuda') for _ in range(64)]
first.replay()
torch.cuda.synchronize()
del held
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, pool=pool):
    out = CALL
gemm.check()                        # nothing has run yet, and nothing has gone wrong
want = CALL
gemm.check()
graph.replay()
torch.cuda.synchronize()
gemm.check()
assert torch.equal(out, want)
gemm.grouped_gemm(A, B, offs, timeout_s=0)
graph.replay()                      # a replay does not take back what was reported
torch.cuda.synchronize()
try:
    gemm.check()
    raise SystemExit('the report is lost')
except RuntimeError:
    pass
print('done')
"""
BLOCK = ('gemm.grouped_gemm_fp8_block(A.to(torch.float8_e4m3fn), torch.ones(256, 4, device="cuda"), '
         'B.to(torch.float8_e4m3fn), torch.ones(2, 2, 4, device="cuda"), offs)')


@needs_cuda
@pytest.mark.parametrize('call', ['gemm.grouped_gemm(A, B, offs)', BLOCK])
def test_first_call_in_a_capture(call):
    p = subprocess.run([sys.executable, '-c', CHILD.replace('CALL', call)], capture_output=True, text=True, timeout=200,
                       cwd=str(Path(__file__).resolve().parents[1]))
    assert p.returncode == 0 and 'done' in p.stdout, p.stdout + p.stderr


@needs_cuda
def test_check_names_a_device_in_any_way():
    from deepep_trn_b200.ops import gemm
    A = torch.zeros(128, 64, device='cuda', dtype=torch.bfloat16)
    for device in (None, 'cuda', 'cuda:0', torch.device('cuda'), torch.device('cuda', 0)):
        gemm.grouped_gemm(A, A[None], torch.tensor([0, 128], device='cuda'), timeout_s=0)
        with pytest.raises(RuntimeError):
            gemm.check(device)
        gemm.check(device)
