"""The expert operators where element offsets pass 32 bits, and captured calls whose offsets change."""
import pytest
import torch

from deepep_trn_b200.ops import gemm
from deepep_trn_b200.ops.moe_ops import router_gate, router_gate_bwd
from deepep_trn_b200.ops.quant import quantize_fp8
from deepep_trn_b200.utils.codec import quantize_fp8_1x128, quantize_fp8_128x128
from deepep_trn_b200.utils.testing import router_gate_bwd_reference, router_gate_reference
from test_gemm_block import _check, _expected, _rows, _weight

pytestmark = pytest.mark.gpu
needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')
F8 = torch.float8_e4m3fn


@needs_cuda
def test_gate_of_more_than_2_to_31_logits():
    T, E = 2_200_000, 1024                                # 2.25e9 logits
    g = torch.Generator(device='cuda').manual_seed(1)
    part = torch.randn(1000, E, generator=g, device='cuda').bfloat16()
    x = part.repeat(T // 1000, 1)
    idx, w = router_gate(x, 8, 'softmax', num_groups=8, topk_groups=4, renormalize=False)
    ridx, rw = router_gate_reference(part.cpu(), 8, 'softmax', num_groups=8, topk_groups=4, renormalize=False)
    dw = torch.randn(1000, 8, generator=g, device='cuda')
    d = router_gate_bwd(x, idx, dw.repeat(T // 1000, 1), 'softmax', False)
    first, last = slice(0, 1000), slice(T - 1000, T)
    assert torch.equal(idx[first].cpu(), ridx) and torch.equal(idx[last], idx[first])
    assert torch.equal(w[last], w[first]) and torch.equal(d[last], d[first])
    ref = router_gate_bwd_reference(part.cpu(), ridx, dw.cpu(), 'softmax', False)
    assert torch.allclose(d[last].float().cpu(), ref.float(), rtol=2 ** -7, atol=1e-5)


@needs_cuda
@pytest.mark.parametrize('epilogue', ['f32', 'swiglu'])
def test_product_of_more_than_2_to_31_values(epilogue):
    rows, N, K = 301_000, 7168, 128                       # 2.16e9 values
    g = torch.Generator().manual_seed(2)
    q, sc = _rows((1000,), K, g)
    B, sb = _weight(2, N, K, g)
    a, sa = q.cuda().view(torch.uint8).repeat(301, 1).view(F8), sc.cuda().repeat(301, 1)
    offs = torch.tensor([0, 1000, rows], device='cuda')
    out = gemm.grouped_gemm_fp8_block(a, sa, B.cuda(), sb.cuda(), offs, epilogue=epilogue, save_preact=True)
    c = out if epilogue == 'f32' else out[2]
    assert c.numel() > 2 ** 31
    for e, at in ((0, slice(0, 1000)), (1, slice(1000, 2000)), (1, slice(rows - 1000, rows))):
        _check(c[at], *_expected(q, sc, B, sb, slice(0, 1000), e, False), K)
    if epilogue == 'swiglu':
        for t in out[:2]:
            assert torch.equal(t.view(torch.uint8)[1000:2000], t.view(torch.uint8)[rows - 1000:])


@needs_cuda
def test_quantisers_of_more_than_2_to_31_values():
    part = torch.randn(1024, 32768, generator=torch.Generator().manual_seed(3)).bfloat16()
    x = part.cuda().repeat(66, 1)                         # 2.2e9 values
    for call, definition in ((gemm.quantize_fp8_weight, quantize_fp8_128x128), (quantize_fp8, quantize_fp8_1x128)):
        q, s = call(x)
        rq, rs = definition(part)
        for at, sat in ((slice(0, 1024), slice(0, rs.shape[0])), (slice(-1024, None), slice(-rs.shape[0], None))):
            assert torch.equal(q.view(torch.uint8)[at].cpu(), rq.view(torch.uint8)) and torch.equal(s[sat].cpu(), rs)
        del q, s


@needs_cuda
@pytest.mark.parametrize('rows,N,K', [(40, 512, 4112), (1500, 512, 400)])     # clusters that divide K; many rows
def test_replays_with_other_offsets(rows, N, K):
    # the launch is shaped by the rows that there are; which group has them is read at each replay
    g = torch.Generator().manual_seed(rows)
    q, sc = _rows((rows,), K, g)
    B, sb = _weight(5, N, K, g)
    args = [t.cuda() for t in (q, sc, B, sb)]
    r = rows // 5
    offs = torch.tensor([0, r, 2 * r, 3 * r, 4 * r, rows], device='cuda')
    assert gemm.fp8_block_plan(5, rows, N, K, False)['form'] == ('few' if rows == 40 else 'many')
    out = torch.empty(rows, N, device='cuda')
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gemm.grouped_gemm_fp8_block(*args, offs, out=out, epilogue='f32')
    for new in ([0, r, 2 * r, 3 * r, 4 * r, rows], [0, 0, 0, rows, rows, rows], [0, 1, 2, 3, 4, rows],
                [3, 3, 3, 3, 3, rows - 1], [0, 0, 0, 0, 0, 0], [0, rows - 4, rows - 3, rows - 2, rows - 1, rows]):
        offs.copy_(torch.tensor(new))
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        used = torch.zeros(rows, dtype=torch.bool)
        for e in range(5):
            at = slice(new[e], new[e + 1])
            used[at] = True
            if new[e + 1] > new[e]:
                _check(out[at], *_expected(q, sc, B, sb, at, e, False), K)
        assert (out.cpu()[~used] == 7).all()
    gemm.check()
