"""The fp8 expert products with one fp32 scale per block of 128 and the weight quantiser: the torch
definitions on the CPU, and the kernels against fp64."""
import pytest
import torch

from deepep_trn_b200.ops.gemm import deinterleave, grouped_gemm_fp8_block, quantize_fp8_weight
from deepep_trn_b200.utils.codec import dequantize_fp8_128x128, quantize_fp8_1x128, quantize_fp8_128x128

needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')
F8 = torch.float8_e4m3fn


def _rows(shape, K, g):
    """e4m3 rows and scales of a random matrix whose blocks differ in magnitude (K may end in a block)."""
    x = torch.randn(*shape, K, generator=g)
    KB = -(-K // 128)
    x = x * torch.pow(10.0, torch.rand(*shape, KB, generator=g) * 3 - 1.5).repeat_interleave(128, -1)[..., :K]
    xp = torch.nn.functional.pad(x, (0, -K % 128))
    q, sc = quantize_fp8_1x128(xp)
    return q[..., :K].contiguous(), sc


def _weight(G, N, K, g):
    w = torch.randn(G, N, K, generator=g)
    NB, KB = -(-N // 128), -(-K // 128)
    f = torch.pow(10.0, torch.rand(G, NB, KB, generator=g) * 2 - 1)
    return quantize_fp8_128x128(w * f.repeat_interleave(128, 1).repeat_interleave(128, 2)[:, :N, :K])


def _deq(q, sc):
    return q.double() * sc.double().repeat_interleave(128, -1)[..., :q.shape[-1]]


def _expected(q, sc, B, sb, at, g, kn):
    """fp64 product of group g's rows, and the sums of the products' magnitudes."""
    a = _deq(q[at], sc[at])
    w = dequantize_fp8_128x128(B[g], sb[g]).double()
    w = w if kn else w.t()
    return a @ w, a.abs() @ w.abs()


def _bound(ref, mag, K, dtype):
    # Within a block the tensor cores add 128 exact products in fp32, perhaps truncating
    # (2^-23 each); the block's scale is a rounded product (2^-24) and every block is added with one
    # rounding (2^-24): (128 + ceil(K / 128) + 2) * 2^-23 of the sum of magnitudes. Then one
    # rounding to the output's type.
    return (130 + -(-K // 128)) * 2.0 ** -23 * mag + torch.finfo(dtype).eps / 2 * ref.abs() + 1e-37


def _check(out, ref, mag, K):
    err = (out.double().cpu() - ref).abs()
    bound = _bound(ref, mag, K, out.dtype)
    assert (err <= bound).all(), (err / bound).max().item()


def _check_swiglu(h, hs, pre, ref, mag, K):
    """h, its scales and the pre-activation against fp64 (rows of one group)."""
    gate, up = deinterleave(ref)
    mg, mu = deinterleave(_bound(ref, mag, K, torch.float64))
    s = torch.sigmoid(gate)
    want = gate * s * up
    # |silu'| <= 1.1, |silu(g)| <= |g|; exp, quotient and products: 8 * 2^-23, and the exponential of
    # a rounded argument |g| * 2^-23
    dh = 1.1 * mg * up.abs() + gate.abs() * mu + mg * mu + (8 + gate.abs()) * 2.0 ** -23 * want.abs()
    R, I = want.shape
    amax = want.abs().reshape(R, I // 128, 128).amax(-1).clamp_min(1e-4)
    dmax = dh.reshape(R, I // 128, 128).amax(-1)
    hs = hs.double().cpu()
    assert ((hs - amax / 448).abs() <= dmax / 448 + 2.0 ** -23 * amax / 448).all()
    # e4m3: half a step is 2^-4 of the value, 2^-10 below the normal range, in units of the scale;
    # the scaled value carries two roundings (2^-23)
    sc = hs.repeat_interleave(128, -1)
    got = h.double().cpu() * sc
    assert ((got - want).abs() <= dh * 1.07 + want.abs() * (2.0 ** -4 + 2.0 ** -22) + sc * 2.0 ** -10).all()
    if pre is not None:
        _check(pre, ref, mag, K)


def _run(q, sc, B, sb, epilogue='bf16', kn=False, offsets=None, counts=None, dev='cuda', **kw):
    put = lambda t: None if t is None else t.to(dev)  # noqa: E731
    return grouped_gemm_fp8_block(put(q), put(sc), put(B), put(sb), put(offsets), put(counts), epilogue=epilogue,
                                  b_layout='kn' if kn else 'nk', **kw)


def _segments(counts, head=0):
    return torch.tensor([head] + [head + sum(counts[:i + 1]) for i in range(len(counts))], dtype=torch.int64)


def _segment_case(counts, N, K, epilogue, kn, dev, head=0, tail=0, limit=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    G = len(counts)
    offs = _segments(counts, head)
    rows = int(offs[-1]) + tail
    q, sc = _rows((rows,), K, g)
    B, sb = _weight(G, *((K, N) if kn else (N, K)), g)
    q.view(torch.uint8)[:head] = 0x7F          # NaN in rows that belong to no group
    q.view(torch.uint8)[rows - tail:] = 0x7F
    cnt = None if limit is None else torch.tensor(limit, dtype=torch.int32)
    kw = {}
    if epilogue == 'swiglu':
        kw = dict(h_out=torch.full((rows, N // 2), 0x11, dtype=torch.uint8, device=dev).view(F8),
                  h_scales=torch.full((rows, N // 256), 7.0, device=dev),
                  out=torch.full((rows, N), 7.0, dtype=torch.bfloat16, device=dev), save_preact=True)
    else:
        kw = dict(out=torch.full((rows, N), 7.0, dtype=torch.float32 if epilogue == 'f32' else torch.bfloat16,
                                 device=dev))
    res = _run(q, sc, B, sb, epilogue, kn, offs, cnt, dev, **kw)
    written = torch.zeros(rows, dtype=torch.bool)
    for e in range(G):
        n = counts[e] if limit is None else max(0, min(counts[e], limit[e]))
        at = slice(int(offs[e]), int(offs[e]) + n)
        written[at] = True
        if n == 0:
            continue
        ref, mag = _expected(q, sc, B, sb, at, e, kn)
        if epilogue == 'swiglu':
            _check_swiglu(res[0][at], res[1][at], res[2][at], ref, mag, K)
        else:
            _check(res[at], ref, mag, K)
    # every other row is as it was
    if epilogue == 'swiglu':
        assert (res[0].view(torch.uint8).cpu()[~written] == 0x11).all() and (res[1].cpu()[~written] == 7).all()
        assert (res[2].float().cpu()[~written] == 7).all()
    else:
        assert (res.float().cpu()[~written] == 7).all()


CASES = [
    ([1], 8, 16, 'f32', False, {}),
    ([1], 2048, 7168, 'bf16', False, {}),
    ([17], 264, 128, 'bf16', False, {}),
    ([128, 0, 256], 256, 256, 'f32', False, {}),
    ([5, 0, 130, 1, 127, 129], 264, 400, 'f32', False, dict(head=3, tail=9)),
    ([5, 0, 130, 1, 127, 129], 272, 400, 'bf16', True, dict(head=3, tail=9)),
    ([300, 31], 144, 1040, 'f32', True, {}),
    ([64, 200], 1000, 272, 'bf16', False, dict(limit=[40, 500])),
    ([64, 200], 512, 272, 'swiglu', False, dict(limit=[64, -3], tail=5)),
    ([5, 0, 130, 1, 127, 129], 512, 640, 'swiglu', False, dict(head=130)),
    ([33, 95], 256, 128, 'swiglu', False, {}),
]


@pytest.mark.parametrize('counts,N,K,epilogue,kn,kw', CASES[:1] + CASES[2:])
def test_block_definition_on_cpu(counts, N, K, epilogue, kn, kw):
    _segment_case(counts, N, K, epilogue, kn, 'cpu', **kw)


@pytest.mark.gpu
@needs_cuda
@pytest.mark.parametrize('counts,N,K,epilogue,kn,kw', CASES)
def test_block_segments(counts, N, K, epilogue, kn, kw):
    _segment_case(counts, N, K, epilogue, kn, 'cuda', **kw)


@pytest.mark.gpu
@needs_cuda
@pytest.mark.parametrize('epilogue,kn', [('bf16', False), ('swiglu', False), ('bf16', True), ('f32', True)])
def test_block_long_reduction(epilogue, kn):
    _segment_case([200, 56, 128], 512, 7168, epilogue, kn, 'cuda', seed=3)


@pytest.mark.gpu
@needs_cuda
@pytest.mark.parametrize('epilogue,kn,N', [('bf16', False, 264), ('swiglu', False, 1024), ('f32', True, 272),
                                          ('f32', False, 2560)])
@pytest.mark.parametrize('counts', [[1], [64], [65, 3], [300], [17, 0, 64, 90]])
def test_block_few_rows_divide_k(counts, epilogue, kn, N):
    # few tiles: clusters divide K (19 blocks, so that the shares differ and end inside a scale unit)
    _segment_case(counts, N, 2320, epilogue, kn, 'cuda', seed=N)


@pytest.mark.gpu
@needs_cuda
@pytest.mark.parametrize('epilogue,G,N,K,num_sms', [
    ('bf16', 3, 768, 2048, 8), ('swiglu', 5, 1024, 1920, 8), ('f32', 9, 256, 7168, 16),   # clusters, several rounds
    ('swiglu', 17, 2560, 2048, 0), ('bf16', 40, 2560, 1024, 0)])
def test_block_few_rows_many_rounds(epilogue, G, N, K, num_sms):
    # slabs of a decoding step: every CTA or cluster works through several tiles
    g = torch.Generator().manual_seed(N)
    counts = torch.randint(0, 50, (G,), generator=g).tolist()
    _masked_case(counts, 64, N, K, epilogue, 'cuda', seed=N, num_sms=num_sms, pre=G % 2 == 0)


@pytest.mark.gpu
@needs_cuda
@pytest.mark.parametrize('epilogue', ['bf16', 'swiglu'])
def test_block_both_forms_in_one_call(epilogue):
    # groups with few and with many rows, more tiles than SMs of each
    _segment_case([1, 400, 64, 0, 65, 1100, 30, 512, 7] * 4, 1280, 400, epilogue, False, 'cuda', seed=6, head=2, tail=3)


@pytest.mark.gpu
@needs_cuda
def test_block_many_groups():
    _segment_case([i % 4 for i in range(1024)], 64, 128, 'f32', False, 'cuda', seed=4)
    _segment_case([3, 0, 200, 64] * 40, 128, 256, 'bf16', True, 'cuda', seed=5)


def _masked_case(counts, cap, N, K, epilogue, dev, strided=False, kn=False, seed=0, num_sms=0, pre=True):
    g = torch.Generator().manual_seed(seed)
    G = len(counts)
    q, sc = _rows((G, cap), K, g)
    B, sb = _weight(G, *((K, N) if kn else (N, K)), g)
    cnt = torch.tensor(counts, dtype=torch.int32)
    for e, n in enumerate(counts):
        q.view(torch.uint8)[e, max(0, min(n, cap)):] = 0x7F
    if strided:   # slabs of a larger buffer, scales in rows of a wider one, as a low-latency receive hands them out
        big = torch.full((G, cap + 5, K + 16), 0x7F, dtype=torch.uint8)
        big[:, :cap, :K] = q.view(torch.uint8)
        q = big.to(dev).view(F8)[:, :cap, :K]
        wide = torch.full((G, cap + 3, sc.shape[-1] + 2), float('nan'))
        wide[:, :cap, :sc.shape[-1]] = sc
        sc = wide.to(dev)[:, :cap, :sc.shape[-1]]
        store = torch.full((G, cap + 2, N + 8), 7.0, dtype=torch.bfloat16, device=dev)
        kw = dict(out=store[:, :cap, :N])
    else:
        kw = dict(out=torch.full((G, cap, N), 7.0, dtype=torch.bfloat16, device=dev))
    if epilogue == 'swiglu':
        kw.update(h_out=torch.full((G, cap, N // 2), 0x11, dtype=torch.uint8, device=dev).view(F8),
                  h_scales=torch.full((G, cap, N // 256), 7.0, device=dev), save_preact=pre)
    if epilogue == 'f32':
        kw['out'] = kw['out'].float()
    res = _run(q, sc, B, sb, epilogue, kn, None, cnt, dev, num_sms=num_sms, **kw)
    for e, n in enumerate(counts):
        n = max(0, min(n, cap))
        out = res[2] if epilogue == 'swiglu' else res
        assert out is None or (out[e, n:].float() == 7).all()
        if epilogue == 'swiglu':
            assert (res[0].view(torch.uint8)[e, n:] == 0x11).all() and (res[1][e, n:] == 7).all()
        if n == 0:
            continue
        ref, mag = _expected(q[e:e + 1].cpu(), sc[e:e + 1].cpu(), B[e:e + 1], sb[e:e + 1], (0, slice(0, n)), 0, kn)
        if epilogue == 'swiglu':
            _check_swiglu(res[0][e, :n], res[1][e, :n], None if out is None else out[e, :n], ref, mag, K)
        else:
            _check(res[e, :n], ref, mag, K)
    if strided:
        assert (store[:, cap:].float() == 7).all() and (store[:, :, N:].float() == 7).all()


MASKED = [
    ([3, 0, 7, 1], 16, 256, 256, 'bf16', False),
    ([3, 0, 70, 128, 200, -1], 150, 512, 384, 'swiglu', False),
    ([3, 0, 70, 128, 200, 31], 150, 328, 400, 'bf16', True),
    ([1], 1, 256, 128, 'swiglu', True),
]


@pytest.mark.parametrize('counts,cap,N,K,epilogue,strided', MASKED)
def test_block_masked_definition_on_cpu(counts, cap, N, K, epilogue, strided):
    _masked_case(counts, cap, N, K, epilogue, 'cpu', strided)


@pytest.mark.gpu
@needs_cuda
@pytest.mark.parametrize('counts,cap,N,K,epilogue,strided', MASKED + [
    ([4, 9, 0, 31, 64, 65, 33, 16], 128, 512, 2048, 'swiglu', False),
    ([4, 9, 0, 31, 64, 65, 33, 16], 128, 1408, 512, 'bf16', True)])
def test_block_masked(counts, cap, N, K, epilogue, strided):
    _masked_case(counts, cap, N, K, epilogue, 'cuda', strided)


@pytest.mark.gpu
@needs_cuda
def test_block_masked_kn_and_no_counts():
    _masked_case([9, 0, 130], 130, 272, 400, 'bf16', 'cuda', kn=True)
    g = torch.Generator().manual_seed(8)
    q, sc = _rows((2, 40), 256, g)
    B, sb = _weight(2, 128, 256, g)
    out = _run(q, sc, B, sb, 'f32')      # without counts every row of the slabs is in use
    for e in range(2):
        ref, mag = _expected(q, sc, B, sb, (e, slice(0, 40)), e, False)
        _check(out[e], ref, mag, 256)


@pytest.mark.gpu
@needs_cuda
def test_block_offsets_out_of_range_are_clamped():
    g = torch.Generator().manual_seed(9)
    q, sc = _rows((100,), 256, g)
    B, sb = _weight(3, 128, 256, g)
    out = torch.full((100, 128), 7.0, device='cuda')
    _run(q, sc, B, sb, 'f32', offsets=torch.tensor([-5, 60, 40, 1000]), out=out)
    ref, mag = _expected(q, sc, B, sb, slice(0, 60), 0, False)
    _check(out[:40], ref[:40], mag[:40], 256)
    ref, mag = _expected(q, sc, B, sb, slice(60, 100), 2, False)
    _check(out[60:], ref, mag, 256)


@pytest.mark.gpu
@needs_cuda
def test_block_streams_graphs_and_concurrent_calls():
    g = torch.Generator().manual_seed(10)
    counts = [30, 0, 129, 64]
    offs = _segments(counts).cuda()
    q, sc = (t.cuda() for t in _rows((sum(counts),), 1024, g))
    B, sb = (t.cuda() for t in _weight(4, 512, 1024, g))
    ref = grouped_gemm_fp8_block(q, sc, B, sb, offs)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(grouped_gemm_fp8_block(q, sc, B, sb, offs))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs)
    static = q.clone()
    graphs, held = [], []
    for _ in range(2):     # two graphs of the same call, replayed side by side
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(grouped_gemm_fp8_block(static, sc, B, sb, offs))
        graphs.append(graph)
    for graph, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held[0], ref) and torch.equal(held[1], ref)


@pytest.mark.gpu
@needs_cuda
def test_block_slabs_on_streams_and_in_graphs():
    # slabs launch both kernels: side by side on three streams, and from two captured graphs
    g = torch.Generator().manual_seed(12)
    counts = torch.tensor([3, 0, 70, 128, 200, 31], dtype=torch.int32)
    q, sc = (t.cuda() for t in _rows((6, 200), 1024, g))
    B, sb = (t.cuda() for t in _weight(6, 512, 1024, g))
    cnt = counts.cuda()

    def call():
        out = torch.full((6, 200, 512), 7.0, dtype=torch.bfloat16, device='cuda')
        return grouped_gemm_fp8_block(q, sc, B, sb, counts=cnt, out=out)

    ref = call()
    for e, n in enumerate(counts.tolist()):
        assert (ref[e, n:] == 7).all()
        if n:
            _check(ref[e, :n], *_expected(q.cpu(), sc.cpu(), B.cpu(), sb.cpu(), (e, slice(0, n)), e, False), 1024)
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
        graphs.append(graph)
    cnt.copy_(counts.flip(0))
    for graph, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    want = call()
    assert torch.equal(held[0], want) and torch.equal(held[1], want)
    cnt.zero_()
    assert (call() == 7).all()


def _refusals(dev):
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=dev).view(F8)  # noqa: E731
    f = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
    a, sa, b, sb = u8(8, 256), f(8, 2), u8(2, 128, 256), f(2, 1, 2)
    offs = torch.tensor([0, 4, 8], device=dev)
    cnt = torch.zeros(2, dtype=torch.int32, device=dev)
    call = grouped_gemm_fp8_block
    w, sw = u8(2, 256, 256), f(2, 2, 2)
    cases = [
        (ValueError, lambda: call(a, sa, b, sb, offs, epilogue='gelu')),
        (ValueError, lambda: call(a, sa, b, sb, offs, b_layout='mn')),
        (RuntimeError, lambda: call(a, sa, b, sb)),                                  # 2-D without offsets
        (RuntimeError, lambda: call(a.view(2, 4, 256), sa.view(2, 4, 2), b, sb, offs)),
        (RuntimeError, lambda: call(u8(3, 4, 256), f(3, 4, 2), b, sb, counts=cnt)),  # slabs != groups
        (RuntimeError, lambda: call(a, sa, b, sb, offs[:2])),
        (RuntimeError, lambda: call(a, sa, b, sb, offs.int())),
        (RuntimeError, lambda: call(a, sa, b, sb, offs, cnt.long())),
        (RuntimeError, lambda: call(a, sa[:, :1], b, sb, offs)),
        (RuntimeError, lambda: call(a, sa.double(), b, sb, offs)),
        (RuntimeError, lambda: call(a, sa, b, sb[:, :, :1], offs)),
        (RuntimeError, lambda: call(a[:, :128], sa[:, :1], b, sb, offs)),            # K disagrees
        (RuntimeError, lambda: call(u8(8, 24), f(8, 1), u8(2, 128, 24), f(2, 1, 1), offs)),   # K % 16
        (RuntimeError, lambda: call(u8(8, 32), f(8, 1), u8(2, 12, 32), f(2, 1, 1), offs)),    # N % 8
        (RuntimeError, lambda: call(u8(8, 32), f(8, 1), u8(2, 32, 24), f(2, 1, 1), offs, b_layout='kn')),
        (RuntimeError, lambda: call(a, sa, b, sb, offs, epilogue='swiglu')),         # N % 256
        (RuntimeError, lambda: call(a, sa, w, sw, offs, epilogue='swiglu', b_layout='kn')),
        (RuntimeError, lambda: call(a, sa, b, sb, offs, out=f(8, 128))),             # fp32 out, bf16 epilogue
        (RuntimeError, lambda: call(a, sa, b, sb, offs, out=f(7, 128).bfloat16())),
        (RuntimeError, lambda: call(a, sa, b, sb, offs, out=f(8, 132).bfloat16()[:, 2:130])),
        (RuntimeError, lambda: call(a, sa, b.transpose(1, 2), sb, offs)),
        (RuntimeError, lambda: call(a.float(), sa, b, sb, offs)),
        (RuntimeError, lambda: call(a, sa, w, sw, offs, epilogue='swiglu', h_out=u8(8, 64))),
        (RuntimeError, lambda: call(a, sa, w, sw, offs, epilogue='swiglu', h_scales=f(8, 2))),
        (RuntimeError, lambda: quantize_fp8_weight(f(8))),
        (RuntimeError, lambda: quantize_fp8_weight(f(8, 8).double())),
        (RuntimeError, lambda: quantize_fp8_weight(f(8, 16).t())),
    ]
    for i, (err, bad) in enumerate(cases):
        with pytest.raises(err):
            bad()
            print('case', i, 'was not refused')


def test_block_refusals():
    from deepep_trn_b200.ops import available
    if not available():
        pytest.skip('the extension is not built')
    _refusals('cpu')


@pytest.mark.gpu
@needs_cuda
def test_block_refusals_on_cuda():
    _refusals('cuda')


# -------------------------------------------------------------------------------------- quantiser
def test_weight_quantiser_definition():
    g = torch.Generator().manual_seed(0)
    w = torch.randn(2, 200, 300, generator=g) * 0.02
    w[0, :128, 128:256] = 0
    q, sc = quantize_fp8_weight(w)
    assert q.shape == w.shape and sc.shape == (2, 2, 3)
    for e in range(2):
        for i in range(2):
            for j in range(3):
                blk = w[e, 128 * i:128 * i + 128, 128 * j:128 * j + 128]
                amax = max(blk.abs().max().item(), 1e-4)
                assert abs(sc[e, i, j].item() - amax / 448) <= 2.0 ** -23 * amax / 448
    err = (dequantize_fp8_128x128(q, sc) - w).abs()
    s = sc.repeat_interleave(128, 1).repeat_interleave(128, 2)[:, :200, :300]
    assert (err <= w.abs() * (2.0 ** -4 + 2.0 ** -22) + s * 2.0 ** -10).all()


@pytest.mark.gpu
@needs_cuda
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('shape', [(1, 1), (128, 128), (3, 130, 264), (2, 257, 129), (5, 64, 7), (1024, 2048)])
def test_weight_quantiser_matches_definition(dtype, shape):
    # the same IEEE operations in the same order: equal bits
    g = torch.Generator().manual_seed(len(shape))
    w = (torch.randn(*shape, generator=g) * 0.05).to(dtype)
    w.view(-1)[:: 97] = 0
    q, sc = quantize_fp8_weight(w.cuda())
    rq, rs = quantize_fp8_128x128(w)
    assert torch.equal(sc.cpu(), rs) and torch.equal(q.cpu().view(torch.uint8), rq.view(torch.uint8))
    # strided input: rows and groups of a larger tensor
    big = torch.zeros(*shape[:-1], shape[-1] + 24, dtype=dtype, device='cuda')
    big[..., 8:8 + shape[-1]] = w.cuda()
    q2, sc2 = quantize_fp8_weight(big[..., 8:8 + shape[-1]])
    assert torch.equal(sc2, sc) and torch.equal(q2.view(torch.uint8), q.view(torch.uint8))


@pytest.mark.gpu
@needs_cuda
def test_weight_quantiser_special_values():
    w = torch.randn(300, 300, generator=torch.Generator().manual_seed(1))
    w[0, 0] = float('nan')
    w[0, 200] = float('inf')
    w[200, 0:128] = 1e-30
    q, sc = quantize_fp8_weight(w.cuda())
    rq, rs = quantize_fp8_128x128(w)
    assert torch.equal(sc.cpu().isnan(), rs.isnan())
    ok = ~rs.isnan()
    assert torch.equal(sc.cpu()[ok], rs[ok])
    a, b = q.cpu().float(), rq.float()
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a[~a.isnan()], b[~b.isnan()])
    assert quantize_fp8_weight(torch.zeros(0, 4, 4, device='cuda'))[0].shape == (0, 4, 4)
