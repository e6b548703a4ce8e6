"""Grouped expert GEMMs on tcgen05 tensor cores (N7) with fused SwiGLU (N8).

``grouped_gemm``       C[seg_e] = A[seg_e] @ B[e]^T      A [rows, K], B [G, N, K]   (forward)
                       C[seg_e] = A[seg_e] @ B[e]        A [rows, K], B [G, K, N]   (``b_layout='kn'``: dX)
``grouped_gemm_wgrad`` C[e] = A[seg_e]^T @ B[seg_e]      A [tok, M], B [tok, N]     (dW)
                       C[e] = A[:, seg_e] @ B[:, seg_e]^T A [M, tok], B [N, tok]    (``layout='mk'``)
``grouped_gemm_fp8``   C[seg_e] = A[seg_e] @ B[e]^T      e4m3 A, B with 1x128 power-of-two scales
``grouped_gemm_fp8_block``  the same with arbitrary fp32 scales (A 1x128, B 128x128), either layout of B,
                       segments of any length or one slab per group, and SwiGLU + e4m3 output in the epilogue

Transposed operands are read in place by the tensor cores (MN-major shared-memory
descriptors), never materialised.

Segments are given by ``offsets`` [G + 1] int64 on the device, multiples of 128
(``permute`` pads every expert's rows to that). The kernels read the offsets on
the device, so the calls are CUDA-graph capturable. A device error word records
a timed-out wait inside a kernel; ``check()`` raises on it.
"""
from __future__ import annotations

import torch

from ..utils.codec import FP8_BLOCK, dequantize_fp8_128x128, quantize_fp8_1x128, quantize_fp8_128x128
from ._ext import available, load

_errors: dict = {}
EPILOGUES = {'bf16': 0, 'f32': 1, 'swiglu': 2}


def _err(dev) -> torch.Tensor:
    index = torch.cuda.current_device() if dev.type == 'cuda' and dev.index is None else dev.index
    key = (dev.type, index)
    if key not in _errors:
        _errors[key] = load().error_word(index) if dev.type == 'cuda' else torch.zeros(1, dtype=torch.int32)
    return _errors[key]


def check(device=None) -> None:
    e = _err(torch.device('cuda' if device is None else device))
    if int(e.item()):
        e.zero_()
        raise RuntimeError("a grouped GEMM or permute kernel gave up on a timed-out wait on the device")


def grouped_gemm(A: torch.Tensor, B: torch.Tensor, offsets: torch.Tensor, out: torch.Tensor | None = None,
                 epilogue: str = 'bf16', h_out: torch.Tensor | None = None, save_preact: bool = True,
                 num_sms: int = 0, timeout_s: float = 10.0, b_layout: str = 'nk',
                 residual: torch.Tensor | None = None):
    """Returns C (or ``(h, pre_activation)`` for ``epilogue='swiglu'``). ``b_layout='kn'``
    takes B as [G, K, N] (e.g. a forward weight, for the input gradient). ``residual``
    (bf16 [rows, N], bf16 epilogue only) is added to the fp32 accumulator before rounding."""
    kn = b_layout == 'kn'
    rows, N = A.shape[0], B.shape[2 if kn else 1]
    if epilogue == 'swiglu':
        h = h_out if h_out is not None else torch.empty(rows, N // 2, dtype=torch.bfloat16, device=A.device)
        c = (out if out is not None else torch.empty(rows, N, dtype=torch.bfloat16, device=A.device)) \
            if save_preact else None
        load().grouped_gemm_m(A, B, offsets, c, h, 2, _err(A.device), num_sms, timeout_s, kn, None)
        return h, c
    dtype = torch.float32 if epilogue == 'f32' else torch.bfloat16
    c = out if out is not None else torch.empty(rows, N, dtype=dtype, device=A.device)
    load().grouped_gemm_m(A, B, offsets, c, None, EPILOGUES[epilogue], _err(A.device), num_sms, timeout_s, kn,
                          residual)
    return c


def grouped_gemm_wgrad(A: torch.Tensor, B: torch.Tensor, offsets: torch.Tensor, out_dtype=torch.float32,
                       out: torch.Tensor | None = None, num_sms: int = 0, timeout_s: float = 10.0,
                       layout: str = 'tok'):
    """Per-expert A_e^T B_e over each token segment: ``[G, M, N]``. ``layout='tok'`` takes the
    activations as they are (A [tok, M], B [tok, N]); ``'mk'`` takes them transposed."""
    G = offsets.numel() - 1
    tok = layout == 'tok'
    M, N = (A.shape[1], B.shape[1]) if tok else (A.shape[0], B.shape[0])
    c = out if out is not None else torch.empty(G, M, N, dtype=out_dtype, device=A.device)
    load().grouped_gemm_k(A, B, offsets, c, _err(A.device), num_sms, timeout_s, tok)
    return c


def quantize_fp8_blocks(w: torch.Tensor):
    """e4m3 copy of ``w`` [.., K] with one power-of-two fp32 scale per (row, 128-channel block):
    the operand format of ``grouped_gemm_fp8`` (the tensor cores apply the scales as UE8M0
    exponents, so they must be powers of two)."""
    q, sc = quantize_fp8_1x128(w, round_scale=True)
    return q.contiguous(), sc.contiguous()


def fp8_scale_tiles(scales: torch.Tensor, groups: int = 1) -> torch.Tensor:
    """Power-of-two fp32 scales [groups * rows, K/128] -> the 512-byte tiles ``grouped_gemm_fp8``
    streams into tensor memory (one per 128 rows and 128-channel block). Build them once for
    weights and pass the tiles instead of the fp32 scales to skip the per-call conversion."""
    sc = scales.reshape(-1, scales.shape[-1]).float().contiguous()
    return load().sf_tiles(sc, groups, sc.shape[0] // groups)


def grouped_gemm_fp8(A, sa, B, sb, offsets, out=None, epilogue: str = 'bf16', h_out=None, save_preact: bool = True,
                     num_sms: int = 0, timeout_s: float = 10.0):
    """Block-scaled fp8 grouped GEMM on the tensor cores (``tcgen05.mma ... kind::mxf8f6f4.block_scale``):
    ``C[seg_e] = (A * sa)[seg_e] @ (B[e] * sb[e])^T`` with A [rows, K] and B [G, N, K] e4m3, and
    power-of-two fp32 scales sa [rows, K/128], sb [G, N, K/128] (``quantize_fp8_blocks``), or
    their ``fp8_scale_tiles``.
    fp32 accumulation; epilogues as ``grouped_gemm``. The SwiGLU epilogue reads each 128-wide
    output tile as [64 gate | 64 up] (``interleave_gate_up(..., block=64)``)."""
    rows, N = A.shape[0], B.shape[1]
    a8, b8 = A.view(torch.uint8), B.view(torch.uint8)
    if sa.dtype != torch.uint8:
        sa = sa.float()
    if sb.dtype != torch.uint8:
        sb = sb.float().contiguous()
    if epilogue == 'swiglu':
        h = h_out if h_out is not None else torch.empty(rows, N // 2, dtype=torch.bfloat16, device=A.device)
        c = (out if out is not None else torch.empty(rows, N, dtype=torch.bfloat16, device=A.device)) \
            if save_preact else None
        load().grouped_gemm_fp8_m(a8, sa, b8, sb, offsets, c, h, 2, _err(A.device), num_sms, timeout_s)
        return h, c
    dtype = torch.float32 if epilogue == 'f32' else torch.bfloat16
    c = out if out is not None else torch.empty(rows, N, dtype=dtype, device=A.device)
    load().grouped_gemm_fp8_m(a8, sa, b8, sb, offsets, c, None, EPILOGUES[epilogue], _err(A.device), num_sms,
                              timeout_s)
    return c


FP8_BLOCK_EPILOGUES = {'bf16': 0, 'f32': 1, 'swiglu': 2}


def quantize_fp8_weight(w: torch.Tensor, out=None):
    """e4m3 copy of ``w`` [N, K] or [G, N, K] (fp32, bf16 or fp16) with one fp32 scale per
    128 x 128 block (the last blocks of a side may be short): ``(q, scales [.., ceil(N/128),
    ceil(K/128)])`` with ``w ~= q * scale``, ``scale = max(amax, 1e-4) / 448``. The operand format
    of ``grouped_gemm_fp8_block``; a transposed product reads the same pair (``b_layout='kn'``).
    ``out``: a contiguous pair ``(q, scales)`` to write, which is returned."""
    q, sc = out if out is not None else (None, None)
    if w.is_cuda:
        res = load().quant_fp8_weight(w, q, sc)
        return out if out is not None else res
    if available():
        load().quant_fp8_weight(w, q, sc)   # the argument checks
    res = quantize_fp8_128x128(w)
    if out is None:
        return res
    q.view(torch.uint8).copy_(res[0].view(torch.uint8))
    sc.copy_(res[1])
    return out


def grouped_gemm_fp8_block(A, sa, B, sb, offsets=None, counts=None, out=None, epilogue: str = 'bf16',
                           b_layout: str = 'nk', h_out=None, h_scales=None, save_preact: bool = False,
                           num_sms: int = 0, timeout_s: float = 10.0):
    """Grouped fp8 GEMM with arbitrary fp32 scales, one per 128 channels:
    ``C[rows of g] = (A * sa)[rows of g] @ (B[g] * sb[g])^T``.

    A and B are e4m3. ``sa`` has one fp32 scale per row of A and 128 channels (``quantize_fp8``, or
    what an fp8 dispatch delivers), ``sb`` [G, ceil(N/128), ceil(K/128)] one per 128 x 128 block of
    B [G, N, K] (``quantize_fp8_weight``). ``b_layout='kn'`` takes B as [G, K, N] with sb
    [G, ceil(K/128), ceil(N/128)], read in place: with a forward weight and its scales that is the
    gradient of the product's input. K is a multiple of 16, N of 8 (``'kn'``: 16).

    Rows: A [rows, K] with ``offsets`` [G + 1] int64 (nondecreasing; any lengths, also zero), or
    A [G, cap, K], one slab per group (a low-latency dispatch's layout, strided slabs included).
    ``counts`` [G] int32, with either, gives the rows in use from the start of each group. Rows
    that belong to no group, or lie behind a count, are not written: a new output holds anything there.

    Sums are fp32 (each block of 128 products is scaled and added in fp32). ``epilogue='bf16'`` and
    ``'f32'`` return C. ``'swiglu'`` reads each 256 columns as [128 gate | 128 up]
    (``interleave_gate_up``) and returns ``(h, h_scales, pre)``: ``h = silu(gate) * up`` in e4m3 with
    fp32 1x128 scales, the operand of the next product, and the bf16 pre-activation with
    ``save_preact`` (else None). ``out``, ``h_out``, ``h_scales`` receive C / pre, h and its scales.

    ``num_sms`` > 0 bounds the SMs that the call's kernels hold at a time (they then run one after the other).
    ``timeout_s`` bounds each wait inside the kernels. One that runs out ends the call, whose output is then
    not to be used, and ``check()`` raises (0: the call gives up without multiplying anything).
    """
    if epilogue not in FP8_BLOCK_EPILOGUES:
        raise ValueError(f'unknown epilogue {epilogue!r}; expected one of {tuple(FP8_BLOCK_EPILOGUES)}')
    if b_layout not in ('nk', 'kn'):
        raise ValueError(f"unknown b_layout {b_layout!r}; expected 'nk' or 'kn'")
    kn = b_layout == 'kn'
    N = B.shape[2 if kn else 1]
    lead = A.shape[:-1]
    h = hs = None
    if epilogue == 'swiglu':
        h = h_out if h_out is not None else torch.empty(*lead, N // 2, dtype=torch.float8_e4m3fn, device=A.device)
        hs = h_scales if h_scales is not None else torch.empty(*lead, N // 256, dtype=torch.float32, device=A.device)
        c = (out if out is not None else torch.empty(*lead, N, dtype=torch.bfloat16, device=A.device)) \
            if save_preact else None
    else:
        dtype = torch.float32 if epilogue == 'f32' else torch.bfloat16
        c = out if out is not None else torch.empty(*lead, N, dtype=dtype, device=A.device)
    if A.is_cuda or available():   # on CPU tensors: the argument checks
        load().grouped_gemm_fp8_block(A, sa, B, sb, offsets, counts, c, h, hs, FP8_BLOCK_EPILOGUES[epilogue],
                                      _err(A.device), num_sms, timeout_s, kn)
    if not A.is_cuda:
        _grouped_gemm_fp8_block_cpu(A, sa, B, sb, offsets, counts, c, h, hs, kn)
    return c if epilogue != 'swiglu' else (h, hs, c)


def fp8_block_plan(G: int, rows: int, N: int, K: int, masked: bool, num_sms: int = 0, counts=None, device=None):
    """What a ``grouped_gemm_fp8_block`` call of these sizes launches, as a dict: ``form`` ('few' or 'many' rows a
    group, or 'both', where the device decides by the counts; with ``counts`` 'both: few', 'both: many' or
    'both: mixed'), ``split`` (CTAs that divide K in the form for few rows), ``few_ctas``, ``many_ctas`` and
    ``overlap`` (whether the kernels run side by side). ``rows`` are those of a slab (``masked``) or of all
    segments. ``device`` gives the SMs and the resident clusters of 2, 4 and 8 CTAs of a device other than the
    current one. The kernels together hold no more SMs than ``num_sms`` grants."""
    plan = load().fp8_block_plan(G, rows, N, K, masked, num_sms, counts, device)
    return dict(zip(('form', 'split', 'few_ctas', 'many_ctas', 'overlap'), plan))


def _grouped_gemm_fp8_block_cpu(A, sa, B, sb, offsets, counts, c, h, hs, kn):
    """The torch definition (fp32), into c and / or h and hs."""
    Bf = dequantize_fp8_128x128(B.view(torch.float8_e4m3fn), sb)
    Bf = Bf if kn else Bf.transpose(1, 2)
    Af = A.view(torch.float8_e4m3fn).float() * sa.repeat_interleave(FP8_BLOCK, -1)[..., :A.shape[-1]]
    for g in range(B.shape[0]):
        rows = A.shape[-2]
        begin, end = (0, rows) if A.dim() == 3 else (min(max(int(offsets[g]), 0), rows), min(int(offsets[g + 1]), rows))
        if counts is not None:
            end = min(end, begin + max(int(counts[g]), 0))
        end = max(end, begin)
        at = (g, slice(begin, end)) if A.dim() == 3 else (slice(begin, end),)
        y = Af[at] @ Bf[g]
        if c is not None:
            c[at] = y.to(c.dtype)
        if h is not None:
            gate, up = deinterleave(y)
            q, sc = quantize_fp8_1x128(torch.nn.functional.silu(gate) * up)
            h.view(torch.uint8)[at] = q.view(torch.uint8)
            hs[at] = sc


def interleave_gate_up(w_gate: torch.Tensor, w_up: torch.Tensor, block: int = 128) -> torch.Tensor:
    """[G, I, K] gate and up weights -> [G, 2I, K] with 128-row blocks alternating gate / up,
    the layout the SwiGLU epilogue expects (each 256-wide output tile = 128 gate + 128 up)."""
    G, I, K = w_gate.shape
    assert I % block == 0
    g = w_gate.reshape(G, I // block, block, K)
    u = w_up.reshape(G, I // block, block, K)
    return torch.stack([g, u], 2).reshape(G, 2 * I, K)


def deinterleave(x: torch.Tensor, block: int = 128):
    """Inverse of the interleaving along the last dim: [.., 2I] -> (gate [.., I], up [.., I])."""
    *lead, n2 = x.shape
    v = x.reshape(*lead, n2 // (2 * block), 2, block)
    return v[..., 0, :].reshape(*lead, n2 // 2), v[..., 1, :].reshape(*lead, n2 // 2)
