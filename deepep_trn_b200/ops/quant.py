"""fp8 e4m3 1x128 quantisation (N6). CUDA tensors run the kernel; CPU tensors run
the torch definition in ``utils.codec`` (the CPU path is the oracle, not a fallback)."""
from __future__ import annotations

import torch

from ..utils.codec import FP8_AMAX_FLOOR, dequantize_fp8_1x128, quantize_fp8_1x128
from ._ext import load


# Gradients have no natural size (a mean over a large batch puts them at 1e-8 or below), so that the floor of
# activations would take them for zeros: 2^-116 keeps amax / 448 normal and 448 / amax finite in fp32.
GRAD_AMAX_FLOOR = 2.0 ** -116


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """Contiguous, on a 16-byte boundary (the kernels move 16 bytes at a time)."""
    x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x


def quantize_fp8(x: torch.Tensor, round_scale: bool = False, amax_floor: float = FP8_AMAX_FLOOR):
    """e4m3 with one fp32 scale ``max(amax, amax_floor) / 448`` per 128 channels (``round_scale``: its power-of-two
    ceiling). Blocks far below the floor lose their values; gradients take ``GRAD_AMAX_FLOOR``. CUDA tensors are
    bf16 or fp16."""
    if not x.is_cuda:
        return quantize_fp8_1x128(x, round_scale, amax_floor)
    x = _aligned(x)
    H = x.shape[-1]
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    s = torch.empty(*x.shape[:-1], H // 128, dtype=torch.float32, device=x.device)
    load().quant_fp8(x, q.view(torch.uint8), s, round_scale, amax_floor)
    return q, s


def dequantize_fp8(q: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """bf16 of e4m3 ``q`` [.., H] times its 1x128 fp32 ``scales`` [.., H/128] (one rounding)."""
    if not q.is_cuda:
        return dequantize_fp8_1x128(q, scales).to(torch.bfloat16)
    q = _aligned(q)
    out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    load().dequant_fp8(q.view(torch.uint8), scales.float().contiguous(), out)
    return out
