"""Expert-parallel MoE layer: router top-k -> dispatch -> grouped SwiGLU experts -> combine.

Forward (per rank, EP group of the Buffer):
    logits = x @ Wr^T ; (idx, w) = router_topk(logits)               # N9
    recv = dispatch(x)  (normal mode, NVLink kernels)                 # N1 + N2
    rows = permute(recv) into 128-row padded expert segments          # N10
    h, pre = grouped_gemm(rows, W1, swiglu epilogue)                  # N7 + N8 (tcgen05)
    o = grouped_gemm(h, W2)                                           # N7
    y = combine(o, pairs=(pos, weights))  (weighted un-permute fused)  # N10 + N3
Backward reuses the dispatch handle: the gradient of combine is a cached dispatch
and the gradient of dispatch is a combine (whose weight channel carries the
routing-weight gradients home). Expert weight gradients come from the variable-K
grouped GEMM over the permuted activations.

Weights: W1 [EL, 2I, H] with gate and up rows interleaved in 128-row blocks
(``ops.gemm.interleave_gate_up``), W2 [EL, H, I], router Wr [E, H]; all bf16.
Router logits come out of the same tensor-core GEMM with an fp32 epilogue, so
expert selection matches an fp32 router up to summation order.

``gate`` replaces the softmax over the chosen k by ``ops.moe_ops.router_gate`` (sigmoid or softmax
scores, expert groups, renormalisation, scale; ``router_bias`` then steers the selection only).
``fp8_block`` runs dispatch and the experts' products in e4m3 with fp32 scales, 1x128 for rows and
128x128 for weights, in training and inference: SwiGLU's result leaves the first product quantised, the
input gradients read the same weights the other way round, the weight gradients stay bf16.
``forward_low_latency`` is its generation step over the low-latency dispatch and combine.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from ..ops import gemm as G
from ..ops import moe_ops as MO
from ..ops.quant import GRAD_AMAX_FLOOR, dequantize_fp8, quantize_fp8
from ..utils.profiling import timer


_OFFS: dict = {}


def _quantize_grad(d):
    return quantize_fp8(d, amax_floor=GRAD_AMAX_FLOOR)


def _single_segment(T: int, device) -> torch.Tensor:
    """Offsets [0, T rounded up to 128] for one-group GEMMs (cached per size and device)."""
    key = (T, str(device))
    if key not in _OFFS:
        _OFFS[key] = torch.tensor([0, (T + 127) // 128 * 128], dtype=torch.int64, device=device)
    return _OFFS[key]


def router_logits(x, Wr):
    """fp32 logits [T, E] = x @ Wr^T on the tensor cores (bf16 inputs, fp32 accumulate and output)."""
    return G.grouped_gemm(x.contiguous(), Wr.unsqueeze(0).contiguous(), _single_segment(x.shape[0], x.device),
                          epilogue='f32')


def _expert_forward(rows, offsets, W1, W2):
    h, pre = G.grouped_gemm(rows, W1, offsets, epilogue='swiglu')
    o = G.grouped_gemm(h, W2, offsets)
    return h, pre, o


def _route(logits, topk, router_bias, gate):
    """(ids, weights): the chosen-k softmax of the biased logits, or ``router_gate``."""
    if gate is None:
        return MO.router_topk(logits if router_bias is None else logits + router_bias, topk)
    return MO.router_gate(logits, topk, bias=router_bias, **gate)


def _route_bwd(logits, idx, w, dw, num_experts, gate):
    if gate is None:
        return MO.router_topk_bwd(idx, w, dw.float(), num_experts)
    kw = {k: gate[k] for k in ('scoring', 'renormalize', 'scale') if k in gate}
    return MO.router_gate_bwd(logits, idx, dw, **kw)


def _router_grads(ctx, x, Wr, logits, idx, w, dw, dx):
    """(dx + dlogits @ Wr, dWr): summed in fp32 in the GEMM's epilogue, one rounding."""
    dlogits = _route_bwd(logits, idx, w, dw, ctx.num_experts, ctx.gate).to(x.dtype)
    seg = _single_segment(x.shape[0], x.device)
    dx = G.grouped_gemm(dlogits, Wr.unsqueeze(0), seg, b_layout='kn', residual=dx.contiguous())
    if ctx.num_experts % 64 == 0:
        dWr = G.grouped_gemm_wgrad(dlogits, x, seg, out_dtype=Wr.dtype)[0]            # [E, H]
    else:  # the token-major operand path tiles M in 64-wide atoms
        if x.shape[0] % 8:   # transposed, the tokens are rows of whole 16-byte words
            pad = (0, 0, 0, -x.shape[0] % 8)
            dlogits, x = nn.functional.pad(dlogits, pad), nn.functional.pad(x, pad)
        dWr = G.grouped_gemm_wgrad(MO.transpose(dlogits), MO.transpose(x), seg, out_dtype=Wr.dtype, layout='mk')[0]
    return dx, dWr


class _MoEFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, Wr, W1, W2, buf, num_experts, topk, router_bias=None, fp8_dispatch=False, gate=None):
        EL = num_experts // buf.group_size
        with timer.stage('moe.router'):
            logits = router_logits(x, Wr)
            idx, w = _route(logits, topk, router_bias, gate)
        with timer.stage('moe.dispatch'):
            ntr, _, nte, itr, _ = buf.get_dispatch_layout(idx, num_experts)
            # fp8_dispatch: tokens travel as e4m3 with 1x128 scales (quantised inside the
            # dispatch kernel) and are dequantised to bf16 by the permute
            recv_x, recv_idx, recv_w, per_expert, handle, _ = buf.dispatch(
                x, topk_idx=idx, topk_weights=w, num_tokens_per_rank=ntr, is_token_in_rank=itr,
                num_tokens_per_expert=nte, use_fp8=fp8_dispatch)
        with timer.stage('moe.permute'):
            rows, pos, offsets, counts = MO.permute(recv_x, recv_idx, EL, per_expert)
        with timer.stage('moe.experts'):
            h, pre, o = _expert_forward(rows, offsets, W1, W2)
        with timer.stage('moe.combine'):
            # the weighted un-permute (sum_k w * o[pos]) is formed inside the combine kernel
            y, _, _ = buf.combine(o, handle, pair_pos=pos, pair_weights=recv_w)
        ctx.save_for_backward(x, Wr, W1, W2, logits if gate is not None else None, idx, w, recv_w, pos, offsets, counts,
                              rows, pre, h, o)
        ctx.buf, ctx.handle, ctx.num_experts, ctx.gate = buf, handle, num_experts, gate
        return y

    @staticmethod
    def backward(ctx, dy):
        x, Wr, W1, W2, logits, idx, w, recv_w, pos, offsets, counts, rows, pre, h, o = ctx.saved_tensors
        buf, handle = ctx.buf, ctx.handle
        dy = dy.contiguous().to(x.dtype)
        with timer.stage('moe.bwd.dispatch'):
            dy_recv, *_ = buf.dispatch(dy, handle=handle)                 # combine backward
        with timer.stage('moe.bwd.unpermute'):
            d_o, d_recv_w = MO.unpermute_bwd(dy_recv, o, pos, recv_w, offsets, counts)
        # transposed operands are read in place by the GEMM (MN-major tiles); fp32 accumulation,
        # one rounding to the weight dtype
        with timer.stage('moe.bwd.dgrad'):
            dh = G.grouped_gemm(d_o, W2, offsets, b_layout='kn')           # [P, I] = d_o @ W2[e]
            dpre = MO.swiglu_bwd(dh, pre)                                  # [P, 2I]
            drows = G.grouped_gemm(dpre, W1, offsets, b_layout='kn')       # [P, H] = dpre @ W1[e]
        with timer.stage('moe.bwd.wgrad'):
            dW2 = G.grouped_gemm_wgrad(d_o, h, offsets, out_dtype=W2.dtype)      # [EL, H, I]
            dW1 = G.grouped_gemm_wgrad(dpre, rows, offsets, out_dtype=W1.dtype)  # [EL, 2I, H]
        with timer.stage('moe.bwd.permute'):
            d_recv_x = MO.permute_bwd(drows, pos)
        with timer.stage('moe.bwd.combine'):
            dx, dw, _ = buf.combine(d_recv_x, handle, topk_weights=d_recv_w)   # dispatch backward
        with timer.stage('moe.bwd.router'):
            dx, dWr = _router_grads(ctx, x, Wr, logits, idx, w, dw, dx)
        return dx, dWr, dW1, dW2, None, None, None, None, None, None


class _MoEBlockFunction(torch.autograd.Function):
    """The layer with e4m3 rows and weights and fp32 block scales. ``wq``: the quantised weights
    (q1, s1, q2, s2) of W1 and W2; the gradients go to W1 and W2 themselves."""

    @staticmethod
    def forward(ctx, x, Wr, W1, W2, wq, buf, num_experts, topk, router_bias, gate, train):
        EL = num_experts // buf.group_size
        q1, s1, q2, s2 = wq
        with timer.stage('moe.router'):
            logits = router_logits(x, Wr)
            idx, w = _route(logits, topk, router_bias, gate)
        with timer.stage('moe.dispatch'):
            ntr, _, nte, itr, _ = buf.get_dispatch_layout(idx, num_experts)
            recv_x, recv_idx, recv_w, per_expert, handle, _ = buf.dispatch(
                x, topk_idx=idx, topk_weights=w, num_tokens_per_rank=ntr, is_token_in_rank=itr,
                num_tokens_per_expert=nte, use_fp8=True)
        with timer.stage('moe.permute'):
            (rq, rs), pos, offsets, counts = MO.permute(recv_x, recv_idx, EL, per_expert, keep_fp8=True)
        with timer.stage('moe.experts'):
            h, hs, pre = G.grouped_gemm_fp8_block(rq, rs, q1, s1, offsets, epilogue='swiglu', save_preact=train)
            o = G.grouped_gemm_fp8_block(h, hs, q2, s2, offsets)
        with timer.stage('moe.combine'):
            y, _, _ = buf.combine(o, handle, pair_pos=pos, pair_weights=recv_w)
        if train:
            ctx.save_for_backward(x, Wr, q1, s1, q2, s2, logits if gate is not None else None, idx, w, recv_w, pos,
                                  offsets, counts, rq, rs, pre, h, hs, o)
            ctx.buf, ctx.handle, ctx.num_experts, ctx.gate = buf, handle, num_experts, gate
            ctx.w_dtypes = W1.dtype, W2.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        (x, Wr, q1, s1, q2, s2, logits, idx, w, recv_w, pos, offsets, counts, rq, rs, pre, h, hs, o) = ctx.saved_tensors
        buf, handle = ctx.buf, ctx.handle
        dy = dy.contiguous().to(x.dtype)
        with timer.stage('moe.bwd.dispatch'):
            dy_recv, *_ = buf.dispatch(dy, handle=handle)                  # combine backward
        with timer.stage('moe.bwd.unpermute'):
            d_o, d_recv_w = MO.unpermute_bwd(dy_recv, o, pos, recv_w, offsets, counts)
        with timer.stage('moe.bwd.dgrad'):
            dh = G.grouped_gemm_fp8_block(*_quantize_grad(d_o), q2, s2, offsets, b_layout='kn')        # d_o @ W2[e]
            dpre = MO.swiglu_bwd(dh, pre)
            drows = G.grouped_gemm_fp8_block(*_quantize_grad(dpre), q1, s1, offsets, b_layout='kn')    # dpre @ W1[e]
        with timer.stage('moe.bwd.wgrad'):
            dW2 = G.grouped_gemm_wgrad(d_o, dequantize_fp8(h, hs), offsets, out_dtype=ctx.w_dtypes[1])
            dW1 = G.grouped_gemm_wgrad(dpre, dequantize_fp8(rq, rs), offsets, out_dtype=ctx.w_dtypes[0])
        with timer.stage('moe.bwd.permute'):
            d_recv_x = MO.permute_bwd(drows, pos)
        with timer.stage('moe.bwd.combine'):
            dx, dw, _ = buf.combine(d_recv_x, handle, topk_weights=d_recv_w)   # dispatch backward
        with timer.stage('moe.bwd.router'):
            dx, dWr = _router_grads(ctx, x, Wr, logits, idx, w, dw, dx)
        return dx, dWr, dW1, dW2, None, None, None, None, None, None, None


class MoELayer(nn.Module):
    """SwiGLU mixture-of-experts layer with expert parallelism over ``buffer``'s EP group."""

    def __init__(self, buffer, hidden: int, intermediate: int, num_experts: int, topk: int,
                 dtype=torch.bfloat16, device=None, init_std: float = 0.02, seed: int = 0,
                 fp8_dispatch: bool = False, fp8_experts: bool = False, gate: dict | None = None,
                 fp8_block: bool = False):
        super().__init__()
        R = buffer.group_size
        if num_experts % R:
            raise ValueError(f'num_experts={num_experts} must be divisible by the EP size {R}')
        if intermediate % 128 or hidden % 128:
            raise ValueError('hidden and intermediate must be multiples of 128')
        self.buffer = buffer
        self.fp8_dispatch = fp8_dispatch   # forward tokens cross NVLink as fp8 e4m3 + 1x128 scales
        # inference (no autograd): fp8 dispatch and block-scaled fp8 expert GEMMs on e4m3 weights
        self.fp8_experts = fp8_experts
        if fp8_experts and (fp8_block or gate is not None):
            raise ValueError('fp8_experts (power-of-two scales) takes neither fp8_block nor gate')
        # keyword arguments of router_gate (scoring, num_groups, topk_groups, group_score, renormalize, scale)
        self.gate = dict(gate) if gate is not None else None
        # e4m3 dispatch and experts with fp32 block scales, in training too
        self.fp8_block = fp8_block
        self._fp8_cache = None    # fp8_experts
        self._block_copy = self._block_key = None   # fp8_block: what quantize_weights made, and of which weights
        self.hidden, self.intermediate = hidden, intermediate
        self.num_experts, self.topk = num_experts, topk
        EL = num_experts // R
        # seeded on the target device (the router is shared by all ranks, the experts are per rank)
        gdev = torch.device(device) if device is not None else torch.device('cpu')
        g = torch.Generator(device=gdev).manual_seed(seed)
        g_local = torch.Generator(device=gdev).manual_seed(seed * 1000 + buffer.rank + 1)
        std = init_std

        def randn(*shape, gen):
            return (torch.randn(*shape, generator=gen, device=gdev) * std).to(dtype)
        self.router = nn.Parameter(randn(num_experts, hidden, gen=g))
        wg = randn(EL, intermediate, hidden, gen=g_local)
        wu = randn(EL, intermediate, hidden, gen=g_local)
        self.w1 = nn.Parameter(G.interleave_gate_up(wg, wu))
        del wg, wu
        self.w2 = nn.Parameter(randn(EL, hidden, intermediate, gen=g_local))
        # fp32 bias added to the router logits before top-k, or with `gate` to its scores for the
        # selection only (not trained here; it steers load, e.g. a Zipf skew for benchmarks or a
        # balancing bias)
        self.register_buffer('router_bias', torch.zeros(num_experts, dtype=torch.float32, device=device))

    def _fp8_weights(self):
        """e4m3 copies of the expert weights with power-of-two 1x128 scales (as scale tiles), rebuilt when
        the weights' version or address changes and after a call with gradients. W1 is re-interleaved in 64-row gate / up blocks, the
        layout of the fp8 GEMM's 128-wide SwiGLU tiles."""
        key = (self.w1._version, self.w2._version, self.w1.data_ptr(), self.w2.data_ptr())
        if self._fp8_cache is None or self._fp8_cache[0] != key:
            with torch.no_grad():
                EL, I2, H = self.w1.shape
                v = self.w1.reshape(EL, I2 // 256, 2, 128, H)
                gate, up = v[:, :, 0].reshape(EL, I2 // 2, H), v[:, :, 1].reshape(EL, I2 // 2, H)
                w1 = G.interleave_gate_up(gate, up, block=64)
                q1, s1 = G.quantize_fp8_blocks(w1)
                q2, s2 = G.quantize_fp8_blocks(self.w2)
                self._fp8_cache = (key, q1, G.fp8_scale_tiles(s1, EL), q2, G.fp8_scale_tiles(s2, EL))
        return self._fp8_cache[1:]

    def _weights_key(self):
        """What a write to the weights usually changes (not one through ``w.data``)."""
        return tuple((w.device, w.data_ptr(), 0 if w.is_inference() else w._version) for w in (self.w1, self.w2))

    @torch.no_grad()
    def quantize_weights(self) -> None:
        """Quantises the expert weights of an ``fp8_block`` layer into a copy that ``forward_low_latency`` and
        calls without gradients then read instead of quantising the weights themselves (0.67 ms for 32
        experts, W1 4096 x 7168 and W2 7168 x 2048).

        Call it again after a change of the weights: it writes into the same storage, so the replays of a
        captured step see the new weights from then on. Calls on other streams are ordered behind it as behind
        any write to the weights. The copy is left aside once the weights' version or address differs, and
        after a call with gradients, which an update follows. What leaves no trace in Python (a write through
        ``w.data`` outside of training, a replayed optimizer step) goes unseen.

        An ``fp8_experts`` layer, which keeps a copy by itself, makes that one anew."""
        if not (self.fp8_block or self.fp8_experts):
            raise ValueError('quantize_weights needs fp8_block=True or fp8_experts=True')
        if self.w1.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError('quantize_weights must be called outside of a capture')
        if self.fp8_experts:
            self._fp8_cache = None
            self._fp8_weights()
            return
        kept = self._block_copy
        if kept is not None and not all(q.shape == w.shape and q.device == w.device
                                        for q, w in ((kept[0], self.w1), (kept[2], self.w2))):
            kept = None
        self._block_key = None
        with torch.inference_mode(False), torch.no_grad():   # (the copy is to be written outside of inference mode too)
            self._block_copy = (*G.quantize_fp8_weight(self.w1, out=kept and kept[:2]),
                                *G.quantize_fp8_weight(self.w2, out=kept and kept[2:]))
        self._block_key = self._weights_key()

    def _block_weights(self, train: bool):
        """(q1, s1, q2, s2): e4m3 expert weights with 128x128 fp32 scales, quantised in this call, or without
        gradients the copy of ``quantize_weights``. (An optimizer that writes through ``w.data`` changes neither
        version nor address: in training no kept copy could be told from an old one.)"""
        if not train and self._block_key is not None and self._block_key == self._weights_key():
            return self._block_copy
        with torch.no_grad():
            return (*G.quantize_fp8_weight(self.w1), *G.quantize_fp8_weight(self.w2))

    @torch.no_grad()
    def forward_low_latency(self, x: torch.Tensor, num_max_tokens_per_rank: int) -> torch.Tensor:
        """A generation step (``fp8_block`` layers): low-latency dispatch -> expert slabs -> combine. ``x`` holds
        at most ``num_max_tokens_per_rank`` tokens, which all ranks give alike. Nothing waits on the host, so
        the step can be captured into a CUDA graph after one call. Captured after ``quantize_weights`` it reads
        that copy, which the next ``quantize_weights`` renews in place; captured without, every replay quantises
        the weights as they are then."""
        if not self.fp8_block:
            raise ValueError('forward_low_latency needs fp8_block=True')
        q1, s1, q2, s2 = self._block_weights(train=False)
        with timer.stage('moe.router'):
            idx, w = _route(router_logits(x, self.router), self.topk, self.router_bias, self.gate)
        (rq, rs), counts, handle, _, _ = self.buffer.low_latency_dispatch(x, idx, num_max_tokens_per_rank,
                                                                          self.num_experts, use_fp8=True)
        with timer.stage('moe.experts'):
            h, hs, _ = G.grouped_gemm_fp8_block(rq, rs, q1, s1, counts=counts, epilogue='swiglu')
            o = G.grouped_gemm_fp8_block(h, hs, q2, s2, counts=counts)
        y, _, _ = self.buffer.low_latency_combine(o, idx, w, handle)
        return y

    def _forward_fp8(self, x: torch.Tensor) -> torch.Tensor:
        buf, E = self.buffer, self.num_experts
        EL = E // buf.group_size
        with timer.stage('moe.router'):
            logits = router_logits(x, self.router) + self.router_bias
            idx, w = MO.router_topk(logits, self.topk)
        with timer.stage('moe.dispatch'):
            ntr, _, nte, itr, _ = buf.get_dispatch_layout(idx, E)
            recv_x, recv_idx, recv_w, per_expert, handle, _ = buf.dispatch(
                x, topk_idx=idx, topk_weights=w, num_tokens_per_rank=ntr, is_token_in_rank=itr,
                num_tokens_per_expert=nte, use_fp8=True, round_scale=True)
        with timer.stage('moe.permute'):
            (rq, rs), pos, offsets, _ = MO.permute(recv_x, recv_idx, EL, per_expert, keep_fp8=True)
        q1, t1, q2, t2 = self._fp8_weights()
        with timer.stage('moe.experts'):
            h, _ = G.grouped_gemm_fp8(rq, rs, q1, t1, offsets, epilogue='swiglu', save_preact=False)
            hq, hs = quantize_fp8(h, round_scale=True)
            o = G.grouped_gemm_fp8(hq, hs, q2, t2, offsets)
        with timer.stage('moe.combine'):
            # the weighted un-permute (sum_k w * o[pos]) is formed inside the combine kernel
            y, _, _ = buf.combine(o, handle, pair_pos=pos, pair_weights=recv_w)
        return y

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        train = torch.is_grad_enabled()
        if train and (self.w1.requires_grad or self.w2.requires_grad):
            # the weights are about to change, perhaps without a trace (see _block_weights)
            self._fp8_cache = self._block_key = None
        if self.fp8_experts and not train:
            return self._forward_fp8(x)
        if self.fp8_block:
            return _MoEBlockFunction.apply(x, self.router, self.w1, self.w2, self._block_weights(train), self.buffer,
                                           self.num_experts, self.topk, self.router_bias, self.gate, train)
        return _MoEFunction.apply(x, self.router, self.w1, self.w2, self.buffer, self.num_experts, self.topk,
                                  self.router_bias, self.fp8_dispatch, self.gate)


def reference_moe(x, Wr, W1, W2, topk, router_bias=None):
    """fp32 torch definition of the layer on one rank holding all experts (W1 interleaved)."""
    logits = x.float() @ Wr.float().t()
    if router_bias is not None:
        logits = logits + router_bias
    idx, w = MO.router_topk(logits.cpu(), topk)
    idx, w = idx.to(x.device), w.to(x.device)
    out = torch.zeros(x.shape, dtype=torch.float32, device=x.device)
    for e in range(W1.shape[0]):
        hit = (idx == e)
        tok = hit.any(1).nonzero().flatten()
        if tok.numel() == 0:
            continue
        a = x[tok].float()
        gu = a @ W1[e].float().t()
        gate, up = G.deinterleave(gu)
        hh = torch.nn.functional.silu(gate) * up
        oo = hh @ W2[e].float().t()
        we = (w[tok] * hit[tok]).sum(1, keepdim=True)
        out[tok] += we * oo
    return out


def smoke_step(buf, dev):
    """One tiny forward + backward of the layer (used by the build/smoke entry point), with the softmax gate in
    bf16, and with the grouped gate and fp8 experts, whose generation step it runs too."""
    torch.manual_seed(0)
    E = 8 * buf.group_size
    x = (torch.randn(64, 256, device=dev) * 0.5).to(torch.bfloat16).requires_grad_()
    for kw in ({}, dict(gate=dict(scoring='sigmoid', num_groups=4, topk_groups=2, scale=2.5), fp8_block=True)):
        layer = MoELayer(buf, hidden=256, intermediate=256, num_experts=E, topk=2, device=dev, **kw)
        x.grad = None
        y = layer(x)
        y.float().square().mean().backward()
        torch.cuda.synchronize()
        assert torch.isfinite(y.float()).all() and torch.isfinite(x.grad.float()).all() and x.grad.abs().amax() > 0
        assert layer.w1.grad is not None and torch.isfinite(layer.w1.grad.float()).all()
    layer.quantize_weights()
    out = layer.forward_low_latency(x.detach(), 64)
    torch.cuda.synchronize()
    assert torch.isfinite(out.float()).all() and out.abs().amax() > 0
