"""Workloads of the expert operators: the gate of an expert-parallel layer, the fp8 products of its
experts with one scale per block of 128, and the quantisation of the weights that they read.

    gate     router_gate (+ router_gate_bwd): scores, selection bias, groups, top-k, weights
    gemm     grouped_gemm_fp8_block: C[rows of g] = (A * sa) @ (B[g] * sb[g])^T, optionally with
             SwiGLU and the e4m3 quantisation of its result in the same pass
    weight   quantize_fp8_weight: e4m3 weights with one fp32 scale per 128 x 128 block

``own = False`` computes the definitions with elementary torch operations, ``own = True`` calls
the library's kernels.
"""
import math

import torch

own = False

BLOCK = 128
FP8_MAX = 448.0
AMAX_FLOOR = 1e-4
DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def _dev():
    return torch.device('cuda' if torch.cuda.is_available() else 'cpu')


# ----------------------------------------------------------------------------- the cases
def _gate(name, T, E, k, scoring, dtype, bias, groups, topk_groups, group_score, renorm, scale, masked, train):
    c = dict(op='gate', T=T, E=E, k=k, scoring=scoring, dtype=dtype, bias=bias, groups=groups, topk_groups=topk_groups,
             group_score=group_score, renorm=renorm, scale=scale, masked=masked, train=train)
    return dict(c, name=name) if name else c


def _gemm(name, layout, G, rows, cap, align, N, K, b, epilogue, pre=False):
    c = dict(op='gemm', layout=layout, G=G, rows=rows, cap=cap, align=align, N=N, K=K, b=b, epilogue=epilogue, pre=pre)
    return dict(c, name=name) if name else c


def _weight(name, G, N, K, dtype):
    c = dict(op='weight', G=G, N=N, K=K, dtype=dtype)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of a generation step through a grouped sigmoid gate: nothing but latency
        _gate('gate 1 token', 1, 256, 8, 'sigmoid', 'f32', True, 8, 4, 'top2', True, 2.5, 0.0, False),
        # a decoding batch through a small softmax gate whose logits come in bf16
        _gate('gate 128 tokens', 128, 64, 6, 'softmax', 'bf16', False, 1, 1, 'max', False, 1.0, 0.0, False),
        # a training step of the usual size: grouped sigmoid gate with its balance bias, and its gradient
        _gate('gate 16k tokens train', 16384, 256, 8, 'sigmoid', 'f32', True, 8, 4, 'top2', True, 2.5, 0.0, True),
        # a long ragged batch; some experts are masked away and some tokens (padding) have none left
        _gate('gate 65k tokens odd train', 65521, 160, 6, 'softmax', 'bf16', False, 8, 3, 'max', False, 16.0, 0.05, True),
        # a generation step, 128 tokens on each of 8 ranks: the first expert product with its activation
        _gemm('decode up', 'masked', 32, 1024, 1024, 1, 4096, 7168, 'nk', 'swiglu'),
        # ... and the second product
        _gemm('decode down', 'masked', 32, 1024, 1024, 1, 7168, 2048, 'nk', 'bf16'),
        # a single token through one expert
        _gemm('one row', 'segments', 1, 1, 0, 1, 7168, 2048, 'nk', 'bf16'),
        # unpadded segments of odd lengths, odd widths and a reduction that ends inside a block
        _gemm('ragged odd', 'segments', 7, 1531, 0, 1, 1416, 1168, 'nk', 'f32'),
        # a training step of 32 experts: first product, activation, and the pre-activation for the backward
        _gemm('train up', 'segments', 32, 32768, 0, 128, 4096, 7168, 'nk', 'swiglu', True),
        # ... and the gradient of its input, which reads the same weights the other way round
        _gemm('train input gradient', 'segments', 32, 32768, 0, 128, 7168, 4096, 'kn', 'bf16'),
        # one expert's second weight, in the master type, with edges inside the blocks
        _weight('weight odd', 1, 2040, 1416, 'f32'),
        # the first weights of 32 experts, once per optimizer step
        _weight('weights of 32 experts', 32, 4096, 7168, 'bf16'),
    ]


def _spread(rng, lo, hi, mult=1):
    """A multiple of `mult` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / mult)) * mult))


def draw(rng):
    op = rng.choice(['gate', 'gate', 'gemm', 'gemm', 'gemm', 'weight'])
    if op == 'gate':
        groups = rng.choice([1, 1, 2, 4, 8, 16])
        E = max(groups * rng.randint(max(1, 8 // groups), 512 // groups), 8)
        topk_groups = rng.randint(1, groups)
        k = rng.randint(1, min(16, E // groups * topk_groups))
        scoring = rng.choice(['sigmoid', 'softmax'])
        return _gate(None, _spread(rng, 1, 40000), E, k, scoring, rng.choice(['f32', 'bf16', 'f16']),
                     rng.random() < 0.6, groups, topk_groups, rng.choice(['top2', 'max']), rng.random() < 0.6,
                     round(rng.uniform(0.5, 4.0), 2), rng.choice([0.0, 0.0, 0.1, 0.5]), rng.random() < 0.5)
    if op == 'weight':
        return _weight(None, _spread(rng, 1, 16), _spread(rng, 100, 5000), _spread(rng, 100, 7000, 8),
                       rng.choice(['f32', 'bf16', 'f16']))
    layout = rng.choice(['masked', 'segments', 'segments'])
    b = 'nk' if layout == 'masked' else rng.choice(['nk', 'nk', 'kn'])
    epilogue = rng.choice(['bf16', 'f32', 'swiglu']) if b == 'nk' else rng.choice(['bf16', 'f32'])
    G = _spread(rng, 1, 48)
    K = _spread(rng, 128, 7168, 16)
    N = _spread(rng, 256, 4096, 256) if epilogue == 'swiglu' else _spread(rng, 64, 7168, 16 if b == 'kn' else 8)
    if layout == 'masked':
        cap = _spread(rng, 16, 512)
        return _gemm(None, layout, G, _spread(rng, 1, max(1, G * cap // 3)), cap, 1, N, K, b, epilogue)
    align = rng.choice([1, 128])
    rows = _spread(rng, 128, 16384, 128) if align == 128 else _spread(rng, 1, 16000)
    return _gemm(None, layout, G, rows, 0, align, N, K, b, epilogue, epilogue == 'swiglu' and rng.random() < 0.5)


def _busy_groups(c):
    """Expected number of groups that have a row (the others' weights need not be read)."""
    units = max(1, c['rows'] // c['align'])
    return c['G'] * (1 - (1 - 1 / c['G']) ** units)


def work(c):
    if c['op'] == 'gate':
        T, E, k = c['T'], c['E'], c['k']
        size = DTYPES[c['dtype']].itemsize
        by = T * E * size + T * k * 12 + (4 * E if c['bias'] else 0)
        fl = T * E * 6
        if c['train']:
            # what the gradient needs of the logits: all of a row for softmax scores, the chosen ones otherwise
            whole = c['scoring'] == 'softmax' and not c['renorm']
            by += T * E * size + T * k * 12 + (T * E * size if whole else T * k * size)
            fl += T * E * 4
        return dict(bytes=by, flops=fl)
    if c['op'] == 'weight':
        n = c['G'] * c['N'] * c['K']
        return dict(bytes=n * DTYPES[c['dtype']].itemsize + n + 4 * n // (BLOCK * BLOCK), flops=3 * n)
    rows, N, K = c['rows'], c['N'], c['K']
    KB, NB = -(-K // BLOCK), -(-N // BLOCK)
    by = rows * (K + 4 * KB) + _busy_groups(c) * (N * K + 4 * NB * KB)
    if c['epilogue'] == 'swiglu':
        by += rows * (N // 2 + 4 * (N // 2 // BLOCK)) + (rows * N * 2 if c['pre'] else 0)
    else:
        by += rows * N * (4 if c['epilogue'] == 'f32' else 2)
    return dict(bytes=by, flops=2 * rows * N * K)


# ----------------------------------------------------------------------------- inputs
def _blocks_of_rows(x):
    """x [.., K] -> e4m3 and one fp32 scale per row and 128 channels (the last block may be short)."""
    K = x.shape[-1]
    xp = torch.nn.functional.pad(x.float(), (0, -K % BLOCK)).unflatten(-1, (-1, BLOCK))
    amax = xp.abs().amax(-1).clamp_min(AMAX_FLOOR)
    top = torch.full_like(amax, FP8_MAX)
    q = (xp * (top / amax).unsqueeze(-1)).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return q.flatten(-2)[..., :K].contiguous(), amax / top


def _blocks_of_weight(w):
    """w [G, N, K] -> e4m3 and one fp32 scale per 128 x 128 block (the last ones may be short)."""
    G, N, K = w.shape
    wp = torch.nn.functional.pad(w.float(), (0, -K % BLOCK, 0, -N % BLOCK))
    wp = wp.unflatten(2, (-1, BLOCK)).unflatten(1, (-1, BLOCK))          # [G, NB, 128, KB, 128]
    amax = wp.abs().amax((2, 4)).clamp_min(AMAX_FLOOR)
    top = torch.full_like(amax, FP8_MAX)
    q = (wp * (top / amax)[:, :, None, :, None]).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return q.flatten(1, 2).flatten(2, 3)[:, :N, :K].contiguous(), amax / top


def prepare(c, seed):
    dev = _dev()
    g = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    s = dict(case=dict(c))
    if c['op'] == 'gate':
        T, E = c['T'], c['E']
        # a trained gate: logits of some spread, experts of unequal popularity
        logits = torch.randn(T, E, generator=g, device=dev) * 1.5 + torch.randn(E, generator=g, device=dev) * 0.5
        if c['masked']:
            gone = torch.rand(T, E, generator=g, device=dev) < c['masked']
            gone |= torch.rand(T, 1, generator=g, device=dev) < c['masked']
            logits = logits.masked_fill(gone, -math.inf)
        s['logits'] = logits.to(DTYPES[c['dtype']])
        s['bias'] = torch.randn(E, generator=g, device=dev) * 0.05 if c['bias'] else None
        s['dw'] = torch.randn(T, c['k'], generator=g, device=dev) if c['train'] else None
        return s
    if c['op'] == 'weight':
        w = torch.randn(c['G'], c['N'], c['K'], generator=g, device=dev, dtype=torch.bfloat16) * 0.02
        s['w'] = w.to(DTYPES[c['dtype']])
        return s
    G, N, K, rows = c['G'], c['N'], c['K'], c['rows']
    masked = c['layout'] == 'masked'
    # rows of each group: every row, or every 128-row unit, falls to a group at random
    units = rows // c['align']
    counts = torch.bincount(torch.randint(0, G, (units,), generator=host), minlength=G) * c['align']
    if masked:
        counts = counts.clamp_max(c['cap'])
    shape = (G, c['cap']) if masked else (rows,)
    x = torch.randn(*shape, K, generator=g, device=dev, dtype=torch.bfloat16)
    if not masked and c['align'] > 1:
        # padded segments: the last rows of each are zeros
        used = counts - torch.minimum(torch.randint(0, c['align'], (G,), generator=host), counts)
        ends = torch.cumsum(counts, 0)
        at = torch.arange(rows)
        of = torch.bucketize(at, ends, right=True)
        x[(at >= (ends - counts + used)[of]).to(dev)] = 0
    s['a'], s['sa'] = _blocks_of_rows(x)
    del x
    shape_b = (G, K, N) if c['b'] == 'kn' else (G, N, K)
    # rows of 64 groups at a time: the fp32 of all weights at once would be the largest tensor by far
    parts = [_blocks_of_weight(torch.randn(1, *shape_b[1:], generator=g, device=dev, dtype=torch.bfloat16) * 0.02)
             for _ in range(G)]
    s['b'] = torch.cat([p[0].view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn)
    s['sb'] = torch.cat([p[1] for p in parts])
    del parts
    s['rows_of'] = counts.tolist()
    s['most'] = max(1, max(s['rows_of']))
    if masked:
        s['counts'] = counts.to(torch.int32).to(dev)
        s['offsets'] = None
    else:
        s['counts'] = None
        s['offsets'] = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(counts, 0)]).to(dev)
    # the outputs are the caller's buffers; rows behind a group's last are left as they are
    if c['epilogue'] == 'swiglu':
        s['h'] = torch.zeros(*shape, N // 2, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        s['hs'] = torch.zeros(*shape, N // 2 // BLOCK, device=dev)
        s['out'] = torch.zeros(*shape, N, dtype=torch.bfloat16, device=dev) if c['pre'] else None
    else:
        s['out'] = torch.zeros(*shape, N, dtype=DTYPES[c['epilogue']], device=dev)
    return s


# ----------------------------------------------------------------------------- the passes
def run(s):
    c = s['case']
    if own:
        return _own(s, c)
    return {'gate': _plain_gate, 'gemm': _plain_gemm, 'weight': _plain_weight}[c['op']](s, c)


def _own(s, c):
    from deepep_trn_b200.ops import gemm, moe_ops
    if c['op'] == 'gate':
        idx, w = moe_ops.router_gate(s['logits'], c['k'], scoring=c['scoring'], bias=s['bias'],
                                     num_groups=c['groups'], topk_groups=c['topk_groups'],
                                     group_score=c['group_score'], renormalize=c['renorm'], scale=c['scale'])
        if not c['train']:
            return dict(idx=idx, w=w)
        d = moe_ops.router_gate_bwd(s['logits'], idx, s['dw'], scoring=c['scoring'], renormalize=c['renorm'],
                                    scale=c['scale'])
        return dict(idx=idx, w=w, dlogits=d)
    if c['op'] == 'weight':
        q, sc = gemm.quantize_fp8_weight(s['w'])
        return dict(q=q, scales=sc)
    if c['epilogue'] == 'swiglu':
        h, hs, pre = gemm.grouped_gemm_fp8_block(s['a'], s['sa'], s['b'], s['sb'], offsets=s['offsets'],
                                                 counts=s['counts'], epilogue='swiglu', h_out=s['h'],
                                                 h_scales=s['hs'], out=s['out'], save_preact=c['pre'])
        return dict(h=h, hs=hs, pre=pre)
    out = gemm.grouped_gemm_fp8_block(s['a'], s['sa'], s['b'], s['sb'], offsets=s['offsets'], counts=s['counts'],
                                      epilogue=c['epilogue'], b_layout=c['b'], out=s['out'])
    return dict(out=out)


def _plain_gate(s, c):
    # scores and selection in 64 bits: two experts whose scores differ by less than a 32-bit rounding
    # are still in order; ties go to the lower index (stable sort)
    x = s['logits'].double().clamp_max(torch.finfo(torch.float32).max)
    T, E = x.shape
    k, n = c['k'], c['groups']
    open_ = x > -math.inf
    low = torch.full_like(x, -math.inf)
    if c['scoring'] == 'sigmoid':
        score = torch.sigmoid(x)
    else:
        top = torch.where(open_, x, torch.full_like(x, -1e300)).amax(1, keepdim=True)
        e = torch.where(open_, torch.exp(x - top), torch.zeros_like(x))
        score = e / e.sum(1, keepdim=True).clamp_min(1e-300)
    pick = score + s['bias'].double() if s['bias'] is not None else score
    pick = torch.where(open_, pick, low)
    if n > 1:
        by = torch.sort(pick.view(T, n, E // n), dim=2, descending=True).values
        two = by[..., :2]
        gs = by[..., 0] if c['group_score'] == 'max' else torch.where(two > -math.inf, two, 0.0).sum(2)
        gs = torch.where(by[..., 0] > -math.inf, gs, -math.inf)
        keep = torch.sort(gs, dim=1, descending=True, stable=True).indices[:, :c['topk_groups']]
        on = torch.zeros(T, n, dtype=torch.bool, device=x.device).scatter_(1, keep, True)
        pick = torch.where(on.repeat_interleave(E // n, 1), pick, low)
    vals, idx = torch.sort(pick, dim=1, descending=True, stable=True)
    vals, idx = vals[:, :k], idx[:, :k]
    has = vals > -math.inf
    got = torch.where(has, score.gather(1, idx), torch.zeros_like(vals))
    total = got.sum(1, keepdim=True).clamp_min(1e-300)
    w = got / total if c['renorm'] else got
    w = w * c['scale']
    out = dict(idx=torch.where(has, idx, -torch.ones_like(idx)), w=w.float())
    if not c['train']:
        return out
    dw = torch.where(has, s['dw'].double() * c['scale'], torch.zeros_like(vals))
    if c['renorm']:
        p = got / total
        ds = (dw - (p * dw).sum(1, keepdim=True)) / total
        ds = torch.where(has, ds, torch.zeros_like(ds))
    else:
        ds = dw
    if c['scoring'] == 'sigmoid':
        d = torch.zeros_like(x).scatter_add_(1, idx, ds * got * (1 - got))
    else:
        full = torch.zeros_like(x).scatter_add_(1, idx, ds)
        d = score * (full - (full * score).sum(1, keepdim=True))
    out['dlogits'] = d.to(s['logits'].dtype)
    return out


def _plain_gemm(s, c):
    G, N, K, most = c['G'], c['N'], c['K'], s['most']
    KB = -(-K // BLOCK)
    a = s['a'].float() * s['sa'].repeat_interleave(BLOCK, -1)[..., :K]
    sb = s['sb'].repeat_interleave(BLOCK, 1).repeat_interleave(BLOCK, 2)
    b = s['b'].float() * sb[:, :s['b'].shape[1], :s['b'].shape[2]]
    del sb
    b = b if c['b'] == 'kn' else b.transpose(1, 2)
    dev = a.device
    at = torch.arange(most, device=dev)
    if c['layout'] == 'masked':
        x = a[:, :most]
        valid = at[None] < s['counts'][:, None]
    else:
        first, last = s['offsets'][:-1, None], s['offsets'][1:, None]
        place = first + at
        valid = place < last
        x = a[place.clamp_max(a.shape[0] - 1)]
    pre = torch.bmm(x, b)
    del x, b

    def lay(v, like):
        """Rows of each group into the caller's buffer; the rows behind them keep what they held."""
        if c['layout'] == 'masked':
            r = like.float() if like.dtype == torch.float8_e4m3fn else like.clone()
            r[:, :most] = torch.where(valid[..., None], v.to(r.dtype), r[:, :most])
            return r.to(like.dtype)
        return v[valid].to(like.dtype)

    if c['epilogue'] != 'swiglu':
        return dict(out=lay(pre, s['out']))
    gate, up = pre.unflatten(-1, (-1, 2, BLOCK)).unbind(-2)
    h = gate / (1 + torch.exp(-gate)) * up                       # [G, most, I / 128, 128]
    amax = h.abs().amax(-1).clamp_min(AMAX_FLOOR)
    top = torch.full_like(amax, FP8_MAX)
    q = (h * (top / amax).unsqueeze(-1)).clamp(-FP8_MAX, FP8_MAX).flatten(-2)
    return dict(h=lay(q.to(torch.float8_e4m3fn).float(), s['h']), hs=lay(amax / top, s['hs']),
                pre=lay(pre, s['out']) if c['pre'] else None)


def _plain_weight(s, c):
    q, sc = _blocks_of_weight(s['w'])
    return dict(q=q, scales=sc)


# ----------------------------------------------------------------------------- 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    return {'gate': _exact_gate, 'gemm': _exact_gemm, 'weight': _exact_weight}[c['op']](s, c)


def _exact_gate(s, c):
    """The weights and the gradient at the chosen experts, by differentiation in 64 bits."""
    idx = _plain_gate(s, dict(c, train=False))['idx']
    x = s['logits'].double().requires_grad_()
    has = idx >= 0
    chosen = torch.where(has, x.gather(1, idx.clamp_min(0)), torch.full_like(idx, -math.inf, dtype=torch.float64))
    some = has.any(1, keepdim=True)
    if c['scoring'] == 'sigmoid':
        logs = torch.nn.functional.logsigmoid(chosen)
        if c['renorm']:
            logs = logs - torch.logsumexp(torch.where(has, logs, torch.full_like(logs, -1e6)), 1, keepdim=True)
    elif c['renorm']:
        logs = chosen - torch.logsumexp(torch.where(has, chosen, torch.full_like(chosen, -1e6)), 1, keepdim=True)
    else:
        z = torch.logsumexp(torch.where(torch.isfinite(x), x, torch.full_like(x, -1e6)), 1, keepdim=True)
        logs = chosen - z
    w = torch.where(has, torch.exp(torch.where(has, logs, torch.zeros_like(logs))), torch.zeros_like(logs)) * c['scale']
    out = dict(idx=None, w=w.detach())
    if c['train']:
        (w * torch.where(has, s['dw'].double(), torch.zeros_like(w))).sum().backward()
        out['dlogits'] = torch.where(some & torch.isfinite(s['logits']), x.grad, torch.zeros_like(x))
    return out


def _exact_gemm(s, c):
    G, N, K = c['G'], c['N'], c['K']
    masked = c['layout'] == 'masked'
    lead = (G, c['cap']) if masked else (c['rows'],)
    res = torch.zeros(*lead, N, dtype=torch.float64, device=s['a'].device)
    pad = -K % BLOCK
    begin = 0
    for g, n in enumerate(s['rows_of']):
        if n:
            q = s['a'][g, :n] if masked else s['a'][begin:begin + n]
            f = s['sa'][g, :n] if masked else s['sa'][begin:begin + n]
            a = torch.nn.functional.pad(q.double(), (0, pad)).reshape(n, -1, BLOCK) * f.double()[..., None]
            a = a.reshape(n, -1)[:, :K]
            w = s['b'][g].double()
            at = torch.arange(w.shape[0], device=w.device)[:, None] // BLOCK
            bt = torch.arange(w.shape[1], device=w.device)[None] // BLOCK
            w = w * s['sb'][g].double()[at, bt]
            y = a @ (w if c['b'] == 'kn' else w.t())
            if masked:
                res[g, :n] = y
            else:
                res[begin:begin + n] = y
        begin += n
    if c['epilogue'] != 'swiglu':
        return dict(out=res)
    pre = res.reshape(*lead, N // 256, 2, BLOCK)
    h = torch.sigmoid(pre[..., 0, :]) * pre[..., 0, :] * pre[..., 1, :]
    sc = h.abs().amax(-1).clamp_min(AMAX_FLOOR) / FP8_MAX
    q = h / sc[..., None]
    if masked:
        behind = torch.arange(c['cap'], device=res.device)[None] >= s['counts'][:, None]
        sc[behind] = 0
    return dict(h=q.reshape(*lead, N // 2), hs=sc, pre=res if c['pre'] else None)


def _exact_weight(s, c):
    w = s['w'].double()
    G, N, K = w.shape
    NB, KB = -(-N // BLOCK), -(-K // BLOCK)
    if G * N * K > 1 << 30:
        return None
    sc = torch.empty(G, NB, KB, dtype=torch.float64, device=w.device)
    for i in range(NB):
        for j in range(KB):
            sc[:, i, j] = w[:, i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK].abs().flatten(1).amax(1)
    sc = sc.clamp_min(AMAX_FLOOR) / FP8_MAX
    rows, cols = torch.arange(N, device=w.device) // BLOCK, torch.arange(K, device=w.device) // BLOCK
    return dict(q=w / sc[:, rows][:, :, cols], scales=sc)
