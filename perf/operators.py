"""The expert-row operators and the 4-bit microscaled product as they are measured: cases, inputs and plain forms.

Three operators: rows sorted by expert and back with their gradients (dispatch, dispatch_grad, combine,
combine_grad), microscaled 4-bit quantisation (quantize: written and read back), and the product on
4-bit weights, plain (dense) and per expert (expert_dense).  `own` selects the library's kernels.

Microscaled 4-bit (MXFP4): blocks of 32 along a row share the power of two 2^(floor(log2 amax) - 2), an
element is x / scale rounded to nearest even on 0, 0.5, 1, 1.5, 2, 3, 4, 6 and saturated at 6.
"""
import math

import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
BLOCK = 32


def listed():
    return [
        # a router's choice for one token in a serving loop: latency
        dict(name='dispatch_token', kind='dispatch', tokens=1, top_k=2, experts=8, width=1024, dtype='bf16', dropped=0.0),
        # a long prompt or a training batch, four of 64 experts a token
        dict(name='dispatch_batch', kind='dispatch', tokens=16384, top_k=4, experts=64, width=2048, dtype='bf16', dropped=0.01),
        # its backward at odd sizes: the level-2 nodes of the road graph, three of seven experts
        dict(name='dispatch_grad_odd', kind='dispatch_grad', tokens=13505, top_k=3, experts=7, width=333, dtype='f16', dropped=0.05),
        # the road graph's nodes, two of four direction experts, 256 wide, float32 as the graph layers keep them
        dict(name='combine_nodes', kind='combine', tokens=96493, top_k=2, experts=4, width=256, dtype='f32', dropped=0.02),
        # a training batch's way back
        dict(name='combine_grad_batch', kind='combine_grad', tokens=16384, top_k=4, experts=64, width=2048, dtype='bf16', dropped=0.01),
        # node features of the level-3 graph at a width that ends inside a block
        dict(name='quantize_odd', kind='quantize', rows=3410, k=1000, dtype='bf16'),
        # a float32 master matrix turned into 4-bit weights and looked at
        dict(name='quantize_weights', kind='quantize', rows=4096, k=8192, dtype='f32'),
        # one token through a square layer: bound by the weights' bytes
        dict(name='dense_token', kind='dense', rows=1, k=4096, n=4096, dtype='bf16', act='linear'),
        # the level-1 nodes of the road graph through a 256-wide layer with bias and ReLU
        dict(name='dense_nodes', kind='dense', rows=48332, k=256, n=256, dtype='f32', act='relu'),
        # a long prompt through a wide layer: bound by the matrix cores
        dict(name='dense_batch', kind='dense', rows=8192, k=8192, n=8192, dtype='bf16', act='linear'),
        # a step of 32 sequences through 32 experts: bound by the weights of the experts that are met
        dict(name='expert_dense_step', kind='expert_dense', tokens=32, top_k=4, experts=32, k=2048, n=4096, dtype='bf16', act='linear'),
        # a long prompt through 16 experts of uneven load
        dict(name='expert_dense_batch', kind='expert_dense', tokens=16384, top_k=2, experts=16, k=2048, n=4096, dtype='bf16', act='relu'),
    ]


def _spread(rng, lo, hi):
    """A size whose logarithm is uniform in the range, odd ones as likely as even ones."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(['dispatch', 'dispatch_grad', 'combine', 'combine_grad', 'quantize', 'dense', 'dense', 'expert_dense'])
    dtype = rng.choice(['f32', 'bf16', 'f16'])
    act = rng.choice(['linear', 'relu'])
    if kind == 'quantize':
        k = _spread(rng, 32, 8192)
        return dict(kind=kind, rows=_spread(rng, 1, min(16384, (4096 * 8192) // k)), k=k, dtype=dtype)
    if kind == 'dense':
        k, n = _spread(rng, 32, 8192), _spread(rng, 16, 8192)
        return dict(kind=kind, rows=_spread(rng, 1, min(49152, (8192 ** 3) // (k * n))), k=k, n=n, dtype=dtype, act=act)
    experts = _spread(rng, 2, 64)
    top_k = rng.randint(1, min(experts, 6))
    if kind == 'expert_dense':
        k, n = _spread(rng, 64, 2048), _spread(rng, 64, 4096)
        experts = min(experts, 32)
        return dict(kind=kind, tokens=_spread(rng, 1, 32768 // top_k), top_k=min(top_k, experts), experts=experts, k=k, n=n,
                    dtype=dtype, act=act)
    width = _spread(rng, 16, 2048)
    return dict(kind=kind, tokens=_spread(rng, 1, 65536 // (2 * top_k)), top_k=top_k, experts=experts, width=width, dtype=dtype,
                dropped=rng.choice([0.0, 0.01, 0.2]))


# ---- inputs ------------------------------------------------------------------------------------------

def _normal(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device='cuda', dtype=torch.float32).to(dtype)


def _router(g, tokens, top_k, experts, dropped):
    """int32 [tokens, top_k]: the largest of uneven random scores; a share is dropped (-1), as by a capacity."""
    lean = torch.randn(experts, generator=g, device='cuda') * 0.5
    scores = torch.randn((tokens, experts), generator=g, device='cuda') + lean
    index = scores.topk(top_k, dim=1).indices.to(torch.int32)
    if dropped:
        gone = torch.rand((tokens, top_k), generator=g, device='cuda') < dropped
        index = torch.where(gone, torch.full_like(index, -1), index)
    return index.contiguous()


def _features(g, rows, k, dtype):
    """Rows of differing size with a few wide columns, as activations have."""
    x = torch.randn((rows, k), generator=g, device='cuda')
    x *= torch.exp(0.5 * torch.randn((rows, 1), generator=g, device='cuda'))
    x *= torch.exp(0.5 * torch.randn((1, k), generator=g, device='cuda'))
    return x.to(dtype)


def _weights(g, shape):
    """4-bit weights as a checkpoint holds them: codes uint8 [.., blocks * 16], the even column in the low four
    bits, rows padded with zeros to whole blocks, and scales uint8 [.., blocks] (exponent + 127)."""
    k = shape[-1]
    kb = -(-k // BLOCK)
    mag = torch.randint(0, 8, shape[:-1] + (kb * BLOCK,), generator=g, device='cuda', dtype=torch.uint8)
    # fewer large codes than small ones, as a bell-shaped matrix has them
    mag = torch.minimum(mag, torch.randint(0, 8, mag.shape, generator=g, device='cuda', dtype=torch.uint8))
    sign = torch.randint(0, 2, mag.shape, generator=g, device='cuda', dtype=torch.uint8)
    code = mag | (sign << 3)
    code[..., k:] = 0
    low = round(math.log2(1.0 / math.sqrt(k))) - 1
    scales = torch.randint(127 + low - 1, 127 + low + 2, shape[:-1] + (kb,), generator=g, device='cuda', dtype=torch.uint8)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).contiguous(), scales


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    kind, dtype = case['kind'], DTYPES[case['dtype']]
    s = {'case': case, 'dtype': dtype}
    if kind == 'quantize':
        s['x'] = _features(g, case['rows'], case['k'], dtype)
        return s
    if kind in ('dense', 'expert_dense'):
        rows = case['rows'] if kind == 'dense' else case['tokens']
        s['x'] = _features(g, rows, case['k'], dtype)
        lead = () if kind == 'dense' else (case['experts'],)
        s['codes'], s['scales'] = _weights(g, lead + (case['n'], case['k']))
        s['bias'] = _normal(g, lead + (case['n'],)) if case['act'] == 'relu' else None
    else:
        rows, width = case['tokens'] * case['top_k'], case['width']
        if kind == 'dispatch':
            s['x'] = _normal(g, (case['tokens'], width), dtype)
        else:
            s['rows'] = _normal(g, (rows, width), dtype)
        if kind == 'combine_grad':
            s['grad'] = _normal(g, (case['tokens'], width), dtype)
        s['weights'] = torch.rand((case['tokens'], case['top_k']), generator=g, device='cuda')
    if kind != 'dense':
        s['index'] = _router(g, case['tokens'], case['top_k'], case['experts'], case.get('dropped', 0.0))
        # the order of an earlier step, which the way back and the experts' products are given
        s['offsets'], s['order'], s['slot'] = _sort(s['index'], case['experts'])
        if kind == 'expert_dense':
            s['most'] = int((s['offsets'][1:] - s['offsets'][:-1]).max())
    if own:
        import gunet_amd
        if 'codes' in s:
            s['w4'] = gunet_amd.Mxfp4Tensor.from_codes(s['codes'], s['scales'], case['k'])
        if 'index' in s and kind != 'dispatch':
            s['plan'] = gunet_amd.expert_plan(s['index'], case['experts'])
    return s


# ---- plain forms -------------------------------------------------------------------------------------

def _sort(index, experts):
    """(offsets [E + 1], order [T * k], slot [T, k]): flat positions sorted by expert, -1 behind the last one."""
    flat = index.reshape(-1)
    n = flat.numel()
    key = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    order = torch.sort(key, stable=True).indices
    counts = (key[None, :] == torch.arange(experts, device=key.device, dtype=key.dtype)[:, None]).sum(1)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    row = torch.arange(n, device=key.device)
    kept = row < offsets[-1]
    slot = torch.empty_like(order)
    slot[order] = torch.where(kept, row, torch.full_like(row, -1))
    order = torch.where(kept, order, torch.full_like(order, -1))
    return offsets.to(torch.int32), order.to(torch.int32), slot.to(torch.int32).reshape(index.shape)


def _of_slots(rows, slot):
    """rows[slot] in 32 bits, zeros where a choice was dropped: [T, k, width]."""
    got = rows[slot.clamp(min=0).long()].float()
    return torch.where((slot >= 0)[..., None], got, torch.zeros_like(got))


def _quantized(x):
    """The 4-bit values of x [rows, k] in 32 bits."""
    rows, k = x.shape
    kb = -(-k // BLOCK)
    v = torch.nn.functional.pad(x.float(), (0, kb * BLOCK - k)).view(rows, kb, BLOCK)
    top = v.abs().amax(-1, keepdim=True)
    # floor(log2 top) from the number's own exponent; below 2^-125 the scale ends at 2^-127
    e = torch.clamp(torch.frexp(top).exponent - 1 - 2, min=-127)
    e = torch.where(top > 0, e, torch.full_like(e, -127))
    a = torch.ldexp(torch.ldexp(v.abs(), -(e // 2)), -(e - e // 2))
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = torch.clamp(torch.round(a / step) * step, max=6.0)
    q = torch.ldexp(torch.ldexp(torch.copysign(q, v), e // 2), e - e // 2)
    q = torch.where(torch.isfinite(top), q, torch.full_like(q, math.nan))
    return q.view(rows, kb * BLOCK)[:, :k]


def _levels(device, dtype=torch.float32):
    return torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=device, dtype=dtype)


def _dequantized(codes, scales, k):
    """The values of 4-bit weights in 32 bits, [.., k]."""
    code = torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[:-1] + (scales.shape[-1], BLOCK))
    v = _levels(codes.device)[code.long()] * torch.exp2(scales.float() - 127)[..., None]
    return v.view(codes.shape[:-1] + (-1,))[..., :k]


def _finish(out, bias, case, dtype):
    if bias is not None:
        out = out + bias
    return (torch.clamp(out, min=0) if case['act'] == 'relu' else out).to(dtype)


def _plain(s):
    case, dtype = s['case'], s['dtype']
    kind = case['kind']
    if kind == 'quantize':
        return _quantized(s['x']).to(dtype)
    if kind == 'dense':
        return _finish(_quantized(s['x']) @ _dequantized(s['codes'], s['scales'], case['k']).t(), s['bias'], case, dtype)
    if kind == 'dispatch':
        offsets, order, slot = _sort(s['index'], case['experts'])
        token = torch.div(order.clamp(min=0), case['top_k'], rounding_mode='floor').long()
        rows = torch.where((order >= 0)[:, None], s['x'][token], torch.zeros_like(s['x'][:1]))
        return {'offsets': offsets, 'order': order, 'slot': slot, 'rows': rows}
    order, slot = s['order'], s['slot']
    if kind == 'dispatch_grad':
        return _of_slots(s['rows'], slot).sum(1).to(dtype)
    if kind == 'combine':
        return (_of_slots(s['rows'], slot) * s['weights'][..., None]).sum(1).to(dtype)
    token = torch.div(order.clamp(min=0), case['top_k'], rounding_mode='floor').long()
    if kind == 'combine_grad':
        w = torch.where(order >= 0, s['weights'].reshape(-1)[order.clamp(min=0).long()], torch.zeros_like(s['weights'].reshape(-1)))
        grad_rows = torch.where((order >= 0)[:, None], s['grad'].float()[token] * w[:, None], torch.zeros_like(w[:, None]))
        grad_weights = (_of_slots(s['rows'], slot) * s['grad'].float()[:, None, :]).sum(-1)
        return {'rows': grad_rows.to(dtype), 'weights': grad_weights}
    # the experts' products as one batched product over groups padded to the fullest one
    q = _quantized(s['x'])
    row = torch.arange(order.numel(), device=order.device)
    expert = (row[:, None] >= s['offsets'][None, 1:]).sum(1).clamp(max=case['experts'] - 1)
    place = torch.where(order >= 0, row - s['offsets'].long()[expert], torch.full_like(row, s['most']))
    padded = q.new_zeros((case['experts'], s['most'] + 1, case['k']))
    padded[expert, place] = q[token]
    out = torch.bmm(padded, _dequantized(s['codes'], s['scales'], case['k']).transpose(1, 2).contiguous())
    if s['bias'] is not None:
        out = out + s['bias'][:, None, :]
    out = out[expert, place]
    out = torch.clamp(out, min=0) if case['act'] == 'relu' else out
    return torch.where((order >= 0)[:, None], out, torch.zeros_like(out)).to(dtype)


def run(s):
    if not own:
        return _plain(s)
    import gunet_amd
    case, kind = s['case'], s['case']['kind']
    if kind == 'dispatch':
        plan = gunet_amd.expert_plan(s['index'], case['experts'])
        return {'offsets': plan.offsets, 'order': plan.order, 'slot': plan.slot, 'rows': gunet_amd.expert_dispatch(s['x'], plan)}
    if kind == 'dispatch_grad':
        return gunet_amd.expert_dispatch_grad(s['rows'], s['plan'])
    if kind == 'combine':
        return gunet_amd.expert_combine(s['rows'], s['weights'], s['plan'])
    if kind == 'combine_grad':
        grad_rows, grad_weights = gunet_amd.expert_combine_grad(s['grad'], s['rows'], s['weights'], s['plan'])
        return {'rows': grad_rows, 'weights': grad_weights}
    if kind == 'quantize':
        return gunet_amd.mxfp4_dequantize(gunet_amd.mxfp4_quantize(s['x']), s['dtype'])
    if kind == 'dense':
        return gunet_amd.mxfp4_dense(s['x'], s['w4'], s['bias'], case['act'])
    return gunet_amd.mxfp4_expert_dense(s['x'], s['w4'], s['plan'], s['bias'], case['act'])


# ---- the work and the definition ---------------------------------------------------------------------

def work(case):
    size = {'f32': 4, 'bf16': 2, 'f16': 2}[case['dtype']]
    kind = case['kind']
    if kind == 'quantize':   # the values read, codes and scales written and read back, the values written
        n = case['rows'] * case['k']
        return {'bytes': n * size * 2 + 2 * n * 17 // 32, 'flops': 4 * n}
    if kind in ('dense', 'expert_dense'):
        k, n, bias = case['k'], case['n'], 4 * case['n'] if case['act'] == 'relu' else 0
        weights = n * (-(-k // BLOCK)) * 17 + bias
        if kind == 'dense':
            return {'bytes': case['rows'] * (k + n) * size + weights, 'flops': 2 * case['rows'] * k * n}
        rows = case['tokens'] * case['top_k']
        met = case['experts'] * (1 - (1 - case['top_k'] / case['experts']) ** case['tokens'])   # experts that are met
        return {'bytes': case['tokens'] * k * size + rows * n * size + round(met * weights) + 4 * rows, 'flops': 2 * rows * k * n}
    t, c = case['tokens'], case['width']
    n = t * case['top_k']
    row = c * size
    if kind == 'dispatch':
        return {'bytes': 12 * n + 4 * case['experts'] + (t + n) * row, 'flops': 0}
    if kind == 'dispatch_grad':
        return {'bytes': 4 * n + (t + n) * row, 'flops': n * c}
    if kind == 'combine':
        return {'bytes': 8 * n + (t + n) * row, 'flops': 2 * n * c}
    return {'bytes': 12 * n + (t + 2 * n) * row, 'flops': 3 * n * c}


def _exact_quantized(x):
    """4-bit values of x in 64 bits: the nearest level by distance, the even code on a tie."""
    rows, k = x.shape
    kb = -(-k // BLOCK)
    v = torch.zeros((rows, kb * BLOCK), dtype=torch.float64, device=x.device)
    v[:, :k] = x.double()
    v = v.view(rows, kb, BLOCK)
    top = v.abs().amax(-1)
    e = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
    # the logarithm may round up to the next whole number just below a power of two
    e = torch.where(torch.exp2(e) > top, e - 1, e)
    e = torch.where(torch.exp2(e + 1) <= top, e + 1, e)
    scale = torch.exp2(torch.where(top > 0, torch.clamp(e - 2, min=-127), torch.full_like(e, -127)))[..., None]
    a = v.abs() / scale
    level = torch.zeros_like(a)
    # the middles between levels; at a middle the lower level wins where its code is even
    for middle, upper, tie_up in ((.25, .5, False), (.75, 1., True), (1.25, 1.5, False), (1.75, 2., True),
                                  (2.5, 3., False), (3.5, 4., True), (5., 6., False)):
        level = torch.where(a >= middle if tie_up else a > middle, torch.full_like(a, upper), level)
    level = torch.where(v < 0, -level, level) * scale
    level = torch.where(torch.isfinite(top)[..., None], level, torch.full_like(level, math.nan))
    return level.view(rows, kb * BLOCK)[:, :k]


def _exact_weights(codes, scales, k):
    v = torch.empty(codes.shape[:-1] + (codes.shape[-1] * 2,), dtype=torch.float64, device=codes.device)
    table = _levels(codes.device, torch.float64)
    v[..., 0::2] = table[(codes % 16).int()]
    v[..., 1::2] = table[torch.div(codes, 16, rounding_mode='floor').int()]
    return (v * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, -1))[..., :k]


def _exact_product(x, w, bias, case):
    out = x @ w.t()
    if bias is not None:
        out += bias.double()
    return out.clamp_(min=0) if case['act'] == 'relu' else out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case['kind']
    if kind == 'quantize':
        return _exact_quantized(s['x'])
    if kind == 'dense':
        return _exact_product(_exact_quantized(s['x']), _exact_weights(s['codes'], s['scales'], case['k']), s['bias'], case)
    index = s['index'].long()
    t, top_k = index.shape
    token = torch.arange(t, device=index.device)[:, None].expand(t, top_k).reshape(-1)
    row = s['slot'].reshape(-1).long()
    kept = (index.reshape(-1) >= 0) & (index.reshape(-1) < case['experts'])
    token, row, n = token[kept], row[kept], t * top_k
    if kind == 'dispatch':
        rows = torch.zeros((n, case['width']), dtype=torch.float64, device=index.device)
        rows[row] = s['x'].double()[token]
        return {'offsets': None, 'order': None, 'slot': None, 'rows': rows}
    if kind == 'expert_dense':
        out = torch.zeros((n, case['n']), dtype=torch.float64, device=index.device)
        q = _exact_quantized(s['x'])
        for e in range(case['experts']):
            mine = index.reshape(-1)[kept] == e
            w = _exact_weights(s['codes'][e], s['scales'][e], case['k'])
            out[row[mine]] = _exact_product(q[token[mine]], w, None if s['bias'] is None else s['bias'][e], case)
        return out
    gate = s['weights'].double().reshape(-1)[kept]
    if kind == 'combine_grad':
        grad = s['grad'].double()[token]
        grad_rows = torch.zeros((n, case['width']), dtype=torch.float64, device=index.device)
        grad_rows[row] = grad * gate[:, None]
        grad_weights = torch.zeros(n, dtype=torch.float64, device=index.device)
        grad_weights[kept] = (grad * s['rows'].double()[row]).sum(1)
        return {'rows': grad_rows, 'weights': grad_weights.view(t, top_k)}
    out = torch.zeros((t, case['width']), dtype=torch.float64, device=index.device)
    part = s['rows'].double()[row]
    return out.index_add_(0, token, part * gate[:, None] if kind == 'combine' else part)
