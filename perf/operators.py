"""What is measured of the operators that sit between the fused projections: attention over packed
sequences, rotary positions with several axes (with the normalisation of query and key heads), and the
norm around a block with its gate, scale, shift and residual sum.

`own` selects the side: the plain form (elementary torch operations in FP32, rounded once) or the
package's kernels. Both take what prepare() gives; everything that a call derives from it is derived
inside run().
"""
import math

import torch

own = False

HEAD_DIM = 128
EPS = 1e-6


# ----------------------------------------------------------------------------------------------
# Cases
# ----------------------------------------------------------------------------------------------
def _attention(name, lengths, heads, kv_heads, causal, train, pad=0):
    return dict(name=name, op='attention', lengths=','.join(map(str, lengths)), heads=heads, kv_heads=kv_heads,
                causal=causal, train=train, pad=pad)


def _rotary(name, tokens, heads, kv_heads, axes, interleaved, norm, train, start=0):
    return dict(name=name, op='rotary', tokens=tokens, heads=heads, kv_heads=kv_heads, axes=axes,
                interleaved=interleaved, norm=norm, train=train, start=start)


def _norm(name, lengths, hidden, center, branch, weight, modulated, train):
    return dict(name=name, op='norm', lengths=','.join(map(str, lengths)), hidden=hidden, center=center,
                branch=branch, weight=weight, modulated=modulated, train=train)


def listed():
    return [
        # A validation step on three short prompts of 1, 5 and 17 tokens: nothing but latency.
        _attention('attention_tiny', (1, 5, 17), 8, 8, False, False),
        # The two-layer training program of the tests: 512 tokens, 8 heads, one sequence.
        _attention('attention_small_train', (512,), 8, 8, False, True),
        # Prompts packed to the workspace capacity of 8192 tokens, odd lengths, 32 query heads on 8 key/value
        # heads, causal, evaluation only; the last rows are padding.
        _attention('attention_prompt_gqa', (4097, 2501, 1, 0, 1213, 333), 32, 8, True, False, pad=47),
        # Video training: one sequence of an odd length, eight local heads, every token sees every other.
        _attention('attention_video_train', (16383,), 8, 8, False, True),
        # Packed causal training with grouped heads (32 query heads, 4 key/value heads).
        _attention('attention_packed_train', (5000, 1777, 129, 1, 1284), 32, 4, True, True),
        # The smallest rotary call: 23 tokens, one axis, far positions, no head norm.
        _rotary('rotary_tiny', 23, 8, 8, 1, False, False, False, start=1000003),
        # Context-parallel video training at CP=8: all 131072 tokens, four local heads, three axes, head norm.
        _rotary('rotary_video_train', 131072, 4, 4, 3, True, True, True),
        # Grouped heads in a longer prompt, one axis, half-split pairs, evaluation.
        _rotary('rotary_prompt_gqa', 16384, 32, 8, 1, False, False, False),
        # A norm with its residual sum on a handful of rows.
        _norm('norm_tiny', (23,), 1024, False, True, True, False, False),
        # The block of a video model: gate on the attention output, residual sum, layer norm with scale and
        # shift for each of the packed samples, training.
        _norm('norm_modulated_train', (9000, 4001, 3383), 4096, True, True, False, True, True),
        # An RMS norm with the residual sum at the width of the widest configuration, evaluation.
        _norm('norm_residual', (8191,), 5120, False, True, True, False, False),
        # The same in training at 4096 columns and an odd number of rows.
        _norm('norm_residual_train', (4097,), 4096, False, True, True, False, True),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def _split(rng, total, parts):
    cuts = sorted(rng.randint(0, total) for _ in range(parts - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def draw(rng):
    op = rng.choice(('attention', 'attention', 'rotary', 'norm'))
    if op == 'attention':
        tokens = _spread(rng, 1, 16383)
        most = max(1, 8 * 16383 ** 2 // tokens ** 2)
        heads = rng.choice([h for h in (1, 2, 3, 4, 5, 8, 16, 24, 32, 40) if h <= most])
        kv_heads = rng.choice([h for h in range(1, heads + 1) if heads % h == 0])
        pad = rng.choice((0, 0, 1, 77))
        lengths = _split(rng, tokens, rng.randint(1, 6))
        case = _attention('', lengths, heads, kv_heads, rng.random() < 0.5, rng.random() < 0.6, pad if tokens < 8000 else 0)
    elif op == 'rotary':
        heads = rng.choice((1, 2, 3, 4, 5, 8, 24, 32, 40))
        kv_heads = rng.choice([h for h in range(1, heads + 1) if heads % h == 0])
        tokens = _spread(rng, 1, 131072 * 8 // (heads + kv_heads))
        case = _rotary('', tokens, heads, kv_heads, rng.choice((1, 2, 3)), rng.random() < 0.5, rng.random() < 0.5,
                       rng.random() < 0.5, rng.choice((0, 0, 5, 250001)))
    else:
        hidden = 8 * _spread(rng, 8, 1024)
        tokens = _spread(rng, 1, min(32768, 16384 * 4096 // hidden))
        case = _norm('', _split(rng, tokens, rng.randint(1, 5)), hidden, rng.random() < 0.5, rng.random() < 0.7,
                     rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5)
    del case['name']
    return case


# ----------------------------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------------------------
def _lengths(case):
    return [int(n) for n in case['lengths'].split(',')]


def _sections(axes):
    return {1: (64,), 2: (32, 32), 3: (16, 24, 24)}[axes]


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=gen, device='cuda') * std + mean).bfloat16()

    state = dict(case)
    if 'lengths' in case:
        ends = [0]
        for n in _lengths(case):
            ends.append(ends[-1] + n)
        state['cu_seqlens'] = torch.tensor(ends, dtype=torch.int32, device='cuda')
    if case['op'] == 'attention':
        tokens = sum(_lengths(case)) + case['pad']
        for name, heads in (('q', case['heads']), ('k', case['kv_heads']), ('v', case['kv_heads'])):
            state[name] = normal(tokens, heads, HEAD_DIM)
        if case['train']:
            state['do'] = normal(tokens, case['heads'], HEAD_DIM)
    elif case['op'] == 'rotary':
        tokens = case['tokens']
        token = torch.arange(tokens, device='cuda') + case['start']
        sections = _sections(case['axes'])
        # frames of 48 x 80 patches, as a video model numbers them; one axis: the token's own position
        axes = {1: (token,), 2: (token // 80, token % 80), 3: (token // 3840, token // 80 % 48, token % 80)}[case['axes']]
        state['positions'] = torch.stack(axes, 1).int()
        state['sections'] = sections
        state['inv_freq'] = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64, device='cuda') / n)
                                       for n in sections])
        for name, heads in (('q', case['heads']), ('k', case['kv_heads'])):
            state[name] = normal(tokens, heads, HEAD_DIM, std=1.5)
            state[name + '_weight'] = normal(HEAD_DIM, std=0.1, mean=1.0) if case['norm'] else None
            if case['train']:
                state['d' + name] = normal(tokens, heads, HEAD_DIM)
    else:
        tokens, hidden, samples = sum(_lengths(case)), case['hidden'], len(_lengths(case))
        state['x'] = normal(tokens, hidden, std=2.0, mean=0.25)
        state['branch'] = normal(tokens, hidden) if case['branch'] else None
        state['weight'] = normal(hidden, std=0.1, mean=1.0) if case['weight'] else None
        for name in ('gate', 'scale', 'shift'):
            present = case['modulated'] and (name != 'gate' or case['branch'])
            state[name] = normal(samples, hidden, std=0.5) if present else None
        if case['train']:
            state['dy'], state['dr'] = normal(tokens, hidden), normal(tokens, hidden)
    return state


def work(case):
    if case['op'] == 'attention':
        lengths, heads, kv_heads = _lengths(case), case['heads'], case['kv_heads']
        tokens = sum(lengths) + case['pad']
        pairs = sum(n * (n + 1) // 2 if case['causal'] else n * n for n in lengths) * heads
        row = 2 * HEAD_DIM * tokens
        moved = row * (2 * heads + 2 * kv_heads)                    # q, o; k, v
        if case['train']:
            moved += row * (2 * heads + 2 * kv_heads)               # do, dq; dk, dv
        return {'bytes': moved, 'flops': pairs * HEAD_DIM * (14 if case['train'] else 4)}
    if case['op'] == 'rotary':
        elements = case['tokens'] * (case['heads'] + case['kv_heads']) * HEAD_DIM
        passes = (3 if case['norm'] else 2) + 2 if case['train'] else 2     # backward of the norm reads its input too
        return {'bytes': passes * 2 * elements + 4 * case['axes'] * case['tokens'], 'flops': 6 * elements}
    tokens, hidden = sum(_lengths(case)), case['hidden']
    moved = 2 + 2 * case['branch']                                  # x, y; branch, r
    if case['train']:
        # dy, dr and the residual sum come in, dx goes out; with a gate the branch comes in and its gradient goes
        # out (without one the branch's gradient is dx)
        moved += 4 + 2 * (case['branch'] and case['modulated'])
    return {'bytes': moved * 2 * tokens * hidden, 'flops': 10 * tokens * hidden}


# ----------------------------------------------------------------------------------------------
# Plain forms
# ----------------------------------------------------------------------------------------------
def _plain_attention(s):
    q, k, v, cu, causal = s['q'], s['k'], s['v'], s['cu_seqlens'], s['causal']
    tokens, heads, _ = q.shape
    group = heads // k.shape[1]
    scale = HEAD_DIM ** -0.5
    row = torch.arange(tokens, device=q.device)
    sample = torch.searchsorted(cu[1:].contiguous(), row.int(), right=True)
    allowed = (sample[:, None] == sample[None, :]) & (row < cu[-1])[:, None]
    if causal:
        allowed &= row[None, :] <= row[:, None]
    qf = q.float().transpose(0, 1)
    kf, vf = (t.float().transpose(0, 1).repeat_interleave(group, 0) for t in (k, v))
    scores = torch.matmul(qf, kf.transpose(1, 2)).mul_(scale).masked_fill_(~allowed, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = scores.sub_(top).exp_()
    p /= p.sum(-1, keepdim=True).clamp_(min=1e-30)
    o = torch.matmul(p, vf)
    out = o.transpose(0, 1).bfloat16()
    if not s['train']:
        return out
    do = s['do'].float().transpose(0, 1) * (row < cu[-1])[:, None]

    def shared(g):          # gradients of a key/value head: the sum over its query heads
        return g.view(heads // group, group, tokens, HEAD_DIM).sum(1).transpose(0, 1).bfloat16()

    dv = shared(torch.matmul(p.transpose(1, 2), do))
    delta = (o * do).sum(-1, keepdim=True)
    ds = torch.matmul(do, vf.transpose(1, 2)).sub_(delta).mul_(p).mul_(scale)
    dq = torch.matmul(ds, kf).transpose(0, 1).bfloat16()
    dk = shared(torch.matmul(ds.transpose(1, 2), qf))
    return out, dq, dk, dv


def _turn(x, cos, sin, interleaved):
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_rotary(s):
    pos, sections = s['positions'], s['sections']
    axis = torch.repeat_interleave(torch.arange(len(sections), device=pos.device),
                                   torch.tensor(sections, device=pos.device), output_size=sum(sections))
    angle = pos.double()[:, axis] * s['inv_freq']
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def forward(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
        return _turn(x, cos, sin, s['interleaved']).bfloat16()

    def backward(x, w, dy):
        g = _turn(dy.float(), cos, -sin, s['interleaved'])
        if w is None:
            return (g.bfloat16(),)
        x = x.float()
        rstd = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        n, gw = x * rstd, g * w.float()
        dx = rstd * (gw - n * (gw * n).mean(-1, keepdim=True))
        return dx.bfloat16(), (g * n).sum((0, 1)).bfloat16()

    outs = [forward(s[name], s[name + '_weight']) for name in 'qk']
    if s['train']:
        for name in 'qk':
            outs += backward(s[name], s[name + '_weight'], s['d' + name])
    return outs


def _plain_norm(s):
    x = s['x'].float()
    tokens, hidden = x.shape
    samples = s['cu_seqlens'].shape[0] - 1
    row = torch.arange(tokens, device=x.device, dtype=torch.int32)
    sample = torch.searchsorted(s['cu_seqlens'][1:].contiguous(), row, right=True)
    member = (sample == torch.arange(samples, device=x.device)[:, None]).float()          # [samples, tokens]
    branch, weight = (None if s[n] is None else s[n].float() for n in ('branch', 'weight'))
    gate, scale, shift = (None if s[n] is None else s[n].float()[sample] for n in ('gate', 'scale', 'shift'))
    r = x
    if branch is not None:
        r = x + (branch if gate is None else gate * branch)
    c = r - r.mean(-1, keepdim=True) if s['center'] else r
    rstd = torch.rsqrt(c.square().mean(-1, keepdim=True) + EPS)
    n = c * rstd
    y = n if weight is None else n * weight
    if scale is not None:
        y = y * (1 + scale) + shift
    outs = [y.bfloat16(), s['x'] if branch is None else r.bfloat16()]
    if not s['train']:
        return outs
    dy, dr = s['dy'].float(), s['dr'].float()
    dz = dy if scale is None else dy * (1 + scale)
    dn = dz if weight is None else dz * weight
    dc = rstd * (dn - n * (dn * n).mean(-1, keepdim=True))
    if s['center']:
        dc = dc - dc.mean(-1, keepdim=True)
    dr = dr + dc
    outs.append(dr.bfloat16())
    if branch is not None:
        outs.append((dr if gate is None else dr * gate).bfloat16())
    if weight is not None:
        outs.append((dz * n).sum(0).bfloat16())
    if gate is not None:
        outs.append((member @ (dr * branch)).bfloat16())
    if scale is not None:
        outs.append((member @ (dy * (n if weight is None else n * weight))).bfloat16())
        outs.append((member @ dy).bfloat16())
    return outs


# ----------------------------------------------------------------------------------------------
# The package's operators, called as a training or evaluation step calls them
# ----------------------------------------------------------------------------------------------


def _package():
    import sys
    if 'fused_gemm_a2a' not in sys.modules:
        sys.path.insert(0, 'fused-gemm-a2a_b200')
    import fused_gemm_a2a
    return fused_gemm_a2a


def _leaves(s, names):
    return [s[n].detach().requires_grad_() for n in names if s[n] is not None]


def _own_attention(s):
    attention = _package().packed_attention
    if not s['train']:
        return attention(s['q'], s['k'], s['v'], s['cu_seqlens'], causal=s['causal'])
    q, k, v = _leaves(s, 'qkv')
    o = attention(q, k, v, s['cu_seqlens'], causal=s['causal'])
    return (o.detach(), *torch.autograd.grad(o, (q, k, v), s['do']))


def _own_rotary(s):
    rotary = _package().rotary_embedding
    names = ('q', 'q_weight', 'k', 'k_weight')
    t = {n: s[n] for n in names}
    if s['train']:
        t = {n: v if v is None else v.detach().requires_grad_() for n, v in t.items()}
    outs = rotary(t['q'], t['k'], s['positions'], s['inv_freq'], s['sections'], interleaved=s['interleaved'],
                  q_weight=t['q_weight'], k_weight=t['k_weight'], eps=EPS)
    if not s['train']:
        return list(outs)
    grads = torch.autograd.grad(outs, [t[n] for n in names if t[n] is not None], (s['dq'], s['dk']))
    return [o.detach() for o in outs] + list(grads)


def _own_norm(s):
    residual_norm = _package().residual_norm
    names = ('x', 'branch', 'weight', 'gate', 'scale', 'shift')
    t = {n: s[n] for n in names}
    if s['train']:
        t = {n: v if v is None else v.detach().requires_grad_() for n, v in t.items()}
    cu = s['cu_seqlens'] if s['modulated'] else None
    y, r = residual_norm(t['x'], t['branch'], weight=t['weight'], gate=t['gate'], scale=t['scale'], shift=t['shift'],
                         cu_seqlens=cu, eps=EPS, center=s['center'])
    if not s['train']:
        return [y, r]
    grads = torch.autograd.grad((y, r), [t[n] for n in names if t[n] is not None], (s['dy'], s['dr']))
    return [y.detach(), r.detach()] + list(grads)


def run(state):
    if own:
        return {'attention': _own_attention, 'rotary': _own_rotary, 'norm': _own_norm}[state['op']](state)
    return {'attention': _plain_attention, 'rotary': _plain_rotary, 'norm': _plain_norm}[state['op']](state)


# ----------------------------------------------------------------------------------------------
# The definitions in 64 bits: sequence by sequence, gradients by differentiation
# ----------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {'attention': _exact_attention, 'rotary': _exact_rotary, 'norm': _exact_norm}[case['op']](s)


def _exact_attention(s):
    lengths, train = _lengths(s), s['train']
    outs = {n: torch.zeros(s[n[-1]].shape if n != 'o' else s['q'].shape, dtype=torch.float64, device='cuda')
            for n in ('o', 'dq', 'dk', 'dv')}
    group = s['heads'] // s['kv_heads']
    first = 0
    for n in lengths:
        rows = slice(first, first + n)
        first += n
        if n == 0:
            continue
        for h in range(s['heads']):
            g = h // group
            q, k, v = (t.double().requires_grad_(train) for t in (s['q'][rows, h], s['k'][rows, g], s['v'][rows, g]))
            scores = q @ k.T / math.sqrt(HEAD_DIM)
            if s['causal']:
                scores = scores.masked_fill(torch.ones(n, n, dtype=torch.bool, device='cuda').triu(1), -math.inf)
            o = scores.softmax(-1) @ v
            outs['o'][rows, h] = o.detach()
            if train:
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), s['do'][rows, h].double())
                outs['dq'][rows, h] = dq
                outs['dk'][rows, g] += dk
                outs['dv'][rows, g] += dv
    return tuple(outs[n] for n in ('o', 'dq', 'dk', 'dv')) if train else outs['o']


def _exact_rotary(s):
    angles, at = [], 0
    for axis, pairs in enumerate(s['sections']):
        angles.append(torch.outer(s['positions'][:, axis].double(), s['inv_freq'][at:at + pairs]))
        at += pairs
    rotation = torch.polar(torch.ones((), dtype=torch.float64, device='cuda'), torch.cat(angles, 1))[:, None]
    outs, grads = [], []
    for name in 'qk':
        x = s[name].double()
        w = None if s[name + '_weight'] is None else s[name + '_weight'].double()
        if w is not None:
            inverse = 1 / torch.sqrt((x * x).sum(-1, keepdim=True) / HEAD_DIM + EPS)
            y = x * inverse * w
        else:
            y = x
        half = HEAD_DIM // 2
        pairs = y.unflatten(-1, (half, 2)) if s['interleaved'] else y.unflatten(-1, (2, half)).transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * rotation)
        outs.append((turned if s['interleaved'] else turned.transpose(-1, -2)).flatten(-2))
        if s['train']:
            d = s['d' + name].double()
            pairs = d.unflatten(-1, (half, 2)) if s['interleaved'] else d.unflatten(-1, (2, half)).transpose(-1, -2)
            back = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * rotation.conj())
            back = (back if s['interleaved'] else back.transpose(-1, -2)).flatten(-2)
            if w is None:
                grads.append(back)
            else:
                inner = (back * w * x).sum(-1, keepdim=True) / HEAD_DIM
                grads.append(inverse * back * w - inverse ** 3 * inner * x)
                grads.append((back * x * inverse).sum((0, 1)))
    return outs + grads


def _exact_norm(s):
    names = ('x', 'branch', 'weight', 'gate', 'scale', 'shift')
    t = {n: None if s[n] is None else s[n].double().requires_grad_(s['train']) for n in names}
    ys, rs, first = [], [], 0
    for i, n in enumerate(_lengths(s)):
        rows = slice(first, first + n)
        first += n
        r = t['x'][rows]
        if t['branch'] is not None:
            r = r + (t['branch'][rows] if t['gate'] is None else t['branch'][rows] * t['gate'][i])
        mean = r.mean(-1, keepdim=True) if s['center'] else 0.0
        y = (r - mean) / torch.sqrt(((r - mean) ** 2).mean(-1, keepdim=True) + EPS)
        if t['weight'] is not None:
            y = y * t['weight']
        if t['scale'] is not None:
            y = y * (1 + t['scale'][i]) + t['shift'][i]
        ys.append(y)
        rs.append(r)
    y, r = torch.cat(ys), torch.cat(rs)
    outs = [y.detach(), r.detach()]
    if s['train']:
        outs += torch.autograd.grad((y, r), [t[n] for n in names if t[n] is not None], (s['dy'].double(), s['dr'].double()))
    return outs
