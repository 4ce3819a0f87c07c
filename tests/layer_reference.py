"""Plain 64-bit forms of the operators around the projections, differentiable, for the tests."""
import math

import torch


def segments(cu, tokens):
    """(first row, end row) of every sequence of `cu` (a list of offsets, or None), and the covered rows."""
    if cu is None:
        return [(0, tokens)]
    return list(zip(cu[:-1], cu[1:]))


def attention(q, k, v, cu=None, causal=False, scale=None):
    """(o, log-sum-exp [heads, tokens]); rows of no sequence give 0 and -inf."""
    tokens, heads, dim = q.shape
    group = heads // k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    outs, lses, at = [], [], 0
    for a, b in segments(cu, tokens):
        kk, vv = (t[a:b].repeat_interleave(group, 1).transpose(0, 1) for t in (k, v))
        s = q[a:b].transpose(0, 1) @ kk.transpose(1, 2) * scale
        if causal:
            s = s.masked_fill(torch.ones(b - a, b - a, dtype=torch.bool, device=q.device).triu(1), -math.inf)
        outs.append((s.softmax(-1) @ vv).transpose(0, 1))
        lses.append(torch.logsumexp(s, -1))
        at = b
    outs.append(torch.zeros(tokens - at, heads, dim, dtype=q.dtype, device=q.device))
    lses.append(torch.full((heads, tokens - at), -math.inf, dtype=q.dtype, device=q.device))
    return torch.cat(outs), torch.cat(lses, 1)


def rotary(x, positions, inv_freq, sections, interleaved=True, weight=None, eps=1e-6):
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    angle = (positions.double()[:, axis] * inv_freq.double())[:, None]
    cos, sin = angle.cos(), angle.sin()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    c, d = a * cos - b * sin, b * cos + a * sin
    return torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1)


def residual_norm(x, branch=None, weight=None, gate=None, scale=None, shift=None, cu=None, eps=1e-6, center=False):
    tokens = x.shape[0]
    ys, rs, at = [], [], 0
    for i, (a, b) in enumerate(segments(cu, tokens)):
        r = x[a:b]
        if branch is not None:
            r = r + (branch[a:b] if gate is None else branch[a:b] * gate[i])
        c = r - r.mean(-1, keepdim=True) if center else r
        y = c / (c.square().mean(-1, keepdim=True) + eps).sqrt()
        if weight is not None:
            y = y * weight
        if scale is not None:
            y = y * (1 + scale[i])
        if shift is not None:
            y = y + shift[i]
        ys.append(y)
        rs.append(r)
        at = b
    rs.append(x[at:] if branch is None or gate is not None else x[at:] + branch[at:])
    return torch.cat(ys + [torch.zeros_like(x[at:])]), torch.cat(rs)
