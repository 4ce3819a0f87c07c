"""One attention layer of a context-parallel trainer from the package's operators alone: norm, fused QKV
projection, rotary positions with head norm, attention over packed sequences, fused output projection, and
the residual sum with the next norm. Forward and backward against FP32 torch with BF16 roundings at the same
places; eager and captured into a CUDA graph.

Tolerance. Between input and output lie seven BF16 roundings, each off by at most 2^-8 of its value and
2^-8 / sqrt(3) of it root mean square, and the backward pass adds as many; their independent sum is
sqrt(14) 2^-8 / sqrt(3) = 0.85 % RMS. The bounds are twice that, rounded up to the ones of
tests/drivers/two_layer_training.py: 2 % relative RMS and 2 % of (peak + value) for every element.
"""
import pytest
import torch

from tests import layer_reference as plain
from tests.drivers.two_layer_training import deviation

HIDDEN, HEADS, LENGTHS = 1024, 8, (301, 1, 0, 150, 60)
SECTIONS = (16, 24, 24)


def parameters(kv_heads, gen):
    def weight(rows):
        return (torch.randn(rows, HIDDEN, generator=gen, device='cuda') * HIDDEN ** -0.5).bfloat16()

    def gain(n):
        return (1 + 0.1 * torch.randn(n, generator=gen, device='cuda')).bfloat16()

    p = dict(qkv=weight(HIDDEN + 2 * kv_heads * 128), out=weight(HIDDEN), norm1=gain(HIDDEN), norm2=gain(HIDDEN),
             q_norm=gain(128), k_norm=gain(128))
    return {n: t.requires_grad_() for n, t in p.items()}


def reference_layer(x, p, positions, freq, cu, kv_heads, causal):
    """The same in FP32, rounded where the operators round."""
    class Round(torch.autograd.Function):
        @staticmethod
        def forward(ctx, t):
            return t.bfloat16().float()

        @staticmethod
        def backward(ctx, g):
            return g.bfloat16().float()

    rnd = Round.apply
    group = HEADS // kv_heads
    y, _ = plain.residual_norm(x, weight=p['norm1'])
    y = rnd(y)
    rows = rnd(y @ p['qkv'].T).view(-1, kv_heads, group + 2, 128)
    q, k, v = rows[:, :, :group].flatten(1, 2), rows[:, :, group], rows[:, :, group + 1]
    q = rnd(plain.rotary(q, positions, freq, SECTIONS, True, p['q_norm']).float())
    k = rnd(plain.rotary(k, positions, freq, SECTIONS, True, p['k_norm']).float())
    o = rnd(plain.attention(q, k, v, cu, causal)[0])
    branch = rnd(o.flatten(1) @ p['out'].T)
    y, r = plain.residual_norm(x, branch, p['norm2'])
    return rnd(y), rnd(r)


@pytest.mark.gpu
@pytest.mark.parametrize('kv_heads,causal', [(8, False), (8, True), (2, True)])
def test_layer_forward_and_backward(cp1, kv_heads, causal):
    from fused_gemm_a2a import (FusedGemmA2AWorkspace, FusedOutputProjection, FusedQKVProjection, packed_attention,
                                residual_norm, rotary_embedding)
    gen = torch.Generator(device='cuda').manual_seed(11)
    tokens = sum(LENGTHS)
    cu = [0]
    for n in LENGTHS:
        cu.append(cu[-1] + n)
    offsets = torch.tensor(cu, dtype=torch.int32, device='cuda')
    p = parameters(kv_heads, gen)
    x = torch.randn(tokens, HIDDEN, generator=gen, device='cuda').bfloat16().requires_grad_()
    dy, dr = (torch.randn(tokens, HIDDEN, generator=gen, device='cuda').bfloat16() for _ in range(2))
    positions = torch.randint(0, 500, (tokens, 3), generator=gen, device='cuda')
    freq = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64, device='cuda') / n) for n in SECTIONS])
    grouped = {} if kv_heads == HEADS else dict(num_kv_heads=kv_heads)
    workspace = FusedGemmA2AWorkspace(HIDDEN, HEADS, 512, **grouped)
    qkv = FusedQKVProjection(HIDDEN, HEADS, weight=p['qkv'], **grouped)
    proj = FusedOutputProjection(HIDDEN, HEADS, weight=p['out'])
    leaves = [x, *p.values()]

    def step():
        y, _ = residual_norm(x, weight=p['norm1'])
        q, k, v = qkv(y, workspace)
        q, k = rotary_embedding(q, k, positions, freq, SECTIONS, q_weight=p['q_norm'], k_weight=p['k_norm'])
        o = packed_attention(q, k, v, offsets, causal=causal)
        y, r = residual_norm(x, proj(o, workspace), weight=p['norm2'])
        return [y.detach(), r.detach(), *torch.autograd.grad((y, r), leaves, (dy, dr))]

    def expected():
        flat = [t.detach().float().requires_grad_() for t in leaves]
        outs = reference_layer(flat[0], dict(zip(p, flat[1:])), positions, freq, cu, kv_heads, causal)
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, flat, (dy.float(), dr.float())))

    names = ['y', 'r', 'dx', *('d' + n for n in p)]

    def check(got, stage):
        for name, a, b in zip(names, got, expected()):
            peak, rms, fine = deviation(a, b)
            assert fine, f'{stage}: {name}: max error over peak {peak:.3g}, relative RMS {rms:.3g}'

    previous = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        check(step(), 'eager')
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = step()
        with torch.no_grad():
            x.normal_()
            dy.normal_()
        graph.replay()
        torch.cuda.synchronize()
        check(captured, 'graph')
        workspace.comm.check_status()
    finally:
        torch.backends.cuda.matmul.allow_tf32 = previous
