"""Attention over packed sequences: refusals on the CPU, the kernels against the 64-bit form on the GPU.

Tolerances. Probabilities are rounded to BF16 for the product with V, each by at most 2^-8 of its value
relative to the row's sum (the sum itself is FP32 and unrounded), so o is off by at most 2^-8 of
sum_j p_j |v_j|, and once more by 2^-8 of its own value for the output. FP32 products, the exponential (2
ulp) and the scores (|s| times 2^-23 as an error of the exponent) come on top: 2^-14 of sum_j p_j |v_j|.
The backward pass rounds P and dS to BF16 in the same way, and reads o rounded: delta = sum(do * o) is off
by 2^-8 sum |do||o| (and o's own error above); the bounds below carry these through with absolute values.
"""
import math

import pytest
import torch

from tests import layer_reference as plain

HALF = 2.0 ** -8
FINE = 2.0 ** -14


def attention(*args, **kwargs):
    import fused_gemm_a2a
    return fused_gemm_a2a.packed_attention(*args, **kwargs)


def offsets(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


# ----------------------------------------------------------------------------------------- CPU
@pytest.mark.parametrize('device', [None, 'cuda', 'cuda:1', torch.device('cuda'), 1])
def test_check_status_reads_the_current_device_for_every_way_to_name_it(monkeypatch, device):
    import fused_gemm_a2a_kernels as kernels
    import fused_layer_ops
    monkeypatch.setattr(kernels, '_local_status', {torch.device('cuda', 1): torch.tensor([3, 70, 5, 0])})
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: 1)
    with pytest.raises(RuntimeError, match='device error 3'):
        fused_layer_ops.check_status(device)


@pytest.mark.parametrize('clear', [False, True])
def test_check_status_waits_for_all_streams(monkeypatch, clear):
    """An error that a kernel on any stream records before it ends is seen, and not erased unseen."""
    import fused_gemm_a2a_kernels as kernels
    import fused_layer_ops
    events = []

    class Word:
        is_cuda, device, code = True, torch.device('cuda', 0), 0

        def tolist(self):
            events.append('read')
            return [self.code, 70, 5, 0]

        def zero_(self):
            events.append('zero')

    def synchronize(device):
        events.append('synchronize')
        word.code = 3                    # what was running has given up meanwhile

    word = Word()
    monkeypatch.setattr(kernels, '_local_status', {word.device: word})
    monkeypatch.setattr(torch.cuda, 'synchronize', synchronize)
    with pytest.raises(RuntimeError, match='device error 3'):
        fused_layer_ops.check_status(word.device, clear=clear)
    assert events == ['synchronize', 'read'] + ['zero', 'synchronize'] * clear


def test_a_call_raises_an_error_that_the_host_has_got(monkeypatch):
    import fused_gemm_a2a_kernels as kernels
    import fused_layer_ops
    device = torch.device('cuda', 0)

    class Copy:
        address, words = 64, [3, 70, 5, 0]

    monkeypatch.setattr(kernels, '_local_host_status', {device: Copy()})
    monkeypatch.setattr(kernels, '_local_status', {device: torch.zeros(4, dtype=torch.int32)})
    with pytest.raises(RuntimeError, match='device error 3.*where=70, detail=5'):
        fused_layer_ops._host_status_address(device)
    fused_layer_ops.check_status(device)          # the device's word has been cleared: nothing to raise any more
    assert fused_layer_ops._host_status_address(device) == 64


def test_the_status_word_is_zero_before_another_thread_can_find_it(monkeypatch):
    """A second thread that found the word earlier could launch on its own stream, in front of the zeros."""
    import fused_gemm_a2a_kernels as kernels
    import fused_layer_ops
    device, found = torch.device('cuda', 0), []

    class Word:
        is_cuda = True

    class Stream:
        def synchronize(self):
            found.append(dict(kernels._local_status))

    class Nothing:
        def __init__(self, *_):
            pass
        __enter__ = __exit__ = lambda *_: None

    monkeypatch.setattr(kernels, '_local_status', {})
    monkeypatch.setattr(torch, 'zeros', lambda *a, **k: Word())
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda *_: Stream())
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    monkeypatch.setattr(torch.cuda, 'device', Nothing)
    word = fused_layer_ops._status(device)
    assert isinstance(word, Word) and found == [{}]        # waited for once, and not to be found meanwhile
    assert kernels._local_status == {device: word} and fused_layer_ops._status(device) is word and len(found) == 1


def test_refusals():
    bf = torch.bfloat16
    q, k = torch.zeros(6, 4, 128, dtype=bf), torch.zeros(6, 2, 128, dtype=bf)
    cu = torch.tensor([0, 2, 6], dtype=torch.int32)
    for message, change in (
            ('BF16', dict(q=q.float())), ('BF16', dict(q=q.half())), ('BF16', dict(k=k[..., :64])), ('BF16', dict(v=k[0])),
            ('head', dict(k=k[:, :0], v=k[:, :0])), ('one shape', dict(v=q)), ('tokens', dict(k=k[:5], v=k[:5])),
            ('multiple', dict(k=q[:, :3], v=q[:, :3])), ('scale', dict(scale=0.0)), ('scale', dict(scale=-1.0)),
            ('scale', dict(scale=math.inf)), ('scale', dict(scale=math.nan)), ('scale', dict(scale=1e-40)),
            ('strides', dict(q=torch.zeros(6, 4, 256, dtype=bf)[..., ::2])),
            ('strides', dict(v=torch.zeros(6, 1, 128, dtype=bf).expand(6, 2, 128))),
            ('strides', dict(q=torch.zeros(6 * 4 * 128 + 4, dtype=bf)[4:].view(6, 4, 128))),
            ('cu_seqlens', dict(cu_seqlens=cu.long())), ('cu_seqlens', dict(cu_seqlens=cu[:1])),
            ('cu_seqlens', dict(cu_seqlens=cu.view(3, 1))),
            ('65535', dict(cu_seqlens=torch.zeros(65537, dtype=torch.int32))), ('CUDA', {})):
        with pytest.raises(ValueError, match=message):
            attention(**(dict(q=q, k=k, v=k, cu_seqlens=cu) | change))


def test_the_c_entry_refuses_what_the_kernels_cannot_do(native):
    import ctypes

    import _fga_native as api
    args = api.FgaAttention(16, 16, 16, 16, 16, tokens=4, heads=4, kv_heads=2, samples=1, scale=0.1, status=16)
    for i in range(3):
        args.token_stride[i], args.head_stride[i] = 512, 128
    assert native.fga_attention_forward(None, None) == -1 and b'null' in native.fga_last_error()
    for field, value, message in (('tokens', 0, b'tokens'), ('tokens', 1 << 31, b'tokens'), ('kv_heads', 3, b'multiple'),
                                  ('kv_heads', 0, b'multiple'), ('samples', 0, b'sequences'), ('samples', 2, b'cu_seqlens'),
                                  ('scale', 0.0, b'scale'), ('scale', math.nan, b'scale'), ('q', 8, b'aligned'),
                                  ('v', None, b'null'), ('status', None, b'null')):
        broken = api.FgaAttention.from_buffer_copy(args)
        setattr(broken, field, value)
        assert native.fga_attention_forward(ctypes.byref(broken), None) == -1, field
        assert message in native.fga_last_error(), (field, native.fga_last_error())
    broken = api.FgaAttention.from_buffer_copy(args)
    broken.head_stride[1] = 130
    assert native.fga_attention_forward(ctypes.byref(broken), None) == -1 and b'strides' in native.fga_last_error()


def test_barriers_without_a_limit_stand_in_front_of_every_wait_that_may_give_up():
    """A warp that gives up on a bounded wait leaves for the end of its block. Another warp of its role that
    then met it at a named barrier, which has no limit, would wait for good."""
    import os
    import re
    import build_native
    source = open(os.path.join(build_native.CSRC, 'attention_sm100a.cu')).read()
    found = 0
    for kernel in source.split('__global__')[1:]:
        for role in re.split(r'// -{20,}', kernel):
            for barrier in re.finditer(r'\bbar(rier)?\.(cta\.)?(sync|red)\b', role):
                found += 1
                assert 'wait' not in re.sub(r'(tmem_ld|tmem_st|bulk)_wait', '', role[:barrier.start()]), role[:80].strip()
    assert found


def test_gradient_of_the_plain_form_against_differences():
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(5, h, 8, generator=g, dtype=torch.float64).requires_grad_() for h in (4, 2, 2))
    for causal in (False, True):
        assert torch.autograd.gradcheck(lambda *t: plain.attention(*t, [0, 3, 3, 4], causal)[0], (q, k, v))


# ----------------------------------------------------------------------------------------- GPU
def normal(gen, *shape, std=1.0):
    return (torch.randn(*shape, generator=gen, device='cuda') * std).bfloat16()


def within(got, want, bound, label):
    got = got.double()
    assert got.shape == want.shape, label
    assert torch.isfinite(got).all(), f'{label}: not finite'
    excess = (got - want).abs() - bound
    assert bool((excess <= 0).all()), f'{label}: over its bound by {excess.max().item():.3g} of {want.abs().max().item():.3g}'


def expected(q, k, v, cu, causal, scale=None, do=None):
    """o, lse and the gradients in 64 bits with the bounds of the kernels' errors."""
    tokens, heads, dim = q.shape
    group = heads // k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    zeros = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=t.device)        # noqa: E731
    o, eo, lse = zeros(q), zeros(q), torch.full((heads, tokens), -math.inf, dtype=torch.float64, device=q.device)
    grads = {n: (zeros(t), zeros(t)) for n, t in (('q', q), ('k', k), ('v', v))}
    for a, b in plain.segments(cu, tokens):
        if a == b:
            continue
        mask = torch.ones(b - a, b - a, dtype=torch.bool, device=q.device).triu(1) if causal else None
        for h in range(heads):
            g = h // group
            qq, kk, vv = q[a:b, h].double(), k[a:b, g].double(), v[a:b, g].double()
            s = qq @ kk.T * scale
            if causal:
                s = s.masked_fill(mask, -math.inf)
            top = s.abs().masked_fill(s.isinf(), 0).amax()
            fine = FINE + top.item() * 2.0 ** -21
            p = s.softmax(-1)
            lse[h, a:b] = torch.logsumexp(s, -1)
            out = p @ vv
            reach = p @ vv.abs()
            o[a:b, h], eo[a:b, h] = out, (HALF * (1 + HALF) + fine) * reach + HALF * out.abs()
            if do is None:
                continue
            d = do[a:b, h].double()
            dp = d @ vv.T
            delta = (d * out).sum(-1, keepdim=True)
            edelta = (d.abs() * eo[a:b, h]).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            # dS: its own rounding, the exponential's and the products' error, and delta's
            eds = HALF * (1 + HALF) * ds.abs() + p * ((1 + HALF) * edelta + fine * (dp.abs() + delta.abs() + d.abs() @ vv.abs().T))
            for n, value, error in (('q', ds @ kk * scale, eds @ kk.abs() * scale),
                                    ('k', ds.T @ qq * scale, eds.T @ qq.abs() * scale),
                                    ('v', p.T @ d, (HALF + fine) * (p.T @ d.abs()))):
                hh = h if n == 'q' else g
                grads[n][0][a:b, hh] += value
                grads[n][1][a:b, hh] += error * (1 + 2 * HALF) + fine * 2.0 ** -6 * value.abs()
    for n in grads:
        grads[n][1].add_(HALF * grads[n][0].abs())
    return o, eo, lse, grads


SHAPES = [
    ([1], 0, 1, 1), ([1, 5, 17], 0, 8, 8), ([127], 0, 2, 1), ([128], 0, 2, 2), ([129], 0, 3, 1), ([255, 1], 0, 4, 2),
    ([256], 5, 2, 1), ([257, 0, 0, 383], 130, 6, 3), ([0], 7, 2, 2), ([0, 3], 0, 1, 1), ([1000], 0, 5, 5),
    ([700, 64, 65, 1, 640], 3, 4, 1), ([2049], 0, 2, 2),
    # one, two and four blocks that share a key/value tile, with and without a mask
    ([1500, 549], 0, 32, 16), ([2100], 0, 40, 40), ([1500, 549], 0, 32, 4), ([2100], 0, 64, 16), ([130], 0, 32, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize('lengths,pad,heads,kv_heads', SHAPES)
@pytest.mark.parametrize('causal', [False, True])
def test_forward_matches_the_plain_form(native, lengths, pad, heads, kv_heads, causal):
    gen = torch.Generator(device='cuda').manual_seed(sum(lengths) + heads)
    tokens, cu = sum(lengths) + pad, offsets(lengths)
    q, k, v = normal(gen, tokens, heads, 128, std=1.5), normal(gen, tokens, kv_heads, 128), normal(gen, tokens, kv_heads, 128)
    o, eo, lse, _ = expected(q, k, v, cu, causal)
    if pad:                              # what padding rows hold must not matter
        for t in (q, k, v):
            t[-pad:] = float('nan')
    got, got_lse = attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device='cuda'), causal=causal, return_lse=True)
    within(got, o, eo + 1e-30, 'o')
    live = cu[-1]
    assert torch.isneginf(got_lse[:, live:]).all()
    within(got_lse[:, :live], lse[:, :live], 1e-5 * (1 + lse[:, :live].abs()), 'lse')
    if pad:
        assert got[live:].abs().max() == 0


@pytest.mark.gpu
@pytest.mark.parametrize('lengths,pad,heads,kv_heads', SHAPES)
@pytest.mark.parametrize('causal', [False, True])
def test_gradients_match_the_plain_form(native, lengths, pad, heads, kv_heads, causal):
    gen = torch.Generator(device='cuda').manual_seed(sum(lengths) + heads)
    tokens, cu = sum(lengths) + pad, offsets(lengths)
    q, k, v = normal(gen, tokens, heads, 128, std=1.5), normal(gen, tokens, kv_heads, 128), normal(gen, tokens, kv_heads, 128)
    do = normal(gen, tokens, heads, 128)
    _, _, _, grads = expected(q, k, v, cu, causal, do=do)
    if pad:
        for t in (q, k, v, do):
            t[-pad:] = float('nan')
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = attention(*leaves, torch.tensor(cu, dtype=torch.int32, device='cuda'), causal=causal)
    for name, got in zip('qkv', torch.autograd.grad(o, leaves, do)):
        within(got, grads[name][0], grads[name][1] + 1e-30, 'd' + name)
        if pad:
            assert got[cu[-1]:].abs().max() == 0


@pytest.mark.gpu
@pytest.mark.parametrize('tokens,heads,kv_heads', [(4200, 1, 1), (4200, 2, 1), (2500, 3, 1)])
def test_blocks_of_a_cluster_without_a_query(native, tokens, heads, kv_heads):
    """Four blocks share a key/value tile; the last tiles of a causal sequence have fewer query tiles than that."""
    gen = torch.Generator(device='cuda').manual_seed(tokens + heads)
    q, k, v = normal(gen, tokens, heads, 128, std=1.5), normal(gen, tokens, kv_heads, 128), normal(gen, tokens, kv_heads, 128)
    do = normal(gen, tokens, heads, 128)
    o, eo, _, grads = expected(q, k, v, None, True, do=do)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    got = attention(*leaves, causal=True)
    within(got.detach(), o, eo + 1e-30, 'o')
    for name, g in zip('qkv', torch.autograd.grad(got, leaves, do)):
        within(g, grads[name][0], grads[name][1] + 1e-30, 'd' + name)


def expected_in_pieces(q, k, v, do, causal, rows=2048):
    """o and the gradients of one sequence and one key/value head in 64 bits, some queries at a time."""
    tokens, heads, dim = q.shape
    kk, vv = k[:, 0].double(), v[:, 0].double()
    o, dq = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    dk, dv = torch.zeros_like(kk), torch.zeros_like(vv)
    at = torch.arange(tokens, device=q.device)
    for h in range(heads):
        for a in range(0, tokens, rows):
            qq, d = q[a:a + rows, h].double(), do[a:a + rows, h].double()
            p = qq @ kk.T * dim ** -0.5
            if causal:
                p.masked_fill_(at > at[a:a + rows, None], -math.inf)
            p = p.softmax(-1)
            o[a:a + rows, h] = p @ vv
            dv += p.T @ d
            p *= d @ vv.T - (d * o[a:a + rows, h]).sum(-1, keepdim=True)
            dq[a:a + rows, h] = p @ kk * dim ** -0.5
            dk += p.T @ qq * dim ** -0.5
    return o, dq, dk[:, None], dv[:, None]


@pytest.mark.gpu
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('tokens', [16383, 131072])
def test_long_sequences(native, tokens, causal):
    """Thousands of keys make every element a small sum of many terms, to which the bounds above (the sum of the terms'
    sizes) say little. The terms' roundings are independent and the sum grows with their root as they do, so the error
    of any 128 rows is the chain of four roundings beside their norm; a missing key tile would be 3 % at 131072."""
    gen = torch.Generator(device='cuda').manual_seed(tokens)
    q, k, v, do = (normal(gen, tokens, h, 128) for h in (2, 1, 1, 2))
    want = expected_in_pieces(q, k, v, do, causal)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = attention(*leaves, causal=causal)
    for name, a, b in zip(('o', 'dq', 'dk', 'dv'), (o.detach(), *torch.autograd.grad(o, leaves, do)), want):
        for first in range(0, tokens, 128):
            error = (a[first:first + 128].double() - b[first:first + 128]).norm() / b[first:first + 128].norm()
            assert error <= 4 * HALF, (name, first, error.item())


@pytest.mark.gpu
@pytest.mark.parametrize('scale,std', [(1.0, 0.5), (0.02, 4.0), (0.3, 3.0)])
def test_other_scales_and_peaked_rows(native, scale, std):
    """Scores that reach the hundreds: the running maximum moves, and most probabilities vanish."""
    gen = torch.Generator(device='cuda').manual_seed(7)
    q, k, v, do = (normal(gen, 900, h, 128, std=s) for h, s in ((4, std), (2, std), (2, 1.0), (4, 1.0)))
    ramp = torch.linspace(0.1, 3.0, 900, device='cuda')[:, None, None]       # later keys weigh more: maxima keep rising
    k = (k.float() * ramp).bfloat16()
    o, eo, lse, grads = expected(q, k, v, None, False, scale, do)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    got, got_lse = attention(*leaves, scale=scale, return_lse=True)
    within(got.detach(), o, eo + 1e-30, 'o')
    within(got_lse, lse, 1e-5 * (1 + lse.abs()), 'lse')
    for name, g in zip('qkv', torch.autograd.grad(got, leaves, do)):
        within(g, grads[name][0], grads[name][1] + 1e-30, 'd' + name)


@pytest.mark.gpu
@pytest.mark.parametrize('causal', [False, True])
def test_scores_at_and_beyond_the_end_of_their_range(native, causal):
    """Where scores are so far apart that a row is its largest key's value, and where FP32 cannot hold them."""
    gen = torch.Generator(device='cuda').manual_seed(17)
    q, k, v, do = (normal(gen, 400, 1, 128) for _ in range(4))
    products = q[:, 0].double() @ k[:, 0].double().T
    if causal:
        products = products.masked_fill(torch.ones(400, 400, dtype=torch.bool, device='cuda').triu(1), -math.inf)
    top, best = products.max(-1)
    # FP32 sums of 128 products are off by 128 * 2^-24 of their absolute sum: rows whose second key is closer are left out
    second = products.scatter(1, best[:, None], -math.inf).max(-1).values
    clear = top - second > 128 * 2.0 ** -24 * (q.double().abs() @ k.double().abs().transpose(1, 2)).max() + 1e-3
    assert clear.sum() > 300
    # The one probability p is a power of two that the rounded shift leaves, rounded to BF16, and the sum it is divided
    # by is p unrounded: o = v (1 + 2^-8)(1 + 2^-8) at most, output rounding included; FP32 steps take 2^-20.
    want = v[best].double()
    bound = (2 * HALF + HALF ** 2 + 2.0 ** -20) * want.abs()
    for scale in (1e5, 5e6):                                   # up to 2^28
        scores = top.abs() * scale
        assert scores.max() < 2 ** 28 * 1.5
        o, lse = attention(q, k, v, causal=causal, scale=scale, return_lse=True)
        within(o[clear], want[clear], bound[clear], f'o at scale {scale}')
        within(lse[0], top * scale, (128 * 2.0 ** -24 + 2.0 ** -20) * scale * 128 * 8 + 10, 'lse')
    scale = 1e8
    beyond = (top.abs() * scale > 2 ** 29.1) & clear           # in units of log2 well above 2^29
    within_range = (top.abs() * scale < 2 ** 28) & clear
    assert beyond.sum() > 300
    o, lse = attention(q, k, v, causal=causal, scale=scale, return_lse=True)
    assert o[beyond].isnan().all() and lse[0, beyond].isnan().all()
    within(o[within_range], want[within_range], bound[within_range], 'o beside rows out of range')
    # gradients: NaN from a largest score of 2^20 on, in every row that such a query reaches
    leaves = [t.requires_grad_() for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(attention(*leaves, causal=causal, scale=1e6), leaves, do)
    far = top.abs() * 1e6 > 2 ** 20.1
    assert far.sum() > 300 and dq[far].isnan().all() and dv[0].isnan().all() and dk[0].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize('pad_is_a_sequence', [False, True])
def test_rows_behind_a_sequence_do_not_change_a_bit_of_it(native, pad_is_a_sequence):
    """The last tile of queries holds rows of padding, or of the next sequence, whose maxima rise from key tile to
    key tile or do not."""
    gen = torch.Generator(device='cuda').manual_seed(18)
    n, pad = 300, 200
    q, k, v, do = (normal(gen, n + pad, 2, 128) for _ in range(4))
    cu = torch.tensor([0, n, n + pad] if pad_is_a_sequence else [0, n], dtype=torch.int32, device='cuda')
    results = []
    for behind in (0.0, k[200:201].float() * 30):
        q[n:] = behind
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        o, lse = attention(*leaves, cu, return_lse=True)
        results.append([o.detach()[:n], lse[:, :n], *(g[:n] for g in torch.autograd.grad(o, leaves, do))])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_strided_heads_and_expanded_gradients(native):
    gen = torch.Generator(device='cuda').manual_seed(8)
    packed = normal(gen, 300, 8, 128)
    q, k = packed[:, 2:6], packed[:, 6:]
    v = normal(gen, 2, 300, 128).transpose(0, 1)
    views = [t.detach().requires_grad_() for t in (q, k, v)]
    whole = [t.detach().contiguous().requires_grad_() for t in (q, k, v)]
    outs = [attention(*t, causal=True) for t in (views, whole)]
    assert torch.equal(*outs)
    grads = [torch.autograd.grad(o.float().sum(), t) for o, t in zip(outs, (views, whole))]
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.gpu
def test_the_same_bits_on_side_streams_and_in_a_graph(native):
    gen = torch.Generator(device='cuda').manual_seed(9)
    cu = torch.tensor([0, 700, 701, 1500], dtype=torch.int32, device='cuda')
    q, k, v, do = (normal(gen, 1500, h, 128) for h in (8, 2, 2, 8))
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def step():
        o = attention(*leaves, cu, causal=True)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    first = step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            results.append(step())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        captured = step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for other in (*results, captured):
        assert all(torch.equal(a, b) for a, b in zip(first, other))
    with torch.no_grad():
        q.normal_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, step()))


@pytest.mark.gpu
def test_no_tokens(native):
    q = torch.zeros(0, 4, 128, dtype=torch.bfloat16, device='cuda', requires_grad=True)
    o = attention(q, q, q)
    assert o.shape == q.shape
    assert torch.autograd.grad(o.sum(), q)[0].shape == q.shape


@pytest.mark.gpu
@pytest.mark.parametrize('causal', [False, True])
def test_thousands_of_short_sequences(native, causal):
    gen = torch.Generator(device='cuda').manual_seed(10)
    count, n, heads = 5000, 3, 2
    q, k, v, do = (normal(gen, count * n, h, 128) for h in (heads, 1, 1, heads))
    cu = torch.arange(0, count * n + 1, n, dtype=torch.int32, device='cuda')
    leaves = [t.requires_grad_() for t in (q, k, v)]
    got = attention(*leaves, cu, causal=causal)
    flat = [t.detach().double().requires_grad_() for t in leaves]
    qq, kk, vv = (t.view(count, n, -1, 128).transpose(1, 2) for t in flat)
    s = qq @ kk.transpose(2, 3) * 128 ** -0.5
    if causal:
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device='cuda').triu(1), -math.inf)
    p = s.softmax(-1)
    o = (p @ vv).transpose(1, 2).reshape(count * n, heads, 128)
    # rounding of P (2^-8 of sum p|v|) and of the output, and the gradients' chain of four such roundings
    reach = (p @ vv.abs()).transpose(1, 2).reshape(o.shape)
    within(got.detach(), o.detach(), (2 * HALF * reach + HALF * o.abs() + 1e-6).detach(), 'o')
    for a, b in zip(torch.autograd.grad(got, leaves, do), torch.autograd.grad(o, flat, do.double())):
        error = (a.double() - b).norm() / b.norm()
        assert error <= 4 * HALF, error


@pytest.mark.gpu
def test_more_than_2_to_31_elements(native):
    """Offsets that do not fit 32 bits: the last sequence comes out like the same sequence alone."""
    tokens, heads, n = 540_000, 32, 1000             # 2.2e9 query elements
    gen = torch.Generator(device='cuda').manual_seed(12)
    q = torch.ones(tokens, heads, 128, dtype=torch.bfloat16, device='cuda')
    q[-n:] = normal(gen, n, heads, 128)
    k, v = normal(gen, tokens, 1, 128), normal(gen, tokens, 1, 128)
    cu = torch.arange(0, tokens + 1, n, dtype=torch.int32, device='cuda')
    leaves = [t.requires_grad_() for t in (q, k, v)]
    whole = attention(*leaves, cu, causal=True)
    grads = torch.autograd.grad(whole, leaves, q.detach())
    part = [t[-n:].detach().clone().requires_grad_() for t in leaves]
    alone = attention(*part, causal=True)
    assert torch.equal(whole[-n:], alone)
    for a, b in zip(grads, torch.autograd.grad(alone, part, q.detach()[-n:])):
        # one block or two share a key/value tile, so its sums may be taken in another order
        assert (a[-n:].double() - b.double()).norm() <= 2 * HALF * b.double().norm()


@pytest.mark.gpu
def test_a_recorded_device_error_is_sticky_and_raises(native):
    import fused_gemm_a2a
    import fused_gemm_a2a_kernels as kernels
    q = torch.ones(4, 1, 128, dtype=torch.bfloat16, device='cuda')
    attention(q, q, q)
    fused_gemm_a2a.check_status()
    word = kernels._local_status[q.device]
    word[0] = 3
    attention(q, q, q)                   # returns at once and computes nothing
    with pytest.raises(RuntimeError, match='pipeline barrier'):
        fused_gemm_a2a.check_status(clear=True)
    fused_gemm_a2a.check_status()
    assert torch.equal(attention(q, q, q), q)


@pytest.mark.gpu
@pytest.mark.parametrize('call', ['forward', 'backward', 'graph'])
def test_an_error_reaches_the_next_call_without_a_synchronizing_one(native, call):
    import fused_gemm_a2a
    import fused_gemm_a2a_kernels as kernels
    q = torch.ones(4, 1, 128, dtype=torch.bfloat16, device='cuda', requires_grad=True)
    o = attention(q, q, q)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        attention(q, q, q)
    fused_gemm_a2a.check_status()
    word = kernels._local_status[q.device]
    word.copy_(torch.tensor([3, 70, 5, 0], dtype=torch.int32))
    try:
        if call == 'graph':
            graph.replay()
        elif call == 'backward':
            torch.autograd.grad(o, q, o.detach(), retain_graph=True)
        else:
            attention(q.detach(), q.detach(), q.detach())
        torch.cuda.current_stream().synchronize()      # the kernel has run; nobody has read the word
        for _ in range(2):
            with pytest.raises(RuntimeError, match='pipeline barrier.*where=70, detail=5'):
                attention(q, q, q)
        with pytest.raises(RuntimeError, match='pipeline barrier.*where=70, detail=5'):
            torch.autograd.grad(o, q, o.detach(), retain_graph=True)
    finally:
        with pytest.raises(RuntimeError, match='pipeline barrier'):
            fused_gemm_a2a.check_status(clear=True)
    assert torch.equal(attention(q, q, q), q)
    fused_gemm_a2a.check_status()


@pytest.mark.gpu
def test_a_capture_that_is_the_first_to_ask_for_the_hosts_copy(native):
    """The device's word may be there without it, made by another operator; pinned memory cannot be had in a capture."""
    import fused_gemm_a2a_kernels as kernels
    q = torch.ones(4, 1, 128, dtype=torch.bfloat16, device='cuda')
    attention(q, q, q)
    copy = kernels._local_host_status.pop(q.device)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = attention(q, q, q)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, q) and not kernels._local_host_status
    finally:
        kernels._local_host_status[q.device] = copy


@pytest.mark.gpu
def test_two_threads_at_once(native):
    """Forward and backward of two sizes, each thread on its own stream: the same bits as alone."""
    import threading
    gen = torch.Generator(device='cuda').manual_seed(20)
    sizes = ((700, 4, 2), (130, 8, 1))
    inputs = [[normal(gen, n, h, 128) for h in (heads, kv, kv, heads)] for n, heads, kv in sizes]

    def step(q, k, v, do):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        o = attention(*leaves, causal=True)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    want, failures, start = [step(*t) for t in inputs], [], threading.Barrier(2)
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(50):
                    got = step(*inputs[i])
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
        except Exception as error:                                                  # noqa: BLE001
            failures.append(repr(error))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failures, failures


@pytest.mark.gpu
def test_check_status_sees_an_error_behind_work_of_another_stream(native):
    import fused_gemm_a2a
    import fused_gemm_a2a_kernels as kernels
    q = torch.ones(4, 1, 128, dtype=torch.bfloat16, device='cuda')
    attention(q, q, q)
    word, code = kernels._local_status[q.device], torch.tensor([3, 0, 0, 0], dtype=torch.int32, device='cuda')
    a, b = (torch.zeros(1 << 28, dtype=torch.uint8, device='cuda') for _ in range(2))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(300):             # tens of milliseconds
            a.copy_(b, non_blocking=True)
        word.copy_(code, non_blocking=True)
    try:
        with pytest.raises(RuntimeError, match='pipeline barrier'):
            fused_gemm_a2a.check_status(clear=True)
    finally:
        side.synchronize()
        word.zero_()
        torch.cuda.synchronize()
    fused_gemm_a2a.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize('lengths,causal', [([1] * 40, False), ([1, 2, 3] * 20, True), ([1] + [128] * 3, True)])
def test_rows_that_see_one_key_have_no_score_gradient(native, lengths, causal):
    """A row with a single key has P = 1 and dS = 0 whatever its output rounds to: dq = 0, dk only from others."""
    gen = torch.Generator(device='cuda').manual_seed(13)
    cu = offsets(lengths)
    q, k, v, do = (normal(gen, cu[-1], h, 128) for h in (4, 2, 2, 4))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = attention(*leaves, torch.tensor(cu, dtype=torch.int32, device='cuda'), causal=causal)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    for a, b in plain.segments(cu, cu[-1]):
        alone = slice(a, b if b - a == 1 else a + 1 if causal else a)
        # FP32: the product of 128 terms and the exponential of a score minus its own logarithm
        assert (dq[alone].abs() <= 128 * 2.0 ** -20 * 40).all()
        if b - a == 1:
            assert (dk[a:b].abs() <= 2 * 128 * 2.0 ** -20 * 40).all()
            want = do[a:b].double().view(1, 2, 2, 128).sum(2)
            within(dv[a:b], want, HALF * want.abs() + 1e-5, 'dv')


@pytest.mark.gpu
def test_gradients_of_some_inputs_only(native):
    gen = torch.Generator(device='cuda').manual_seed(14)
    q, k, v, do = (normal(gen, 200, h, 128) for h in (4, 2, 2, 4))
    full = [t.detach().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(attention(*full), full, do)
    for i in range(3):
        some = [t.detach().requires_grad_(n == i) for n, t in enumerate((q, k, v))]
        assert torch.equal(torch.autograd.grad(attention(*some), some[i], do)[0], want[i])
    o, lse = attention(*full, return_lse=True)
    assert not lse.requires_grad
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(o, full, do), want))
