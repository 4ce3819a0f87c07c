"""Rotary positions and the norm around a block: refusals and formulas on the CPU, the kernels against
the 64-bit forms on the GPU.

Tolerances. A BF16 output is off by at most half a step, 2^-8 of its value; FP32 arithmetic in front of it
by a few 2^-24 of the terms it is made of, for which 2^-20 of the largest term is allowed (sixteen
roundings). The backward pass of an RMS norm without a gate reads the residual sum as the forward stored it, each
element off by 2^-8 of its value; what that does to each gradient is carried through with absolute values below.
Other norms compute the sum again and stay within these bounds by far; theirs without that rounding are tested apart.
"""
import pytest
import torch

from tests import layer_reference as plain

HALF = 2.0 ** -8          # half a BF16 step, relative
FINE = 2.0 ** -20
VIDEO = (16, 24, 24)


def frequencies(sections, dtype=torch.float64):
    return torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)) for n in sections]).to(dtype)


def within(got, want, bound, label):
    got = got.double()
    assert got.shape == want.shape, label
    assert torch.isfinite(got).all(), f'{label}: not finite'
    excess = (got - want).abs() - bound
    assert bool((excess <= 0).all()), f'{label}: over its bound by {excess.max().item():.3g}'


# ----------------------------------------------------------------------------------------- CPU
def ops():
    import fused_gemm_a2a
    return fused_gemm_a2a.rotary_embedding, fused_gemm_a2a.residual_norm


def test_refusals_of_the_rotary_call():
    rotary, _ = ops()
    bf = torch.bfloat16
    q, k = torch.zeros(5, 4, 128, dtype=bf), torch.zeros(5, 2, 128, dtype=bf)
    pos, freq = torch.zeros(5, 1, dtype=torch.int32), frequencies((64,))
    bad = [
        ('BF16', dict(q=q.float())), ('BF16', dict(q=q[..., :64])), ('head', dict(k=k[:, :0])),
        ('tokens', dict(k=k[:4])), ('strides', dict(q=torch.zeros(5, 4, 256, dtype=bf)[..., ::2])),
        ('strides', dict(q=torch.zeros(5, 1, 128, dtype=bf).expand(5, 4, 128))),
        ('strides', dict(q=torch.zeros(5 * 4 * 128 + 1, dtype=bf)[1:].view(5, 4, 128))),
        ('positions', dict(positions=pos.float())), ('positions', dict(positions=pos[:4])),
        ('positions', dict(sections=VIDEO)), ('sections', dict(sections=(16, 24, 23))),
        ('sections', dict(sections=(65, -1))), ('sections', dict(sections=(16, 16, 16, 8, 8))),
        ('inv_freq', dict(inv_freq=freq[:32])), ('inv_freq', dict(inv_freq=freq.half())),
        ('q_weight', dict(q_weight=torch.ones(64, dtype=bf))), ('k_weight', dict(k_weight=torch.ones(128))),
        ('eps', dict(eps=-1e-6)), ('CUDA', {}),
    ]
    for message, change in bad:
        args = dict(q=q, k=k, positions=pos, inv_freq=freq) | change
        with pytest.raises(ValueError, match=message):
            rotary(**args)


def test_refusals_of_the_norm_call():
    _, norm = ops()
    bf = torch.bfloat16
    x, w, rows = torch.zeros(6, 64, dtype=bf), torch.ones(64, dtype=bf), torch.zeros(2, 64, dtype=bf)
    cu = torch.tensor([0, 2, 6], dtype=torch.int32)
    bad = [
        ('x must', dict(x=x.float())), ('x must', dict(x=x[:, ::2])), ('x must', dict(x=x[0])),
        ('hidden', dict(x=x[:, :60].contiguous())), ('hidden', dict(x=torch.zeros(1, 8200, dtype=bf))),
        ('branch', dict(branch=x[:5])), ('branch', dict(branch=x.float())),
        ('pass one', dict(gate=rows, cu_seqlens=cu)), ('weight', dict(weight=w[:32])), ('weight', dict(weight=w.float())),
        ('scale', dict(scale=rows)), ('shift', dict(shift=rows[:1], cu_seqlens=cu)),
        ('gate', dict(branch=x, gate=rows.float(), cu_seqlens=cu)),
        ('cu_seqlens', dict(cu_seqlens=cu.long())), ('cu_seqlens', dict(cu_seqlens=cu[:1])),
        ('65535', dict(cu_seqlens=torch.zeros(65537, dtype=torch.int32))),
        ('eps', dict(eps=float('nan'))), ('CUDA', dict(weight=w)),
    ]
    for message, change in bad:
        with pytest.raises(ValueError, match=message):
            norm(**(dict(x=x) | change))


@pytest.fixture
def calls_without_kernels(monkeypatch):
    """The three public calls on CPU tensors, with what launches the kernels replaced by something of the right shape."""
    import fused_layer_ops as module
    monkeypatch.setattr(module, '_same_device', lambda *_: None)
    monkeypatch.setattr(module, '_attend', lambda q, k, v, cu, causal, scale, keep: (q.clone(), q[:, :, 0].T.float()))
    monkeypatch.setattr(module, '_rotate', lambda q, k, *_: (q.clone(), k.clone()))
    monkeypatch.setattr(module, '_normalise', lambda x, branch, *_: (x.clone(), x.clone()))
    heads, rows = torch.ones(4, 2, 128, dtype=torch.bfloat16), torch.ones(4, 256, dtype=torch.bfloat16)
    pos, freq = torch.arange(4), frequencies((64,))
    return [(lambda t: module.packed_attention(t, heads, heads), heads),
            (lambda t: module.rotary_embedding(t, heads, pos, freq)[0], heads),
            (lambda t: module.residual_norm(rows, t)[0], rows)]


@pytest.mark.parametrize('which', [0, 1, 2])
def test_derivatives_that_do_not_exist_are_refused_not_dropped(calls_without_kernels, which):
    call, t = calls_without_kernels[which]
    with torch.autograd.forward_ad.dual_level():
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match='jvp'):
                call(torch.autograd.forward_ad.make_dual(t, t))
    for transform in (lambda: torch.func.jvp(call, (t,), (t,)), lambda: torch.func.vmap(call)(torch.stack((t, t))),
                      lambda: torch.func.grad(lambda u: call(u).float().sum())(t)):
        with pytest.raises(RuntimeError, match='functorch transforms|data pointer'):
            transform()
    assert call(t).shape == t.shape                     # and nothing of it stays behind


@pytest.mark.parametrize('which', [0, 1, 2])
@pytest.mark.filterwarnings('ignore')
def test_a_trace_records_the_operator(calls_without_kernels, which):
    call, t = calls_without_kernels[which]
    graph = str(torch.jit.trace(call, t, check_trace=False).graph)
    assert ('^_Attention', '^_Rotary', '^_ResidualNorm')[which] in graph


def test_the_c_entries_refuse_what_the_kernels_cannot_do(native):
    import ctypes

    import _fga_native as api
    for entry in (native.fga_rotary_forward, native.fga_rotary_backward, native.fga_norm_forward, native.fga_norm_backward):
        assert entry(None, None) == -1 and b'null' in native.fga_last_error()
    norm = api.FgaNorm(16, tokens=4, hidden=64, samples=1)
    for field, value, message in (('tokens', 0, b'tokens'), ('hidden', 60, b'hidden'), ('hidden', 8200, b'hidden'),
                                  ('samples', 0, b'samples'), ('samples', 2, b'cu_seqlens'), ('gate', 16, b'branch'),
                                  ('x', 8, b'aligned'), ('tokens', 1 << 31, b'tokens')):
        broken = api.FgaNorm.from_buffer_copy(norm)
        setattr(broken, field, value)
        assert native.fga_norm_forward(ctypes.byref(broken), None) == -1 and message in native.fga_last_error()
    rotary = api.FgaRotary(tokens=4, axes=1, positions=16, inv_freq=16)
    rotary.sections[0] = 64
    for t in range(2):
        rotary.x[t], rotary.out[t], rotary.heads[t] = 16, 16, 1
    for change, message in ((lambda r: setattr(r, 'tokens', 0), b'tokens'), (lambda r: setattr(r, 'axes', 5), b'axes'),
                            (lambda r: r.sections.__setitem__(0, 63), b'sections'),
                            (lambda r: r.heads.__setitem__(1, 0), b'heads'),
                            (lambda r: r.x.__setitem__(0, 24), b'aligned'),
                            (lambda r: r.x.__setitem__(0, None), b'null'),
                            (lambda r: r.x_head_stride.__setitem__(1, 130), b'strides')):
        broken = api.FgaRotary.from_buffer_copy(rotary)
        change(broken)
        assert native.fga_rotary_forward(ctypes.byref(broken), None) == -1 and message in native.fga_last_error()


def test_the_norm_takes_a_branch_gradient_exactly_where_there_is_a_gate(native):
    import ctypes

    import _fga_native as api
    for gate, dbranch in ((16, None), (None, 16)):
        norm = api.FgaNorm(16, 16, tokens=4, hidden=64, samples=1, gate=gate, dbranch=dbranch, dx=16, rstd=16)
        assert native.fga_norm_backward(ctypes.byref(norm), None) == -1 and b'dbranch' in native.fga_last_error()


@pytest.mark.gpu
def test_the_c_entry_takes_the_stored_residual_sum_too(native):
    """backward with r and, for a gate, the branch, as a caller that keeps no x has them."""
    import _fga_native as api
    gen = torch.Generator(device='cuda').manual_seed(21)
    tokens, hidden = 50, 512
    t = dict(x=normal(gen, tokens, hidden), branch=normal(gen, tokens, hidden), weight=None,
             gate=normal(gen, 1, hidden), scale=None, shift=None)
    dy, dr = normal(gen, tokens, hidden), normal(gen, tokens, hidden)
    y, r, dx, dbranch = (torch.empty_like(dy) for _ in range(4))
    dgate, rstd = torch.empty_like(t['gate']), torch.empty(tokens, device='cuda')
    scratch = torch.empty(native.fga_norm_scratch_floats(tokens, hidden, 1, 0, 1), device='cuda')
    stream = torch.cuda.current_stream().cuda_stream
    gate, branch = t['gate'].data_ptr(), t['branch'].data_ptr()
    assert native.fga_norm_forward(api.NORM_BYTES.pack(
        t['x'].data_ptr(), branch, 0, gate, 0, 0, 0, y.data_ptr(), r.data_ptr(), rstd.data_ptr(), *(0,) * 10,
        tokens, hidden, 1, 0, 0, 0, 1e-6), stream) == 0
    assert native.fga_norm_backward(api.NORM_BYTES.pack(
        0, branch, 0, gate, 0, 0, 0, 0, r.data_ptr(), rstd.data_ptr(), 0, dy.data_ptr(), dr.data_ptr(), dx.data_ptr(),
        dbranch.data_ptr(), 0, dgate.data_ptr(), 0, 0, scratch.data_ptr(), tokens, hidden, 1, 0, 0, 0, 1e-6), stream) == 0
    _, _, grads, bounds = norm_bounds(t, [0, tokens], False, dy, dr, True)
    for name, value in (('x', dx), ('branch', dbranch), ('gate', dgate)):
        within(value, grads[name], bounds[name], name)


@pytest.mark.parametrize('tokens', [(1 << 31) - 1, (1 << 31) - (1 << 16) + 1])
def test_norm_rows_leave_room_for_32_bit_sums(native, tokens):
    import ctypes

    import _fga_native as api
    norm = api.FgaNorm(16, tokens=tokens, hidden=8, samples=1)
    for entry in (native.fga_norm_forward, native.fga_norm_backward):
        assert entry(ctypes.byref(norm), None) == -1 and b'tokens' in native.fga_last_error()


def test_gradients_of_the_plain_forms_against_differences():
    g = torch.Generator().manual_seed(3)

    def leaf(*shape):
        return torch.randn(*shape, generator=g, dtype=torch.float64).requires_grad_()

    pos = torch.tensor([[0, 3, 5], [7, 1, 2]])
    for interleaved in (True, False):
        assert torch.autograd.gradcheck(
            lambda x, w: plain.rotary(x, pos, frequencies(VIDEO), VIDEO, interleaved, w), (leaf(2, 2, 128), leaf(128)))
    for center in (True, False):
        assert torch.autograd.gradcheck(
            lambda x, b, w, gt, sc, sh: plain.residual_norm(x, b, w, gt, sc, sh, [0, 1, 1, 3], center=center),
            (leaf(4, 16), leaf(4, 16), leaf(16), leaf(3, 16), leaf(3, 16), leaf(3, 16)))


# ----------------------------------------------------------------------------------------- GPU
def normal(gen, *shape, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=gen, device='cuda') * std + mean).bfloat16()


@pytest.mark.gpu
@pytest.mark.parametrize('tokens,heads,kv_heads,sections,start,dtype', [
    (1, 1, 1, (64,), 0, torch.int32),
    (23, 8, 8, (64,), 1000003, torch.int64),
    (7, 5, 3, VIDEO, -9, torch.int32),
    (1025, 32, 4, (32, 32), 5, torch.int64),
    (5000, 3, 1, VIDEO, 2 ** 30, torch.int32),
    (300, 40, 2, (0, 10, 54, 0), 17, torch.int32),
])
@pytest.mark.parametrize('interleaved', [True, False])
@pytest.mark.parametrize('norm', ['none', 'both', 'q'])
def test_rotary_matches_the_plain_form(native, tokens, heads, kv_heads, sections, start, dtype, interleaved, norm):
    rotary, _ = ops()
    gen = torch.Generator(device='cuda').manual_seed(tokens + heads)
    q, k = normal(gen, tokens, heads, 128, std=2.0), normal(gen, tokens, kv_heads, 128)
    gq, gk = normal(gen, tokens, heads, 128), normal(gen, tokens, kv_heads, 128)
    wq = normal(gen, 128, std=0.2, mean=1.0) if norm != 'none' else None
    wk = normal(gen, 128, std=0.2, mean=1.0) if norm == 'both' else None
    pos = (torch.randint(0, 1000, (tokens, len(sections)), generator=gen, device='cuda') + start).to(dtype)
    freq = frequencies(sections).cuda()
    leaves = [t if t is None else t.detach().requires_grad_() for t in (q, wq, k, wk)]
    outs = rotary(leaves[0], leaves[2], pos, freq, sections, interleaved=interleaved, q_weight=leaves[1], k_weight=leaves[3])
    grads = iter(torch.autograd.grad(outs, [t for t in leaves if t is not None], (gq, gk)))
    for x, w, dy, y in ((q, wq, gq, outs[0]), (k, wk, gk, outs[1])):
        x64, w64 = x.double().requires_grad_(), None if w is None else w.double().requires_grad_()
        want = plain.rotary(x64, pos, freq, sections, interleaved, w64)
        back = torch.autograd.grad(want, [t for t in (x64, w64) if t is not None], dy.double())
        want = want.detach()
        reach = want.abs().amax(-1, keepdim=True)
        within(y, want, HALF * want.abs() + FINE * reach, 'output')
        dx = back[0]
        size = dy.abs().double().amax(-1, keepdim=True) if w is None else dx.abs().amax(-1, keepdim=True) + (
            dy.double().abs().amax(-1, keepdim=True) * w.double().abs().max()
            / (x.double().square().mean(-1, keepdim=True) + 1e-6).sqrt())
        within(next(grads), dx, HALF * dx.abs() + FINE * size, 'gradient')
        if w is not None:
            n = x.double() / (x.double().square().mean(-1, keepdim=True) + 1e-6).sqrt()
            terms = (dy.double().abs().amax(-1, keepdim=True) * n.abs()).sum((0, 1)) * 2 ** 0.5
            within(next(grads), back[1], HALF * back[1].abs() + FINE * terms, 'weight gradient')


@pytest.mark.gpu
@pytest.mark.parametrize('position,fastest', [(2 ** 31 - 5, 1e7), (2 ** 48 + 12345, 1.0), (-2 ** 50 + 7, 3.0), (5, 1e9)])
def test_rotary_angles_of_far_positions_and_high_frequencies(native, position, fastest):
    """Against angles in 60 digits. One position's rounding of a frequency, |position| * 2^-64 turns, and 2^-27 turns of
    FP32 steps are all that the angle may be off by; it moves an element by that times the length of its pair."""
    from mpmath import mp
    rotary, _ = ops()
    gen = torch.Generator(device='cuda').manual_seed(19)
    freq = (fastest * 1.07 ** -torch.arange(64, dtype=torch.float64)) * 0.9173
    x = normal(gen, 1, 4, 128)
    with mp.workdps(60):
        angles = [mp.mpf(f) * position for f in freq.tolist()]
        turn = torch.tensor([[float(mp.cos(a)), float(mp.sin(a))] for a in angles], dtype=torch.float64, device='cuda')
    a, b = x.double()[..., 0::2], x.double()[..., 1::2]
    want = torch.stack((a * turn[:, 0] - b * turn[:, 1], b * turn[:, 0] + a * turn[:, 1]), -1).flatten(-2)
    length = torch.stack((a.hypot(b),) * 2, -1).flatten(-2)
    off = 2 * 3.1416 * (abs(position) * 2.0 ** -64 + 2.0 ** -27)
    assert off < HALF / 8                                    # far below the rounding of the output
    got = rotary(x, x, torch.tensor([position], device='cuda'), freq.cuda())[0]
    within(got, want, HALF * want.abs() + (off + FINE) * length, 'output')


@pytest.mark.gpu
@pytest.mark.parametrize('heads,kv_heads', [(1, 1), (6, 2), (3, 3), (5, 1), (4, 4)])
def test_rotary_weight_gradients_without_an_epsilon(native, heads, kv_heads):
    """eps = 0 and head counts that do not fill a group of four head rows."""
    rotary, _ = ops()
    gen = torch.Generator(device='cuda').manual_seed(heads)
    tokens, pos, freq = 70, torch.arange(70, device='cuda'), frequencies((64,)).cuda()
    q, k = normal(gen, tokens, heads, 128, std=2.0), normal(gen, tokens, kv_heads, 128)
    gq, gk = normal(gen, tokens, heads, 128), normal(gen, tokens, kv_heads, 128)
    wq, wk = (normal(gen, 128, std=0.2, mean=1.0).requires_grad_() for _ in range(2))
    outs = rotary(q, k, pos, freq, q_weight=wq, k_weight=wk, eps=0.0)
    for x, w, dy, y, dw in zip((q, k), (wq, wk), (gq, gk), outs, torch.autograd.grad(outs, (wq, wk), (gq, gk))):
        w64 = w.detach().double().requires_grad_()
        want = plain.rotary(x.double(), pos[:, None], freq, (64,), True, w64, eps=0.0)
        dwant = torch.autograd.grad(want, w64, dy.double())[0]
        within(y.detach(), want.detach(), HALF * want.detach().abs() + FINE * want.detach().abs().amax(-1, keepdim=True), 'output')
        n = x.double() / x.double().square().mean(-1, keepdim=True).sqrt()
        terms = (dy.double().abs().amax(-1, keepdim=True) * n.abs()).sum((0, 1)) * 2 ** 0.5
        within(dw, dwant, HALF * dwant.abs() + FINE * terms, 'weight gradient')


@pytest.mark.gpu
def test_rotary_reads_strided_heads_and_leaves_its_inputs(native):
    rotary, _ = ops()
    gen = torch.Generator(device='cuda').manual_seed(1)
    packed = normal(gen, 33, 6, 128)
    q, k = packed[:, :4], normal(gen, 2, 33, 128).transpose(0, 1)
    pos, freq = torch.arange(33, device='cuda'), frequencies((64,), torch.float32).cuda()
    w = normal(gen, 128, mean=1.0)
    before = packed.clone()
    kwargs = dict(q_weight=w, k_weight=w, interleaved=False)
    a = rotary(q.requires_grad_(), k.requires_grad_(), pos, freq, **kwargs)
    b = rotary(q.detach().contiguous().requires_grad_(), k.detach().contiguous().requires_grad_(), pos, freq, **kwargs)
    dq, dk = torch.autograd.grad(sum(t.float().sum() for t in a), (q, k))      # expanded gradients
    assert all(torch.equal(s, t) for s, t in zip(a, b)) and torch.equal(packed, before)
    want = plain.rotary(q.detach().double().requires_grad_(), pos[:, None], freq, (64,), False, w.double())
    within(a[0], want.detach(), HALF * want.detach().abs() + FINE * want.abs().amax().item(), 'output')
    assert dq.shape == q.shape and dk.shape == k.shape


@pytest.mark.gpu
def test_rotary_accumulates_into_main_grad_and_takes_no_tokens(native):
    rotary, _ = ops()
    gen = torch.Generator(device='cuda').manual_seed(2)
    q, k = normal(gen, 50, 4, 128), normal(gen, 50, 2, 128)
    pos, freq = torch.arange(50, device='cuda'), frequencies((64,)).cuda()
    plain_w = normal(gen, 128, mean=1.0)

    def grads(weight):
        outs = rotary(q, k, pos, freq, q_weight=weight)
        return torch.autograd.grad(outs, weight, [torch.ones_like(t) for t in outs])[0]

    want = grads(plain_w.clone().requires_grad_())
    owned = torch.nn.Parameter(plain_w.clone())
    owned.main_grad = torch.full((128,), 3.0, device='cuda')
    grads(owned)
    grads(owned)
    assert owned.grad_added_to_main_grad
    within((owned.main_grad - 3.0) / 2, want.double(), 2 * HALF * want.double().abs() + 1e-5, 'main_grad')
    empty = rotary(q[:0], k[:0], pos[:0], freq, q_weight=owned)
    assert empty[0].shape == (0, 4, 128)
    bare = plain_w.clone().requires_grad_()
    outs = rotary(q[:0], k[:0], pos[:0], freq, q_weight=bare)
    assert torch.autograd.grad(outs, bare, [torch.ones_like(t) for t in outs])[0].abs().max() == 0


def test_one_weight_gradient_for_both_tensors_has_to_accumulate(native):
    import ctypes

    import _fga_native as api
    rotary = api.FgaRotary(tokens=4, axes=1, positions=16, inv_freq=16, scratch=16)
    rotary.sections[0] = 64
    for t in range(2):
        rotary.x[t], rotary.dy[t], rotary.out[t], rotary.weight[t], rotary.dweight[t] = 16, 16, 16, 16, 32
        rotary.heads[t] = 1
    for f32, accumulate in (((1, 1), (0, 0)), ((1, 1), (1, 0)), ((0, 0), (1, 1)), ((1, 0), (1, 1))):
        for t in range(2):
            rotary.dweight_f32[t], rotary.dweight_accumulate[t] = f32[t], accumulate[t]
        assert native.fga_rotary_backward(ctypes.byref(rotary), None) == -1 and b'accumulate' in native.fga_last_error()


@pytest.mark.gpu
def test_one_head_norm_weight_for_queries_and_keys(native):
    """A weight tied between q and k gets the sum of both gradients in its main_grad, in every run."""
    rotary, _ = ops()
    gen = torch.Generator(device='cuda').manual_seed(16)
    q, k = normal(gen, 64, 8, 128), normal(gen, 64, 8, 128)
    gq, gk = normal(gen, 64, 8, 128), normal(gen, 64, 8, 128)
    pos, freq = torch.arange(64, device='cuda'), frequencies((64,)).cuda()
    w = normal(gen, 128, mean=1.0)
    apart = [torch.nn.Parameter(w.clone()) for _ in range(2)]
    for p in apart:
        p.main_grad = torch.zeros(128, device='cuda')
    torch.autograd.backward(rotary(q, k, pos, freq, q_weight=apart[0], k_weight=apart[1]), (gq, gk))
    want = apart[0].main_grad + apart[1].main_grad            # what adding q's, then k's to zero rounds to
    for _ in range(200):
        tied = torch.nn.Parameter(w.clone())
        tied.main_grad = torch.zeros(128, device='cuda')
        torch.autograd.backward(rotary(q, k, pos, freq, q_weight=tied, k_weight=tied), (gq, gk))
        assert torch.equal(tied.main_grad, want)


def norm_bounds(t, cu, center, dy, dr, has_branch, rounded=True):
    """Expected values and error bounds of y, r and every gradient, in 64 bits."""
    names = ('x', 'branch', 'weight', 'gate', 'scale', 'shift')
    leaves = {n: None if t[n] is None else t[n].double().requires_grad_() for n in names}
    y, r = plain.residual_norm(*(leaves[n] for n in names), cu=cu, center=center)
    present = [n for n in names if t[n] is not None]
    grads = dict(zip(present, torch.autograd.grad((y, r), [leaves[n] for n in present], (dy.double(), dr.double()))))
    y, r = y.detach(), r.detach()
    tokens, hidden = r.shape
    one = torch.ones(tokens, hidden, dtype=torch.float64, device=r.device)
    ends = torch.tensor([b for _, b in plain.segments(cu, tokens)], device=r.device)
    sample = torch.searchsorted(ends, torch.arange(tokens, device=r.device), right=True)
    inside = (sample < len(ends))[:, None]
    at = sample.clamp(max=len(ends) - 1)
    row = {n: one if t[n] is None else t[n].double()[at] for n in ('gate', 'scale', 'shift')}
    w = one if t['weight'] is None else t['weight'].double().expand(tokens, hidden)
    gain = 1 + row['scale'] if t['scale'] is not None else one
    c = r - r.mean(-1, keepdim=True) if center else r
    rstd = 1 / (c.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    n = c * rstd
    stored = HALF * r.abs() * rstd if has_branch and rounded else 0 * r    # error of n from the stored residual sum
    stored = stored + FINE * (r.abs() + r.abs().mean(-1, keepdim=True)) * rstd
    bounds = {'y': HALF * y.abs() + FINE * ((r.abs() + r.abs().mean(-1, keepdim=True)) * rstd * w.abs() * gain.abs()
                                            + n.abs() * w.abs() * gain.abs() + row['shift'].abs() * (t['shift'] is not None)),
              'r': HALF * r.abs() + FINE * r.abs() + 1e-30}
    dyd, drd = dy.double() * inside, dr.double()
    dn = dyd * gain * w
    dot = (dn * n).mean(-1, keepdim=True)
    ddot = (dn.abs() * stored).mean(-1, keepdim=True) + FINE * (dn * n).abs().mean(-1, keepdim=True)
    dxe = rstd * (n.abs() * ddot + stored * dot.abs() + FINE * (dn.abs() + dn.abs().mean(-1, keepdim=True)))
    dxe = dxe + FINE * drd.abs()                                       # before the output's rounding
    dx = grads['x']
    bounds['x'] = HALF * dx.abs() * (1 + HALF) + dxe * (1 + HALF)
    if has_branch:
        g = row['gate'].abs() if t['gate'] is not None else one
        bounds['branch'] = HALF * grads['branch'].abs() + g * dxe * (1 + HALF) + FINE * grads['branch'].abs()
        if t['gate'] is None:
            bounds['branch'] = bounds['x']

    def summed(terms):           # per sample
        out = torch.zeros(len(ends), hidden, dtype=torch.float64, device=r.device)
        return out.index_add_(0, at, terms * inside)

    if t['gate'] is not None:
        b = t['branch'].double().abs()
        bounds['gate'] = HALF * grads['gate'].abs() + summed((dxe + FINE * dx.abs()) * b) + 1e-30
    if t['scale'] is not None:
        bounds['scale'] = HALF * grads['scale'].abs() + summed(dyd.abs() * w.abs() * (stored + FINE * n.abs())) + 1e-30
    if t['shift'] is not None:
        bounds['shift'] = HALF * grads['shift'].abs() + summed(FINE * dyd.abs()) + 1e-30
    if t['weight'] is not None:
        bounds['weight'] = (HALF * grads['weight'].abs()
                            + (dyd.abs() * gain.abs() * (stored + FINE * n.abs())).sum(0) + 1e-30)
    return y, r, grads, bounds


@pytest.mark.gpu
@pytest.mark.parametrize('lengths,pad,hidden', [
    ([1], 0, 8), ([23], 0, 1024), ([5, 0, 1, 94], 0, 2048), ([300, 1, 700], 13, 2056), ([1000], 0, 4096),
    ([0, 0, 17], 0, 5120), ([3, 130], 300, 8192), ([0], 9, 512),
])
@pytest.mark.parametrize('parts', ['plain', 'weight', 'branch', 'branch+weight', 'gate', 'all', 'scale', 'shift+branch'])
@pytest.mark.parametrize('center', [False, True])
def test_norm_matches_the_plain_form(native, lengths, pad, hidden, parts, center):
    _, norm = ops()
    gen = torch.Generator(device='cuda').manual_seed(sum(lengths) + hidden)
    tokens, samples = sum(lengths) + pad, len(lengths)
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    t = dict(x=normal(gen, tokens, hidden, std=2.0, mean=0.5), branch=None, weight=None, gate=None, scale=None, shift=None)
    if parts in ('branch', 'branch+weight', 'gate', 'all', 'shift+branch'):
        t['branch'] = normal(gen, tokens, hidden)
    if parts in ('weight', 'branch+weight', 'all'):
        t['weight'] = normal(gen, hidden, std=0.2, mean=1.0)
    for name, uses in (('gate', ('gate', 'all')), ('scale', ('scale', 'all')), ('shift', ('shift+branch', 'all'))):
        if parts in uses:
            t[name] = normal(gen, samples, hidden, std=0.5)
    dy, dr = normal(gen, tokens, hidden), normal(gen, tokens, hidden)
    if pad:
        dy[-pad:] = float('nan')        # what padding rows hold is nobody's business ...
    leaves = {n: None if v is None else v.detach().requires_grad_() for n, v in t.items()}
    y, r = norm(leaves['x'], leaves['branch'], **{n: leaves[n] for n in ('weight', 'gate', 'scale', 'shift')},
                cu_seqlens=torch.tensor(cu, dtype=torch.int32, device='cuda'), center=center)
    present = [n for n in leaves if leaves[n] is not None]
    got = dict(zip(present, torch.autograd.grad((y, r), [leaves[n] for n in present], (dy, dr))))
    if pad:
        dy[-pad:] = 0                   # ... and nothing of it reaches a gradient
    want_y, want_r, grads, bounds = norm_bounds(t, cu, center, dy, dr, t['branch'] is not None)
    within(y.detach(), want_y, bounds['y'], 'y')
    within(r.detach(), want_r, bounds['r'], 'r')
    for name in present:
        within(got[name], grads[name], bounds[name], f'gradient of {name}')


@pytest.mark.gpu
@pytest.mark.parametrize('parts', ['branch', 'branch+weight', 'gate', 'all', 'scale'])
@pytest.mark.parametrize('hidden', [512, 4096])
@pytest.mark.parametrize('center', [False, True])
def test_norm_gradients_of_rows_far_from_zero(native, parts, hidden, center):
    """Rows whose mean is many deviations from zero: a residual sum that has been rounded to BF16 would leave little of
    what a centred norm makes of it. Bounds without that rounding; an RMS norm with a gate has none either."""
    if not center and parts not in ('gate', 'all'):
        pytest.skip('reads the rounded residual sum')
    _, norm = ops()
    gen = torch.Generator(device='cuda').manual_seed(hidden)
    lengths, pad = [70, 0, 1, 40], 5
    tokens, cu = sum(lengths) + pad, [0, 70, 70, 71, 111]
    t = dict(x=normal(gen, tokens, hidden, mean=40.0), branch=normal(gen, tokens, hidden), weight=None, gate=None, scale=None,
             shift=None)
    if parts in ('branch+weight', 'all'):
        t['weight'] = normal(gen, hidden, std=0.2, mean=1.0)
    for name, uses in (('gate', ('gate', 'all')), ('scale', ('scale', 'all')), ('shift', ('all',))):
        if parts in uses:
            t[name] = normal(gen, 4, hidden, std=0.5)
    dy, dr = normal(gen, tokens, hidden), normal(gen, tokens, hidden)
    leaves = {n: None if v is None else v.detach().requires_grad_() for n, v in t.items()}
    outs = norm(leaves['x'], leaves['branch'], **{n: leaves[n] for n in ('weight', 'gate', 'scale', 'shift')},
                cu_seqlens=torch.tensor(cu, dtype=torch.int32, device='cuda'), center=center)
    present = [n for n in leaves if leaves[n] is not None]
    got = torch.autograd.grad(outs, [leaves[n] for n in present], (dy, dr))
    _, _, grads, bounds = norm_bounds(t, cu, center, dy, dr, True, rounded=False)
    for name, value in zip(present, got):
        within(value, grads[name], bounds[name], f'gradient of {name}')


@pytest.mark.gpu
def test_norm_is_the_same_twice_and_in_a_graph_and_on_a_side_stream(native):
    _, norm = ops()
    gen = torch.Generator(device='cuda').manual_seed(5)
    x, b = normal(gen, 777, 1536), normal(gen, 777, 1536)
    rows = [normal(gen, 2, 1536) for _ in range(3)]
    w = normal(gen, 1536, mean=1.0)
    cu = torch.tensor([0, 400, 777], dtype=torch.int32, device='cuda')
    leaves = [t.requires_grad_() for t in (x, b, w, *rows)]
    dy = normal(gen, 777, 1536)

    def step():
        y, r = norm(leaves[0], leaves[1], weight=leaves[2], gate=leaves[3], scale=leaves[4], shift=leaves[5], cu_seqlens=cu)
        return [y.detach(), r.detach(), *torch.autograd.grad((y, r), leaves, (dy, dy))]

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, c, d in zip(first, second, captured):
        assert torch.equal(a, c) and torch.equal(a, d)


@pytest.mark.gpu
def test_more_than_2_to_31_elements(native):
    """Offsets that do not fit 32 bits: the last rows come out like the same rows alone."""
    rotary, norm = ops()
    gen = torch.Generator(device='cuda').manual_seed(6)
    tokens, heads = 540_000, 32                      # 2.2e9 elements
    q = torch.empty(tokens, heads, 128, dtype=torch.bfloat16, device='cuda')
    q[:8], q[-8:] = normal(gen, 8, heads, 128), normal(gen, 8, heads, 128)
    q[8:-8] = 1.0
    k, w = normal(gen, tokens, 1, 128), normal(gen, 128, mean=1.0)
    pos, freq = torch.arange(tokens, device='cuda'), frequencies((64,)).cuda()
    whole = rotary(q, k, pos, freq, q_weight=w)
    alone = rotary(q[-8:], k[-8:], pos[-8:], freq, q_weight=w)
    assert torch.equal(whole[0][-8:], alone[0]) and torch.equal(whole[1][-8:], alone[1])
    dq = torch.autograd.grad(rotary(q.requires_grad_(), k, pos, freq, q_weight=w)[0], q, whole[0])[0]
    part = q[-8:].detach().requires_grad_()
    assert torch.equal(dq[-8:], torch.autograd.grad(rotary(part, k[-8:], pos[-8:], freq, q_weight=w)[0], part, whole[0][-8:])[0])
    del whole, dq
    x = q.detach().view(-1, 8192)
    y, r = norm(x, x, weight=normal(gen, 8192, mean=1.0).fill_(0.5))
    assert torch.equal(r[-2:], (x[-2:].float() * 2).bfloat16())
    want = plain.residual_norm(x[-2:].double(), x[-2:].double(), torch.full((8192,), 0.5, device='cuda').double())[0]
    within(y[-2:], want, HALF * want.abs() + FINE * want.abs().max(), 'y')


@pytest.mark.gpu
def test_norms_of_several_widths_from_several_threads(native):
    """The limits a launch needs are the kernel's: threads with other widths must not lower them in between."""
    import threading

    import _fga_native as api
    widths, calls, failures = (8192, 4608, 6144, 5120), 20000, []
    start = threading.Barrier(len(widths))

    def work(hidden):
        try:
            stream = torch.cuda.Stream()
            x, b, y, r = (torch.ones(2, hidden, dtype=torch.bfloat16, device='cuda') for _ in range(4))
            torch.cuda.synchronize()
            args = api.NORM_BYTES.pack(x.data_ptr(), b.data_ptr(), 0, 0, 0, 0, 0, y.data_ptr(), r.data_ptr(), *(0,) * 11,
                                       2, hidden, 1, 0, 0, 0, 1e-6)
            start.wait()
            refused = sum(native.fga_norm_forward(args, stream.cuda_stream) != 0 for _ in range(calls))
            stream.synchronize()
            assert (r == 2).all() and (y == 1).all()
            if refused:
                failures.append(f'{hidden}: {refused} of {calls} launches refused')
        except Exception as error:                                                  # noqa: BLE001
            failures.append(f'{hidden}: {error!r}')

    threads = [threading.Thread(target=work, args=(hidden,)) for hidden in widths]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failures, failures


@pytest.mark.gpu
def test_gradients_are_not_differentiable_twice(native):
    _, norm = ops()
    x = torch.ones(4, 64, dtype=torch.bfloat16, device='cuda', requires_grad=True)
    dx, = torch.autograd.grad(norm(x)[0].float().square().sum(), x, create_graph=True)   # depends on y, so on x
    with pytest.raises(RuntimeError, match='once_differentiable'):
        dx.float().sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize('used', ['y', 'r'])
@pytest.mark.parametrize('modulated', [False, True])
def test_norm_gradients_where_one_output_is_not_used(native, used, modulated):
    _, norm = ops()
    gen = torch.Generator(device='cuda').manual_seed(15)
    t = dict(x=normal(gen, 70, 256), branch=normal(gen, 70, 256), weight=normal(gen, 256, mean=1.0), gate=None, scale=None,
             shift=None)
    if modulated:
        t.update({n: normal(gen, 2, 256, std=0.5) for n in ('gate', 'scale', 'shift')})
    cu, g, none = [0, 33, 70], normal(gen, 70, 256), torch.zeros(70, 256, dtype=torch.bfloat16, device='cuda')
    leaves = {n: None if v is None else v.detach().requires_grad_() for n, v in t.items()}
    outs = norm(leaves['x'], leaves['branch'], **{n: leaves[n] for n in ('weight', 'gate', 'scale', 'shift')},
                cu_seqlens=torch.tensor(cu, dtype=torch.int32, device='cuda'))
    present = [n for n in leaves if leaves[n] is not None]
    got = torch.autograd.grad(outs[used == 'r'], [leaves[n] for n in present], g)
    _, _, grads, bounds = norm_bounds(t, cu, False, g if used == 'y' else none, g if used == 'r' else none, True)
    for name, value in zip(present, got):
        within(value, grads[name], bounds[name], name)
