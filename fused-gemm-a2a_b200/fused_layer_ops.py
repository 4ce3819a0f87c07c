"""Operators around the fused projections of an attention layer (B200 / sm_100a): attention over packed
sequences, rotary positions and the norm around a block, forward and backward, on the layouts the
projections use: head side BF16 [tokens, heads, 128], sequence side BF16 [tokens, hidden].

    y, x = residual_norm(x, branch, weight=w)             # x + branch, normalised for the next block
    q, k, v = FusedQKVProjection(...)(y, workspace)
    q, k = rotary_embedding(q, k, positions, inv_freq, sections)
    branch = FusedOutputProjection(...)(packed_attention(q, k, v, cu_seqlens), workspace)

The reference leaves these to its callers. As with the projections, weights are caller-owned BF16
tensors; a weight with a Megatron `main_grad` gets its gradient accumulated there. Packed sequences are
described by `cu_seqlens`, an int32 device tensor [samples + 1] of ascending offsets into the token axis
that starts at 0 and is never read by the host; rows from its last offset on belong to no sequence.
All device work is one or a few launches of libfga.so on the current stream of the tensors' device; there
is no CPU or PyTorch fallback. Gradients are of first order and in reverse; forward-mode derivatives and function
transforms (torch.func) raise. Calls may be captured into CUDA graphs, backward passes included; as with any
autograd code, no graph recorded outside the capture may then still hold the same leaves (autograd ties a
leaf to the stream of the first graph that uses it and would wait on that stream from inside the capture).
"""
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

import _fga_native as _native
import fused_gemm_a2a_kernels as _k

HEAD_DIM = 128
MAX_HIDDEN = 8192


def _address(t):
    return 0 if t is None else t.data_ptr()


def _same_device(first, *others):
    if not first.is_cuda:
        raise ValueError('The fused kernels only run on CUDA tensors; there is no CPU path')
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError('All tensors of a call must be on the same CUDA device')


def _launch(entry, args, device):
    """Call a libfga entry point with packed arguments on the current stream of `device`, whichever device is
    current."""
    index = device.index
    if torch.cuda.current_device() == index:
        rc = entry(args, torch._C._cuda_getCurrentRawStream(index))
        if rc:
            _native.check(rc)
        return
    with torch.cuda.device(device):
        _native.check(entry(args, torch._C._cuda_getCurrentRawStream(index)))


def _floats(entry, device, *sizes):
    """FP32 scratch of the size the library asks for on `device`."""
    if torch.cuda.current_device() == device.index:
        return torch.empty(entry(*sizes), device=device, dtype=torch.float32)
    with torch.cuda.device(device):
        return torch.empty(entry(*sizes), device=device, dtype=torch.float32)


def _fresh(t):
    """Contiguous, uninitialised storage for a tensor like `t`."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format)


def _through_autograd(*tensors):
    """Whether autograd has to see a call: for gradients; for forward-mode derivatives and function transforms, which
    it refuses there, where a plain call would drop them; and for a trace, which would record no kernel."""
    return (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
            or forward_ad._current_level >= 0 or torch._C._are_functorch_transforms_active() or torch._C._is_tracing())


def _head_tensor(t, label):
    """[tokens, heads, 128] BF16 whose heads are contiguous 16-byte aligned rows, with any token and head
    stride that keeps them so."""
    shape = t.shape
    if (len(shape) == 3 and shape[2] == HEAD_DIM and shape[1] and t.dtype is torch.bfloat16 and t.is_contiguous()
            and not t.data_ptr() & 15):
        return
    if t.ndim != 3 or t.shape[2] != HEAD_DIM or t.dtype != torch.bfloat16:
        raise ValueError(f'{label} must be a BF16 tensor [tokens, heads, {HEAD_DIM}], got {t.dtype} {tuple(t.shape)}')
    if t.shape[1] < 1:
        raise ValueError(f'{label} needs at least one head')
    token, head, inner = t.stride()
    if (inner != 1 or t.data_ptr() % 16 or (t.shape[0] > 1 and (token % 8 or token < HEAD_DIM))
            or (t.shape[1] > 1 and (head % 8 or head < HEAD_DIM))):
        raise ValueError(f'{label} needs contiguous 16-byte aligned heads: strides {t.stride()}')


def _strides(t):
    """Token and head stride; those of extents of one are never used and may be anything."""
    token, head, _ = t.stride()
    return token if t.shape[0] > 1 else t.shape[1] * HEAD_DIM, head if t.shape[1] > 1 else HEAD_DIM


def _vector(t, length, label):
    if t is None:
        return
    if tuple(t.shape) != (length,) or t.dtype != torch.bfloat16 or not t.is_contiguous() or t.data_ptr() % 16:
        raise ValueError(f'{label} must be a contiguous, 16-byte aligned BF16 vector of {length} entries')


def _epsilon(eps):
    if not 0.0 <= eps < float('inf'):
        raise ValueError('eps must be finite and not negative')


def _offsets(cu_seqlens, label='cu_seqlens'):
    if (cu_seqlens.ndim != 1 or cu_seqlens.dtype != torch.int32 or not cu_seqlens.is_contiguous()
            or cu_seqlens.shape[0] < 2):
        raise ValueError(f'{label} must be a contiguous int32 vector of at least two offsets')


def _grad_rows(g, like):
    """A gradient in the layout the kernels read: contiguous and 16-byte aligned (autograd may hand over
    expanded or transposed ones)."""
    if g.dtype != torch.bfloat16 or g.shape != like:
        raise ValueError(f'gradients must be BF16 of shape {tuple(like)}')
    g = g.contiguous()
    return g if g.data_ptr() % 16 == 0 else g.clone()


def _weight_target(weight, wanted):
    """(tensor the gradient of `weight` goes to, accumulate): its FP32 main_grad where it has one, else a
    fresh tensor of its own type."""
    if weight is None or not wanted:
        return None, False
    main_grad = getattr(weight, 'main_grad', None)
    if main_grad is None:
        return torch.empty_like(weight), False
    if (main_grad.shape != weight.shape or main_grad.dtype != torch.float32 or not main_grad.is_contiguous()
            or main_grad.device != weight.device):
        raise ValueError('main_grad must match the weight shape with contiguous FP32 storage')
    return main_grad, True


def _weight_result(weight, target, accumulated):
    if target is None or not accumulated:
        return target
    from fused_gemm_a2a import _accumulated
    return _accumulated(weight)


# ----------------------------------------------------------------------------------------------
# Attention
# ----------------------------------------------------------------------------------------------
def _status(device):
    """The device's status word for kernels outside a CP group, which the check_status() of any group on
    the device covers. Never created from inside a capture."""
    word = _k._local_status.get(device)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError('Call packed_attention once on this device before capturing it into a CUDA graph')
        word = _k._status_word(device)
    return word


def check_status(device=None, *, clear=False):
    """Synchronize with all streams of `device` (default: the current one) and raise if an attention kernel gave up
    on a bounded wait. Such an error is sticky: the kernels of later attention calls on the device return without
    computing, and every attention call raises as soon as the host has got the error, without waiting for it, until it
    has been cleared, here with clear=True or by a group's clear_status()."""
    device = torch.device('cuda' if device is None else device)
    if device.index is None:
        device = torch.device('cuda', torch.cuda.current_device())
    word = _k._local_status.get(device)
    if word is None:
        return
    _k._synchronize(word)
    code, where, detail, _ = word.tolist()
    if clear:
        word.zero_()
        _k._synchronize(word)     # before any other stream may launch on it
    if clear or not code:
        _k._forget_host_status(device)
    _raise_for(code, where, detail)


def _raise_for(code, where, detail):
    if code:
        reason = _native.DEVICE_ERRORS.get(code, 'unknown device error')
        raise RuntimeError(f'Attention device error {code}: {reason} (where={where}, detail={detail}). Outputs and '
                           'gradients produced since then are not valid; check_status(clear=True) clears it')


def _host_status_address(device):
    """Where kernels leave an error for the host. Raises what an earlier one has left there."""
    copy = _k._host_status(device)
    if copy is None:
        return 0
    words = copy.words
    if words[0]:
        _raise_for(*words[:3])
    return copy.address


def _attention_args(q, k, v, o, lse, cu_seqlens, causal, scale, d_o=None, dq=None, dk=None, dv=None, delta=None):
    (q_token, q_head), (k_token, k_head), (v_token, v_head) = _strides(q), _strides(k), _strides(v)
    tokens, heads, _ = q.shape
    return _native.ATTENTION_BYTES.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _address(lse), _address(d_o), _address(dq), _address(dk),
        _address(dv), _address(delta), _address(cu_seqlens), _status(q.device).data_ptr(), _k.DEVICE_TIMEOUT_NS, q_token,
        k_token, v_token, q_head, k_head, v_head, tokens, heads, k.shape[1],
        1 if cu_seqlens is None else cu_seqlens.shape[0] - 1, causal, scale, _host_status_address(q.device))


def _attend(q, k, v, cu_seqlens, causal, scale, keep_lse):
    tokens, heads, _ = q.shape
    o = _fresh(q)
    lse = torch.empty((heads, tokens), device=q.device, dtype=torch.float32) if keep_lse else None
    if tokens:
        _launch(_native.lib().fga_attention_forward, _attention_args(q, k, v, o, lse, cu_seqlens, causal, scale), q.device)
    return o, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, causal, scale, return_lse):
        o, lse = _attend(q, k, v, cu_seqlens, causal, scale, True)
        ctx.save_for_backward(q, k, v, o, lse, cu_seqlens)
        ctx.rule = (causal, scale)
        ctx.set_materialize_grads(False)
        if not return_lse:
            return o
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o, *_):
        if d_o is None:
            return (None,) * 7
        q, k, v, o, lse, cu_seqlens = ctx.saved_tensors
        d_o = _grad_rows(d_o, o.shape)
        grads = [_fresh(t) for t in (q, k, v)]
        if q.shape[0]:
            _launch(_native.lib().fga_attention_backward,
                    _attention_args(q, k, v, o, lse, cu_seqlens, *ctx.rule, d_o, *grads, torch.empty_like(lse)), q.device)
        return (*grads, None, None, None, None)


def packed_attention(q, k, v, cu_seqlens=None, *, causal=False, scale=None, return_lse=False):
    """softmax(scale * q k^T) v within each packed sequence, for each query head: q [tokens, heads, 128],
    k and v [tokens, kv_heads, 128] BF16 -> o [tokens, heads, 128], contiguous. kv_heads divides heads;
    query head h reads key/value head h // (heads // kv_heads). That is what FusedQKVProjection returns and
    FusedOutputProjection takes.

    cu_seqlens: sequence offsets (default: all tokens are one sequence); a token sees the tokens of its own
    sequence, with `causal` those up to itself. Lengths may be anything, zero and one included. Rows behind
    the last sequence give o = 0 and gradients of 0, and what they hold in q, k, v and in the incoming
    gradient is not looked at. A NaN or infinity inside a sequence may reach every row of that sequence, of
    others none. scale: positive, default 128 ** -0.5. return_lse: also return the FP32
    [heads, tokens] logarithms of the rows' sums of exponentials (-inf behind the last sequence; no gradient
    flows through them).

    Range of the scores: the output holds its precision while a row's largest |scale * q k| is below 2^28,
    and the row is NaN from 2^29 on. In the backward pass probabilities are off by about 2^-23 of the score:
    less than their rounding to BF16 up to scores of 2^14, an eighth at 2^20; gradients of and through rows
    beyond that are NaN.

    Scores, softmax statistics and all sums are FP32; the probabilities (and in the backward pass the
    gradients of the scores) are rounded to BF16 for the second product. The backward pass takes the row
    sums of do * o from o as it was returned, rounded to BF16, for rows that may see more than 128 keys.
    Results, gradients included, are the same bits in every run. Kernel waits are bounded as in the
    projections. One that expires is recorded in the device's status word, which check_status() and a
    group's comm.check_status() read, and raised by the first later call, forward or backward, that finds it
    in host memory."""
    for t, label in ((q, 'q'), (k, 'k'), (v, 'v')):
        _head_tensor(t, label)
    if k.shape != v.shape or k.shape[0] != q.shape[0]:
        raise ValueError('k and v must have one shape, and q, k and v the same number of tokens')
    if q.shape[1] % k.shape[1]:
        raise ValueError('Query heads must be a multiple of key/value heads')
    scale = HEAD_DIM ** -0.5 if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:
        raise ValueError('scale must be positive, from 1e-30 to 1e30')
    if cu_seqlens is not None:
        _offsets(cu_seqlens)
        if cu_seqlens.shape[0] > 65536:
            raise ValueError('at most 65535 packed sequences')
    _same_device(q, k, v, cu_seqlens)
    if _through_autograd(q, k, v):
        return _Attention.apply(q, k, v, cu_seqlens, bool(causal), scale, bool(return_lse))
    o, lse = _attend(q, k, v, cu_seqlens, bool(causal), scale, return_lse)
    return (o, lse) if return_lse else o


# ----------------------------------------------------------------------------------------------
# Rotary positions
# ----------------------------------------------------------------------------------------------
def _rotary_args(xs, outs, weights, positions, inv_freq, sections, interleaved, eps, dys=(None, None),
                 targets=((None, False), (None, False)), scratch=None):
    (q_token, q_head), (k_token, k_head) = ((0, 0) if x is None else _strides(x) for x in xs)
    pairs = sections + (0,) * (4 - len(sections))
    (dwq, add_q), (dwk, add_k) = targets
    return _native.ROTARY_BYTES.pack(
        _address(xs[0]), _address(xs[1]), q_token, k_token, q_head, k_head, _address(dys[0]), _address(dys[1]),
        outs[0].data_ptr(), outs[1].data_ptr(), _address(weights[0]), _address(weights[1]), _address(dwq), _address(dwk),
        positions.data_ptr(), inv_freq.data_ptr(), _address(scratch), outs[0].shape[0], outs[0].shape[1], outs[1].shape[1],
        positions.dtype is torch.int64, inv_freq.dtype is torch.float64, len(sections), *pairs, interleaved,
        dwq is not None and dwq.dtype is torch.float32, dwk is not None and dwk.dtype is torch.float32, add_q, add_k, eps)


def _rotate(q, k, q_weight, k_weight, positions, inv_freq, sections, interleaved, eps):
    outs = _fresh(q), _fresh(k)
    if q.shape[0]:
        _launch(_native.lib().fga_rotary_forward,
                _rotary_args((q, k), outs, (q_weight, k_weight), positions, inv_freq, sections, interleaved, eps), q.device)
    return outs


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, inv_freq, sections, interleaved, eps):
        outs = _rotate(q, k, q_weight, k_weight, positions, inv_freq, sections, interleaved, eps)
        # without a head norm the rotation's gradient does not need its input
        ctx.save_for_backward(q if q_weight is not None else None, k if k_weight is not None else None, q_weight,
                              k_weight, positions, inv_freq)
        ctx.owners = (q_weight, k_weight)      # the caller's own parameters, which carry main_grad
        ctx.shapes, ctx.rule = (q.shape, k.shape), (sections, interleaved, eps)
        return outs

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, positions, inv_freq = ctx.saved_tensors
        sections, interleaved, eps = ctx.rule
        grads = [_grad_rows(g, shape) for g, shape in zip((dq_out, dk_out), ctx.shapes)]
        outs = [_fresh(g) for g in grads]
        targets = [_weight_target(w, needed) for w, needed in zip(ctx.owners, ctx.needs_input_grad[2:4])]
        tokens = outs[0].shape[0]
        if tokens:
            lib, scratch = _native.lib(), None
            if q_weight is not None or k_weight is not None:
                scratch = _floats(lib.fga_rotary_scratch_floats, positions.device, tokens, outs[0].shape[1], outs[1].shape[1])
            _launch(lib.fga_rotary_backward,
                    _rotary_args((q, k), outs, (q_weight, k_weight), positions, inv_freq, sections, interleaved, eps,
                                 grads, targets, scratch), positions.device)
        else:
            for target, accumulate in targets:
                if target is not None and not accumulate:
                    target.zero_()
        dw = [_weight_result(w, *target) for w, target in zip(ctx.owners, targets)]
        return (*outs, *dw, None, None, None, None, None)


def rotary_embedding(q, k, positions, inv_freq, sections=None, *, interleaved=True, q_weight=None, k_weight=None,
                     eps=1e-6):
    """Rotary positions of the query and key heads, with several axes: q [tokens, heads, 128], k [tokens,
    kv_heads, 128] BF16 -> new contiguous tensors of the same shapes. One launch for both.

    positions: int32 or int64 [tokens, axes] (or [tokens] for one axis), negative ones included. inv_freq:
    FP32 or FP64 [64], radians per position of each pair of elements; the first sections[0] pairs turn with
    axis 0 (time), the next sections[1] with axis 1 (height), and so on (default: all with one axis). Pairs
    are elements (2i, 2i+1) when `interleaved`, (i, i+64) otherwise. Angles are kept modulo a turn in 64-bit
    fixed point: they are off by less than 2^-27 turns at positions up to 2^36, and beyond (int64) by |position| *
    2^-64 turns.

    q_weight / k_weight (BF16 [128], each optional): the head is first divided by its root mean square
    (mean of squares + eps) and multiplied by the weight, in FP32 with the rotation. Gradients flow to q,
    k and the weights."""
    _head_tensor(q, 'q')
    _head_tensor(k, 'k')
    if q.shape[0] != k.shape[0]:
        raise ValueError('q and k must have the same number of tokens')
    positions = positions.unsqueeze(1) if positions.ndim == 1 else positions
    sections = (HEAD_DIM // 2,) if sections is None else tuple(sections)
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) != HEAD_DIM // 2:
        raise ValueError(f'sections must split {HEAD_DIM // 2} pairs over one to four axes, got {sections}')
    if (tuple(positions.shape) != (q.shape[0], len(sections)) or positions.dtype not in (torch.int32, torch.int64)
            or not positions.is_contiguous()):
        raise ValueError(f'positions must be contiguous int32 or int64 [tokens, {len(sections)}]')
    if (tuple(inv_freq.shape) != (HEAD_DIM // 2,) or inv_freq.dtype not in (torch.float32, torch.float64)
            or not inv_freq.is_contiguous()):
        raise ValueError(f'inv_freq must be a contiguous FP32 or FP64 vector of {HEAD_DIM // 2} frequencies')
    _epsilon(eps)
    _vector(q_weight, HEAD_DIM, 'q_weight')
    _vector(k_weight, HEAD_DIM, 'k_weight')
    _same_device(q, k, positions, inv_freq, q_weight, k_weight)
    rotate = _Rotary.apply if _through_autograd(q, k, q_weight, k_weight) else _rotate
    return rotate(q, k, q_weight, k_weight, positions, inv_freq, sections, bool(interleaved), float(eps))


# ----------------------------------------------------------------------------------------------
# Norm around a block
# ----------------------------------------------------------------------------------------------
def _normalise(x, branch, weight, gate, scale, shift, cu_seqlens, samples, eps, center, rstd=None, mean=None):
    tokens, hidden = x.shape
    y = torch.empty_like(x)
    r = None if branch is None else torch.empty_like(x)
    if tokens:
        args = _native.NORM_BYTES.pack(
            x.data_ptr(), _address(branch), _address(weight), _address(gate), _address(scale), _address(shift),
            _address(cu_seqlens), y.data_ptr(), _address(r), _address(rstd), _address(mean), 0, 0, 0, 0, 0, 0, 0, 0, 0,
            tokens, hidden, samples, center, 0, 0, eps)
        _launch(_native.lib().fga_norm_forward, args, x.device)
    return y, x if r is None else r


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, weight, gate, scale, shift, cu_seqlens, samples, eps, center):
        rstd = torch.empty(x.shape[0], device=x.device, dtype=torch.float32)
        mean = torch.empty_like(rstd) if center else None
        y, r = _normalise(x, branch, weight, gate, scale, shift, cu_seqlens, samples, eps, center, rstd, mean)
        ctx.set_materialize_grads(False)
        # r as it is returned has been rounded, which a centred norm may not bear; a gate keeps the branch anyway
        ctx.rebuild = branch is not None and (gate is not None or center)
        kept = (x, branch) if ctx.rebuild else (r, None)
        ctx.save_for_backward(*kept, weight, gate, scale, cu_seqlens, rstd, mean)
        ctx.owner, ctx.has_branch, ctx.has_shift = weight, branch is not None, shift is not None
        ctx.rule = (samples, eps, center)
        return y, r

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dr):
        base, branch, weight, gate, scale, cu_seqlens, rstd, mean = ctx.saved_tensors
        samples, eps, center = ctx.rule
        tokens, hidden = base.shape
        needs = ctx.needs_input_grad
        dy, dr = (None if g is None else _grad_rows(g, base.shape) for g in (dy, dr))
        dx = torch.empty_like(base)
        dbranch = torch.empty_like(base) if gate is not None else None
        target, accumulate = _weight_target(ctx.owner, needs[2])
        rows = [torch.empty((samples, hidden), device=base.device, dtype=base.dtype) if present and needed else None
                for present, needed in ((gate is not None, needs[3]), (scale is not None, needs[4]),
                                        (ctx.has_shift, needs[5]))]
        if tokens:
            lib = _native.lib()
            modulated = any(t is not None for t in rows)
            scratch = None
            if target is not None or modulated:
                scratch = _floats(lib.fga_norm_scratch_floats, base.device, tokens, hidden, samples, target is not None,
                                  modulated)
            x, r = (base.data_ptr(), 0) if ctx.rebuild else (0, base.data_ptr())
            args = _native.NORM_BYTES.pack(
                x, _address(branch), _address(weight), _address(gate), _address(scale), 0, _address(cu_seqlens), 0, r,
                rstd.data_ptr(), _address(mean), _address(dy), _address(dr), dx.data_ptr(), _address(dbranch),
                _address(target), *(_address(t) for t in rows), _address(scratch), tokens, hidden, samples, center,
                target is not None and target.dtype is torch.float32, accumulate, eps)
            _launch(lib.fga_norm_backward, args, base.device)
        else:
            for t in (*rows, None if accumulate else target):
                if t is not None:
                    t.zero_()
        if ctx.has_branch and gate is None:
            dbranch = dx
        return (dx, dbranch, _weight_result(ctx.owner, target, accumulate), *rows, None, None, None, None)


def residual_norm(x, branch=None, *, weight=None, gate=None, scale=None, shift=None, cu_seqlens=None, eps=1e-6,
                  center=False):
    """The step between two blocks: r = x + gate * branch, y = norm(r) * weight * (1 + scale) + shift, in
    one pass. Returns (y, r); without a branch r is x. All BF16; sums and statistics in FP32, y computed
    from the unrounded r. Where there is a gate or a centred norm, the backward pass computes r again from x
    and the branch, which it keeps; for an RMS norm without a gate it keeps r as it is returned, rounded.

    x, branch: contiguous [tokens, hidden], hidden a multiple of 8 up to 8192, at most 2^31 - 2^16 tokens.
    The norm divides by the root mean square of the row, after subtracting its mean with `center` (a layer
    norm). weight: [hidden]. gate, scale, shift: [samples, hidden], one row for each packed sequence of
    cu_seqlens (one sample, or [hidden], without it). With cu_seqlens, rows behind the last sequence have
    y = 0 and r = x, or x + branch where there is no gate, and pass dr through to what r is the sum of.
    Gradients flow to everything but cu_seqlens."""
    if x.ndim != 2 or x.dtype != torch.bfloat16 or not x.is_contiguous() or x.data_ptr() % 16:
        raise ValueError('x must be a contiguous, 16-byte aligned BF16 tensor [tokens, hidden]')
    tokens, hidden = x.shape
    if hidden < 8 or hidden % 8 or hidden > MAX_HIDDEN:
        raise ValueError(f'hidden must be a multiple of 8 up to {MAX_HIDDEN}, got {hidden}')
    if branch is not None and (branch.shape != x.shape or branch.dtype != x.dtype or not branch.is_contiguous()
                               or branch.data_ptr() % 16):
        raise ValueError('branch must be a contiguous, 16-byte aligned BF16 tensor of the shape of x')
    if gate is not None and branch is None:
        raise ValueError('gate scales the branch: pass one')
    _epsilon(eps)
    _vector(weight, hidden, 'weight')
    samples = 1
    if cu_seqlens is not None:
        _offsets(cu_seqlens)
        samples = cu_seqlens.shape[0] - 1
        if samples > 65535:
            raise ValueError('at most 65535 packed sequences')
    rows = []
    for label, t in (('gate', gate), ('scale', scale), ('shift', shift)):
        if t is not None and t.ndim == 1 and samples == 1:
            t = t.unsqueeze(0)
        if t is not None and (tuple(t.shape) != (samples, hidden) or t.dtype != torch.bfloat16
                              or not t.is_contiguous() or t.data_ptr() % 16):
            raise ValueError(f'{label} must be a contiguous, 16-byte aligned BF16 tensor [{samples}, {hidden}]')
        rows.append(t)
    _same_device(x, branch, weight, cu_seqlens, *rows)
    normalise = _ResidualNorm.apply if _through_autograd(x, branch, weight, *rows) else _normalise
    return normalise(x, branch, weight, *rows, cu_seqlens, samples, float(eps), bool(center))
