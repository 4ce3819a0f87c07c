"""ctypes binding of libfga.so, the C ABI declared in include/fga.h.

The library is built in-tree by build_native.py (nvcc, sm_100a only). There is no fallback: if the
shared object is missing or a call fails, an exception is raised.
"""
import ctypes
import os
import struct
from ctypes import c_char_p, c_float, c_int, c_int32, c_int64, c_size_t, c_uint64, c_void_p, POINTER

_HERE = os.path.dirname(os.path.realpath(__file__))
LIB_PATH = os.environ.get('FGA_LIB') or os.path.join(_HERE, 'libfga.so')  # FGA_LIB: another build of the same ABI

_lib = None


class FgaRotary(ctypes.Structure):
    """Arguments of fga_rotary_forward / fga_rotary_backward (include/fga.h)."""
    _fields_ = [('x', c_void_p * 2), ('x_token_stride', c_int64 * 2), ('x_head_stride', c_int64 * 2),
                ('dy', c_void_p * 2), ('out', c_void_p * 2), ('weight', c_void_p * 2), ('dweight', c_void_p * 2),
                ('positions', c_void_p), ('inv_freq', c_void_p), ('scratch', c_void_p), ('tokens', c_int64),
                ('heads', c_int32 * 2), ('positions_int64', c_int32), ('inv_freq_f64', c_int32), ('axes', c_int32),
                ('sections', c_int32 * 4), ('interleaved', c_int32), ('dweight_f32', c_int32 * 2),
                ('dweight_accumulate', c_int32 * 2), ('eps', c_float)]


class FgaNorm(ctypes.Structure):
    """Arguments of fga_norm_forward / fga_norm_backward (include/fga.h)."""
    _fields_ = ([(name, c_void_p) for name in (
        'x', 'branch', 'weight', 'gate', 'scale', 'shift', 'cu_seqlens', 'y', 'r', 'rstd', 'mean', 'dy', 'dr', 'dx',
        'dbranch', 'dweight', 'dgate', 'dscale', 'dshift', 'scratch')]
        + [('tokens', c_int64), ('hidden', c_int32), ('samples', c_int32), ('center', c_int32),
           ('dweight_f32', c_int32), ('dweight_accumulate', c_int32), ('eps', c_float)])


class FgaAttention(ctypes.Structure):
    """Arguments of fga_attention_forward / fga_attention_backward (include/fga.h)."""
    _fields_ = ([(name, c_void_p) for name in (
        'q', 'k', 'v', 'o', 'lse', 'd_o', 'dq', 'dk', 'dv', 'delta', 'cu_seqlens', 'status')]
        + [('timeout_ns', c_uint64), ('token_stride', c_int64 * 3), ('head_stride', c_int64 * 3), ('tokens', c_int64),
           ('heads', c_int32), ('kv_heads', c_int32), ('samples', c_int32), ('causal', c_int32), ('scale', c_float),
           ('host_status', c_void_p)])


# The same layouts as packed bytes, which a launch builds in a fraction of the time of a ctypes structure.
ROTARY_BYTES = struct.Struct('@2P2q2q2P2P2P2P3Pq2i3i4ii2i2if0q')
NORM_BYTES = struct.Struct('@20Pq5if0q')
ATTENTION_BYTES = struct.Struct('@12PQ6qq4ifP0q')
for _layout, _fields in ((ROTARY_BYTES, FgaRotary), (NORM_BYTES, FgaNorm), (ATTENTION_BYTES, FgaAttention)):
    assert _layout.size == ctypes.sizeof(_fields), _fields.__name__


class FgaError(RuntimeError):
    """A libfga entry point returned a non-zero status."""


def lib():
    """The loaded library (loads on first use; raises if it was never built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FgaError(f'{LIB_PATH} is missing: run `python build_native.py` (needs nvcc); '
                           'there is no CPU or PyTorch fallback for the fused kernels')
        _lib = ctypes.CDLL(LIB_PATH)
        _declare(_lib)
    return _lib


def _declare(l):
    vp, i, i64 = c_void_p, c_int, c_int64
    pp = POINTER(c_void_p)
    l.fga_version.restype = i
    l.fga_last_error.restype = c_char_p
    l.fga_sm_count.restype = i
    l.fga_launch_count.restype = c_uint64
    l.fga_symm_alloc.argtypes = [c_size_t, pp]
    l.fga_symm_export.argtypes = [vp, c_char_p]
    l.fga_symm_open.argtypes = [c_char_p, pp]
    l.fga_symm_close.argtypes = [vp]
    l.fga_symm_free.argtypes = [vp]
    l.fga_symm_vmm_size.argtypes = [c_size_t]
    l.fga_symm_vmm_size.restype = i64
    l.fga_symm_alloc_vmm.argtypes = [c_size_t, pp, POINTER(c_int)]
    l.fga_symm_open_vmm.argtypes = [i, c_size_t, pp]
    l.fga_symm_release_vmm.argtypes = [vp, c_size_t]
    l.fga_barrier.argtypes = [vp, vp, i, i, i, vp, i, vp, vp, c_uint64, vp]
    l.fga_gemm_push.argtypes = [vp, i, i, i, vp, i, vp, i, i, pp, i64, i, i, vp, c_uint64, vp]
    l.fga_gemm_recv.argtypes = [vp, i, i, vp, i, i, vp, vp, vp, vp, pp, i, i, i, i, i, i, vp, vp, vp,
                                c_uint64, vp]
    l.fga_gemm_push_gqa.argtypes = [vp, i, i, i, vp, vp, i, i, i, pp, i64, i, i, vp, c_uint64, vp]
    l.fga_gemm_recv_gqa.argtypes = [vp, i, vp, i, vp, vp, vp, vp, pp, i, i, i, i, i, i, i, i, vp, vp, c_uint64, vp]
    l.fga_gemm_local.argtypes = [vp, i, vp, i, i, i, i, i64, i64, vp, i64, i, i, vp, c_uint64, vp]
    l.fga_gemm_local_mx.argtypes = [vp, vp, i64, vp, vp, i64, i, i, i, vp, i64, i, i, vp, c_uint64, vp]
    l.fga_gemm_push_mx.argtypes = [vp, vp, i64, i, i, vp, vp, i64, vp, i, i, pp, i64, i, i, vp, c_uint64, vp]
    l.fga_gemm_recv_mx.argtypes = [vp, vp, vp, i, i, vp, vp, i64, i, i, vp, vp, vp, vp, pp, i, i, i, i, i, i,
                                   vp, vp, vp, c_uint64, vp]
    l.fga_gemm_push_gqa_mx.argtypes = [vp, vp, i64, i, i, vp, vp, i64, vp, i, i, i, pp, i64, i, i, vp, c_uint64, vp]
    l.fga_gemm_recv_gqa_mx.argtypes = [vp, vp, vp, i, vp, vp, i64, i, i, vp, vp, vp, vp, pp, i, i, i, i, i, i, i, i,
                                       vp, vp, c_uint64, vp]
    l.fga_copy_rank_rows.argtypes = [pp, pp, i, i, i64, i64, i, vp, i, i, vp]
    l.fga_bias_grad_scratch_floats.argtypes = [i64, i]
    l.fga_bias_grad_scratch_floats.restype = i64
    l.fga_bias_grad.argtypes = [vp, i64, i, vp, i, i, vp, vp]
    l.fga_bias_grad_static_capacity_floats.restype = i64
    l.fga_bias_grad_static.argtypes = [vp, i64, i, vp, i, i, vp]
    l.fga_mx_quantize.argtypes = [vp, i64, i, i64, i64, vp, vp, i64, i, vp]
    l.fga_rotary_forward.argtypes = [vp, vp]
    l.fga_rotary_backward.argtypes = [vp, vp]
    l.fga_rotary_scratch_floats.argtypes = [i64, i, i]
    l.fga_rotary_scratch_floats.restype = i64
    l.fga_norm_forward.argtypes = [vp, vp]
    l.fga_attention_forward.argtypes = [vp, vp]
    l.fga_attention_backward.argtypes = [vp, vp]
    l.fga_norm_backward.argtypes = [vp, vp]
    l.fga_norm_scratch_floats.argtypes = [i64, i, i, i, i]
    l.fga_norm_scratch_floats.restype = i64
    for name in ('fga_symm_alloc', 'fga_symm_export', 'fga_symm_open', 'fga_symm_close',
                 'fga_symm_free', 'fga_symm_alloc_vmm', 'fga_symm_open_vmm', 'fga_symm_release_vmm', 'fga_barrier', 'fga_gemm_push', 'fga_gemm_recv',
                 'fga_gemm_push_gqa', 'fga_gemm_recv_gqa',
                 'fga_gemm_local', 'fga_gemm_local_mx', 'fga_gemm_push_mx', 'fga_gemm_recv_mx',
                 'fga_gemm_push_gqa_mx', 'fga_gemm_recv_gqa_mx', 'fga_copy_rank_rows', 'fga_bias_grad', 'fga_bias_grad_static',
                 'fga_mx_quantize', 'fga_rotary_forward', 'fga_rotary_backward', 'fga_norm_forward',
                 'fga_norm_backward', 'fga_attention_forward', 'fga_attention_backward'):
        getattr(l, name).restype = i


EXPORTS = ('fga_version', 'fga_last_error', 'fga_sm_count', 'fga_launch_count', 'fga_symm_alloc', 'fga_symm_export',
           'fga_symm_open', 'fga_symm_close', 'fga_symm_free', 'fga_symm_vmm_size', 'fga_symm_alloc_vmm',
           'fga_symm_open_vmm', 'fga_symm_release_vmm', 'fga_barrier', 'fga_gemm_push',
           'fga_gemm_recv', 'fga_gemm_push_gqa', 'fga_gemm_recv_gqa', 'fga_gemm_local', 'fga_gemm_local_mx', 'fga_gemm_push_mx', 'fga_gemm_recv_mx',
           'fga_gemm_push_gqa_mx', 'fga_gemm_recv_gqa_mx', 'fga_copy_rank_rows', 'fga_bias_grad_scratch_floats',
           'fga_bias_grad', 'fga_bias_grad_static_capacity_floats', 'fga_bias_grad_static', 'fga_mx_quantize',
           'fga_rotary_forward', 'fga_rotary_backward', 'fga_rotary_scratch_floats', 'fga_norm_forward',
           'fga_norm_backward', 'fga_norm_scratch_floats', 'fga_attention_forward',
           'fga_attention_backward')


def check(rc, exc=FgaError):
    """Raise `exc` with the library's message when an entry point failed."""
    if rc != 0:
        message = lib().fga_last_error().decode(errors='replace')
        if rc == -1:
            raise ValueError(message)
        raise exc(f'libfga error {rc}: {message}')


def ptr_array(addresses):
    """A C array of void* from integer addresses."""
    arr = (c_void_p * len(addresses))(*addresses)
    return arr


DEVICE_ERRORS = {
    1: 'group barrier timed out: a CP peer never published its epoch',
    2: 'receive GEMM timed out: a row block never collected all peer arrivals',
    3: 'GEMM pipeline barrier timed out',
    4: 'receive-side quantizer timed out',
}
