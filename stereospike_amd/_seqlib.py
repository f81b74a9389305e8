"""ctypes binding of libss_sequence.so (include/ss_sequence.h): the sequence operators' only way to their kernels.

As with the neuron library there is no fallback: a missing library, a CPU tensor or an operand of another type raises SSNeuronError.
"""
import ctypes as C
import os

import torch  # before the CDLL, so that one HIP runtime is shared

from ._lib import SSNeuronError, _check

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, 'lib', 'libss_sequence.so')
ABI_VERSION = 1
DT_CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_HEAD_DIM = 256
MAX_NORM_WIDTH = 16384
MAX_INT8_K = 131071

_lib = None


class LeakyDesc(C.Structure):
    """struct ss_seq_leaky_desc (include/ss_sequence.h)."""
    _fields_ = ([('size', C.c_uint), ('dtype', C.c_int), ('out_dtype', C.c_int)] + [(n, C.c_int) for n in ('T', 'B', 'H', 'DA', 'DC', 'reverse')] +
                [('b_scale', C.c_float), ('o_scale', C.c_float)] + [(n, C.c_void_p) for n in ('a', 'b', 'c', 'out')] +
                [(f'{n}_{s}', C.c_longlong) for n in 'abco' for s in 'tbh'] + [(f'{n}_group', C.c_int) for n in 'abc'] +
                [('log_decay', C.c_void_p), ('lengths', C.c_void_p), ('s_in', C.c_void_p), ('s_out', C.c_void_p)] +
                [(n, C.c_int) for n in ('s_in_row', 's_in_col', 's_out_row', 's_out_col')] + [('ws', C.c_void_p)])


class LeakyBwdDesc(C.Structure):
    """struct ss_seq_leaky_bwd_desc (include/ss_sequence.h)."""
    _fields_ = ([('size', C.c_uint)] + [(n, C.c_int) for n in ('dtype', 'T', 'B', 'H', 'Hk', 'Dk', 'Dv')] + [('scale', C.c_float)] +
                [(n, C.c_void_p) for n in 'qkvg'] + [(f'{n}_{s}', C.c_longlong) for n in 'qkvg' for s in 'tbh'] +
                [(n, C.c_void_p) for n in ('g_q', 'g_k', 'g_v', 'log_decay', 'lengths', 's_in', 'g_last', 'g_s', 'states', 'ws')])


EXPORTS = ('ss_seq_abi_version', 'ss_seq_leaky_ws_floats', 'ss_seq_leaky', 'ss_seq_leaky_bwd_ws_floats', 'ss_seq_leaky_bwd', 'ss_seq_group_sum', 'ss_seq_rms_norm_fwd', 'ss_seq_rms_norm_ws_floats',
           'ss_seq_rms_norm_bwd', 'ss_seq_rms_norm_int8', 'ss_seq_dequant_int8', 'ss_seq_int8_linear_ws_ints', 'ss_seq_int8_linear')


def lib():
    """Load (once) and return the library.  Raises loudly when it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise SSNeuronError(f'{LIB_PATH} not found: the HIP extension is not built.  Run `python -c "import __graft_entry__ as g; g.build()"` or '
                            f'`make -C stereospike_amd/csrc` (hipcc --offload-arch=gfx950).  There is no CPU fallback.')
    L = C.CDLL(LIB_PATH)
    p, i32, i64, f32, desc, bdesc = C.c_void_p, C.c_int, C.c_longlong, C.c_float, C.POINTER(LeakyDesc), C.POINTER(LeakyBwdDesc)
    for name, res, args in (('ss_seq_abi_version', i32, []), ('ss_seq_leaky_ws_floats', i64, [desc]), ('ss_seq_leaky', i32, [desc, p]),
                            ('ss_seq_leaky_bwd_ws_floats', i64, [bdesc]), ('ss_seq_leaky_bwd', i32, [bdesc, p]),
                            ('ss_seq_group_sum', i32, [p, p, i64, i32, i32, i32, p]),
                            ('ss_seq_rms_norm_fwd', i32, [p, i64, p, i64, p, p, p, p, i64, i32, f32, i32, p]),
                            ('ss_seq_rms_norm_ws_floats', i64, [i64, i32, i32]),
                            ('ss_seq_rms_norm_bwd', i32, [p, p, p, p, p, p, p, p, i64, i32, i32, p]),
                            ('ss_seq_rms_norm_int8', i32, [p, i64, p, i64, p, p, p, p, i64, i32, f32, i32, p]),
                            ('ss_seq_dequant_int8', i32, [p, p, p, i64, i32, i32, p]),
                            ('ss_seq_int8_linear_ws_ints', i64, [p, i64, p, i64, i64, i32, i32]),
                            ('ss_seq_int8_linear', i32, [p, i64, p, p, i64, p, p, p, i64, i32, i32, i32, p, p])):
        f = getattr(L, name)
        f.restype, f.argtypes = res, args
    if L.ss_seq_abi_version() != ABI_VERSION:
        raise SSNeuronError(f'libss_sequence.so ABI {L.ss_seq_abi_version()} != expected {ABI_VERSION}; rebuild')
    _lib = L
    return _lib


def _p(t):
    return None if t is None else t.data_ptr()


_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)
_device = getattr(torch._C, '_cuda_getDevice', None)


def _call(name, dev, *args):
    """One entry point on torch's current stream of `dev`, with that device current.  A context manager per launch costs as much as the launch, so it is
    entered only for another device than the current one."""
    f = getattr(_lib or lib(), name)
    if _device is not None and _device() == dev.index:
        rc = f(*args, _raw_stream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = f(*args, torch.cuda.current_stream(dev).cuda_stream)
    if rc:
        _check(rc, name)


def leaky(q, k, v, out, log_decay, scale, lengths=None, s_in=None, s_out=None):
    """The forward map: q, k, v, out [T, B, heads, D] views with a contiguous last axis ([B, heads, D]: one step); states [B, H, Dk, Dv] contiguous.
    Returns the workspace, which holds the states between segments (None where there are none)."""
    sq, sk, sv, so = q.stride(), k.stride(), v.stride(), out.stride()
    if len(so) == 3:
        T, (B, H, Dv) = 1, out.shape
        sq, sk, sv, so = (0, *sq), (0, *sk), (0, *sv), (0, *so)
    else:
        T, B, H, Dv = out.shape
    dt, group = DT_CODE[q.dtype], H // k.shape[-2]
    d = LeakyDesc(_DESC_SIZE, dt, dt, T, B, H, q.shape[-1], Dv, 0, 1.0, scale, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                  sq[0], sq[1], sq[2], sk[0], sk[1], sk[2], sv[0], sv[1], sv[2], so[0], so[1], so[2], 1, group, group,
                  log_decay.data_ptr(), _p(lengths), _p(s_in), _p(s_out), Dv, 1, Dv, 1)
    ref = C.byref(d)
    ws = None
    if T > 1:
        n = (_lib or lib()).ss_seq_leaky_ws_floats(ref)
        if n:
            ws = torch.empty(n, dtype=torch.float32, device=q.device)
            d.ws = ws.data_ptr()
    _call('ss_seq_leaky', q.device, ref)
    return ws


def leaky_bwd(q, k, v, g, g_q, g_k, g_v, log_decay, scale, lengths, s_in, g_last, g_s, states):
    """Gradients of `leaky` (None: not wanted); g_q, g_k, g_v contiguous."""
    T, B, H, Dk = q.shape
    d = LeakyBwdDesc(_BWD_SIZE, DT_CODE[q.dtype], T, B, H, k.shape[2], Dk, v.shape[3], scale, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(),
                     *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *g.stride()[:3], _p(g_q), _p(g_k), _p(g_v), log_decay.data_ptr(), _p(lengths),
                     _p(s_in), _p(g_last), _p(g_s), _p(states))
    ref = C.byref(d)
    n = (_lib or lib()).ss_seq_leaky_bwd_ws_floats(ref)
    ws = torch.empty(n, dtype=torch.float32, device=q.device) if n else None
    d.ws = _p(ws)
    _call('ss_seq_leaky_bwd', q.device, ref)


_DESC_SIZE, _BWD_SIZE = C.sizeof(LeakyDesc), C.sizeof(LeakyBwdDesc)


def rms_norm_fwd(x, residual, weight, y, total, rstd, eps):
    """x, residual: [rows, C] with a contiguous last axis; y, total contiguous; rstd fp32 [rows] or None."""
    rows, C_ = x.shape
    _call('ss_seq_rms_norm_fwd', x.device, x.data_ptr(), x.stride(0), _p(residual), 0 if residual is None else residual.stride(0), weight.data_ptr(), y.data_ptr(),
          _p(total), _p(rstd), rows, C_, eps, DT_CODE[x.dtype])


def rms_norm_bwd(g_y, g_sum, h, weight, rstd, g_h, g_w):
    rows, C_ = h.shape
    dt = DT_CODE[h.dtype]
    ws = None if g_w is None else torch.empty((_lib or lib()).ss_seq_rms_norm_ws_floats(rows, C_, dt), dtype=torch.float32, device=h.device)
    _call('ss_seq_rms_norm_bwd', h.device, _p(g_y), _p(g_sum), h.data_ptr(), weight.data_ptr(), rstd.data_ptr(), g_h.data_ptr(), _p(g_w), _p(ws), rows, C_, dt)


def rms_norm_int8(x, residual, weight, codes, scales, total, eps):
    rows, C_ = x.shape
    _call('ss_seq_rms_norm_int8', x.device, x.data_ptr(), x.stride(0), _p(residual), 0 if residual is None else residual.stride(0), weight.data_ptr(),
          codes.data_ptr(), scales.data_ptr(), _p(total), rows, C_, eps, DT_CODE[x.dtype])


def dequant_int8(codes, scales, out):
    """codes, out contiguous, rows of the last axis; a scale for each row."""
    C_ = codes.shape[-1]
    _call('ss_seq_dequant_int8', codes.device, codes.data_ptr(), scales.data_ptr(), out.data_ptr(), codes.numel() // C_, C_, DT_CODE[out.dtype])


def int8_linear(a, a_scale, w, w_scale, bias, out):
    """a [M, K], w [N, K] int8 with contiguous last axes; out [M, N] contiguous."""
    (M, K), N = a.shape, w.shape[0]
    pa, la, pw, lw = a.data_ptr(), a.stride(0), w.data_ptr(), w.stride(0)
    n = (_lib or lib()).ss_seq_int8_linear_ws_ints(pa, la, pw, lw, M, N, K)
    ws = torch.empty(n, dtype=torch.int32, device=a.device) if n else None
    _call('ss_seq_int8_linear', a.device, pa, la, a_scale.data_ptr(), pw, lw, w_scale.data_ptr(), _p(bias), out.data_ptr(), M, N, K, DT_CODE[out.dtype], _p(ws))
