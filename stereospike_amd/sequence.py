"""Sequence operators on the C-ABI of include/ss_sequence.h.

    leaky_attention(q_seq, k_seq, v_seq, log_decay, ...)   a leaky matrix state per head over a whole [T, B, ...] sequence (differentiable)
    leaky_attention_step(q, k, v, log_decay, state, ...)   the same, one time step, the state updated in place (serving)
    add_rms_norm(x, weight, residual)                      residual addition + root-mean-square norm (differentiable)
    add_rms_norm_int8(x, weight, residual)                 the same, handed on as 8-bit codes with a scale per row
    dequantize_int8 / quantize_channels                    codes -> values; a weight matrix -> codes with a scale per output channel
    int8_linear(codes, scales, weight, weight_scale)       8-bit integer product, exact sums

They stand beside the fused neuron layers of `fused.py`: a leaky integrator whose state is a matrix and is read by a query, the gain / skip-add epilogue of a
layer without spikes, and the product of small-integer activations (spike counts are 8-bit codes of scale 1) with a weight.  Like those they need the HIP
library and HIP tensors, launch on torch's current stream of the tensors' device, allocate their workspaces from torch's caching allocator and may be recorded
into a HIP graph; there is no eager fallback, and tracers (torch.jit.trace, torch.fx) and
forward-mode derivatives are refused.  A backward pass that is itself captured needs leaves whose gradients no live eager graph reaches
(engine.GraphedTrainer shows how).  Gradients are first derivatives: differentiating them again raises.
Nothing is cast: torch.autocast does not reach these functions (cast a 16-bit x and its residual to one type), and log_decay, norm weights and scales stay fp32
(net.half() and the like turn the layers' into a type that is refused; convert the activations instead).

Calls go straight to the library (csrc/ss_seq_torch.cpp), which checks, allocates and launches; it hands a call with unfit operands back, and the functions
here then raise the SSNeuronError that names the operand.
"""
from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from . import _seqlib
from ._lib import SSNeuronError, _require_hip

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _operand(t, name, dev, dtype, shape):
    """Raises unless t is a tensor of this device, type and shape."""
    _require_hip(t, name)
    if t.device != dev:
        raise SSNeuronError(f'{name} is on {t.device}, expected {dev}')
    if t.dtype != dtype:
        raise SSNeuronError(f'{name}: expected {dtype}, got {t.dtype}')
    if tuple(t.shape) != tuple(shape):
        raise SSNeuronError(f'{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}')


def _refuse_recording(name, args):
    """Raises where a tracer records or an operand has a forward-mode tangent: the trace would hold no launch, the outputs no tangent."""
    if torch.jit.is_tracing() or get_proxy_mode() is not None:
        raise SSNeuronError(f'{name} cannot be traced: its kernels are launched outside of torch\'s operators (a HIP graph records them)')
    if any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in args):
        raise SSNeuronError(f'{name} has no forward-mode derivative')


def _call(name, refuse, *args):
    """The library's answer, or the error that `refuse` raises for operands it does not take."""
    try:
        r = getattr(_seqlib.ops(), name)(*args)
    except TypeError:
        r = None                                           # something that is no tensor
    if r is None:
        _refuse_recording(name, args)
        refuse()
        raise SSNeuronError(f'{name}: operands refused')
    return r


# ----------------------------------------------------------------------------------------------------------------------------------------------------------
# leaky attention
# ----------------------------------------------------------------------------------------------------------------------------------------------------------
def _refuse_attention(q, k, v, log_decay, state, lengths, lead):
    _require_hip(q, 'q')
    dt, dev = q.dtype, q.device
    if dt not in _FLOATS:
        raise SSNeuronError(f'q: expected float32, float16 or bfloat16, got {dt}')
    for t, name in ((k, 'k'), (v, 'v')):
        _require_hip(t, name)
    if q.dim() != lead + 2 or k.dim() != lead + 2 or v.dim() != lead + 2:
        raise SSNeuronError(f'q, k, v: expected {lead + 2} axes ([{"T, " if lead == 2 else ""}B, heads, D]), got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}')
    B, H, Dk = q.shape[-3:]
    Hk, Dv = v.shape[-2:]
    _operand(k, 'k', dev, dt, (*q.shape[:lead], Hk, Dk))
    _operand(v, 'v', dev, dt, (*q.shape[:lead], Hk, Dv))
    if H < 1 or Hk < 1 or H % Hk:
        raise SSNeuronError(f'{H} query heads cannot share {Hk} key / value heads')
    if not (1 <= Dk <= _seqlib.MAX_HEAD_DIM and 1 <= Dv <= _seqlib.MAX_HEAD_DIM):
        raise SSNeuronError(f'head sizes {Dk} and {Dv}: 1 .. {_seqlib.MAX_HEAD_DIM} are implemented')
    if B * H > _seqlib.MAX_STATES:
        raise SSNeuronError(f'B * heads = {B * H}: at most {_seqlib.MAX_STATES} states in one call')
    if lead == 2 and q.shape[0] > _seqlib.MAX_STEPS:
        raise SSNeuronError(f'{q.shape[0]} steps: at most {_seqlib.MAX_STEPS} in one call')
    _operand(log_decay, 'log_decay', dev, torch.float32, (H,))
    if lead == 2 and log_decay.requires_grad and torch.is_grad_enabled():
        raise SSNeuronError('log_decay: the decay of a head is a constant here (as tau of a LIFNode, unlike a ParametricLIFNode\'s); it has no gradient — pass log_decay.detach()')
    if state is not None:
        _operand(state, 'state', dev, torch.float32, (B, H, Dk, Dv))
    if lengths is not None:
        _operand(lengths, 'lengths', dev, torch.int32, (B,))
    if lead == 1:
        _operand(state, 'state', dev, torch.float32, (B, H, Dk, Dv))
        if not state.is_contiguous():
            raise SSNeuronError('state: tensor must be contiguous (it is updated in place)')
        if state.requires_grad:
            raise SSNeuronError('state: it is updated in place, outside of any graph, and requires a gradient — pass state.detach().clone()')
        if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, log_decay)):
            raise SSNeuronError('leaky_attention_step has no gradient: call it under torch.no_grad(), or leaky_attention with T = 1')


def leaky_attention(q_seq: torch.Tensor, k_seq: torch.Tensor, v_seq: torch.Tensor, log_decay: torch.Tensor, scale: Optional[float] = None,
                    state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None, return_state: bool = False):
    """Linear attention with a decay per head over a sequence:

        S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T,     o_t = scale * q_t^T S_t

    q_seq [T, B, H, Dk], k_seq [T, B, Hk, Dk], v_seq [T, B, Hk, Dv] in one of float32 / float16 / bfloat16 with any strides (a last axis that is not
    contiguous is copied); H is a multiple of Hk and query head h reads key / value head h // (H // Hk).  Dk, Dv <= 256.  log_decay fp32 [H], <= 0: the log of
    lambda (1 - 1 / tau of a leaky integrator; -inf forgets at once); it has no gradient.  scale: Dk ** -0.5 by default.
    state: fp32 [B, H, Dk, Dv], S before the first step (None: zero).  lengths: int32 [B] on the device, the valid steps of each stream (clamped to 0 .. T);
    rows behind them are not read, their outputs and gradients are zero.
    A NaN or an infinity reaches its own step's output and, through the state, its head's later steps (a value's: in its column), never an earlier step, another
    stream or another head; the state's entries that held it are infinite or NaN from there on.
    Returns o_seq [T, B, H, Dv]; with return_state also the state after the last valid step (fp32).  States, sums and decays are fp32, outputs and gradients are
    rounded once.  Gradients: q, k, v and state, from both results."""
    out, last = _call('leaky_attention', lambda: _refuse_attention(q_seq, k_seq, v_seq, log_decay, state, lengths, 2), q_seq, k_seq, v_seq, log_decay, scale, state, lengths)
    return (out, last) if return_state else out


def leaky_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor,
                         scale: Optional[float] = None) -> torch.Tensor:
    """One time step of `leaky_attention`: q [B, H, Dk], k [B, Hk, Dk], v [B, Hk, Dv]; `state` (fp32 [B, H, Dk, Dv], contiguous) is updated IN PLACE.
    Returns o [B, H, Dv].  No gradients: a state that requires one, or q, k, v that do while gradients are enabled, are refused (use leaky_attention with T = 1)."""
    return _call('leaky_attention_step', lambda: _refuse_attention(q, k, v, log_decay, state, None, 1), q, k, v, log_decay, state, scale)


# ----------------------------------------------------------------------------------------------------------------------------------------------------------
# add + root-mean-square norm
# ----------------------------------------------------------------------------------------------------------------------------------------------------------
def _refuse_norm(x, weight, residual, eps):
    _require_hip(x, 'x')
    if x.dtype not in _FLOATS:
        raise SSNeuronError(f'x: expected float32, float16 or bfloat16, got {x.dtype}')
    if x.dim() < 1 or not 1 <= x.shape[-1] <= _seqlib.MAX_NORM_WIDTH:
        raise SSNeuronError(f'x: shape {tuple(x.shape)}; rows of 1 .. {_seqlib.MAX_NORM_WIDTH} values are implemented')
    _operand(weight, 'weight', x.device, torch.float32, x.shape[-1:])
    if residual is not None:
        _operand(residual, 'residual', x.device, x.dtype, x.shape)
    if not float(eps) >= 0.:
        raise SSNeuronError(f'eps: expected a number >= 0, got {eps}')


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """h = x + residual, kept in x's type;  y = h / sqrt(mean(h^2) + eps) * weight over the last axis.  Returns (y, h); without a residual h is x itself.

    x, residual: [..., C] in float32 / float16 / bfloat16, C <= 16384; weight fp32 [C].  Sums are fp32; y is rounded once.  Gradients: x, residual, weight."""
    return _call('add_rms_norm', lambda: _refuse_norm(x, weight, residual, eps), x, weight, residual, eps)


def add_rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """`add_rms_norm` handed on in 8 bits: returns (codes int8 [..., C], scales fp32 [...], h) with codes * scales the norm; the largest value of a row has the
    code +-127, ties go to the even code.  A row of zeros has scale 0; a row with a NaN or an infinity, its own or
    the weight's, has codes 0 and scale NaN.  Codes and scales have no gradient (nor has the weight); h has that of the addition."""
    return _call('add_rms_norm_int8', lambda: _refuse_norm(x, weight, residual, eps), x, weight, residual, eps)


def dequantize_int8(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that 8-bit codes [..., C] with a scale per row [...] stand for, codes * scales rounded once to dtype.  No gradients."""
    def refuse():
        _require_hip(codes, 'codes')
        if codes.dim() < 1 or codes.shape[-1] < 1:
            raise SSNeuronError(f'codes: expected [..., C], got {tuple(codes.shape)}')
        _operand(codes, 'codes', codes.device, torch.int8, codes.shape)
        _operand(scales, 'scales', codes.device, torch.float32, codes.shape[:-1])
        if dtype not in _FLOATS:
            raise SSNeuronError(f'dtype: expected float32, float16 or bfloat16, got {dtype}')
        if torch.is_grad_enabled() and scales.requires_grad:
            raise SSNeuronError('dequantize_int8 has no gradient: call it under torch.no_grad() or detach scales')
    return _call('dequantize_int8', refuse, codes, scales, dtype)


# ----------------------------------------------------------------------------------------------------------------------------------------------------------
# 8-bit integer product
# ----------------------------------------------------------------------------------------------------------------------------------------------------------
@torch.no_grad()
def quantize_channels(weight: torch.Tensor):
    """A weight matrix [N, K] as 8-bit codes with a scale per output channel: (codes int8 [N, K], scales fp32 [N]), |codes| <= 127.  Done once, when a layer
    is built; runs on any device."""
    if weight.dim() != 2 or not weight.is_floating_point():
        raise SSNeuronError(f'weight: expected a floating matrix [N, K], got {weight.dtype} {tuple(weight.shape)}')
    w = weight.detach().double()
    scale = (w.abs().amax(1) / 127.).float()
    codes = torch.round(w / scale.double().clamp_min(1e-300)[:, None]).clamp_(-127, 127)
    return codes.to(torch.int8), scale


def int8_linear(codes: torch.Tensor, scales: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """out[..., n] = (sum_k codes[..., k] * weight[n, k]) * scales[...] * weight_scale[n] + bias[n], the sum exact in 32-bit integers.

    codes int8 [..., K] (spike counts are codes of scale 1), scales fp32 [...], weight int8 [N, K], weight_scale fp32 [N], bias fp32 [N]; K < 131072, at most 2^27 rows and channels, less than 2^24
    tiles of 128 x 128 outputs.  Scaled in
    fp32, rounded once to out_dtype (float32 / float16 / bfloat16).  No gradients."""
    def refuse():
        _require_hip(codes, 'codes')
        _require_hip(weight, 'weight')
        if codes.dim() < 1 or weight.dim() != 2:
            raise SSNeuronError(f'codes [..., K], weight [N, K]: got {tuple(codes.shape)}, {tuple(weight.shape)}')
        dev, (N, K) = codes.device, weight.shape
        _operand(codes, 'codes', dev, torch.int8, codes.shape[:-1] + (K,))
        _operand(scales, 'scales', dev, torch.float32, codes.shape[:-1])
        _operand(weight, 'weight', dev, torch.int8, (N, K))
        _operand(weight_scale, 'weight_scale', dev, torch.float32, (N,))
        if bias is not None:
            _operand(bias, 'bias', dev, torch.float32, (N,))
        if not 1 <= K <= _seqlib.MAX_INT8_K or N < 1:
            raise SSNeuronError(f'weight: [N, K] = [{N}, {K}]; N >= 1 and 1 <= K <= {_seqlib.MAX_INT8_K} (sums stay within 32 bits) are implemented')
        if max(N, codes.numel() // K) > _seqlib.MAX_SIDE:
            raise SSNeuronError(f'{codes.numel() // K} rows, {N} channels: at most {_seqlib.MAX_SIDE} of each')
        if -(-(codes.numel() // K) // 128) * -(-N // 128) >= _seqlib.MAX_TILES:
            raise SSNeuronError(f'{codes.numel() // K} rows by {N} channels: less than {_seqlib.MAX_TILES} tiles of 128 x 128 outputs in one call')
        if out_dtype not in _FLOATS:
            raise SSNeuronError(f'out_dtype: expected float32, float16 or bfloat16, got {out_dtype}')
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (scales, weight_scale, bias)):
            raise SSNeuronError('int8_linear has no gradient: call it under torch.no_grad() or detach scales and bias')
    return _call('int8_linear', refuse, codes, scales, weight, weight_scale, bias, out_dtype)
