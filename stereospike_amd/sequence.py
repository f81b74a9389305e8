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
into a HIP graph; there is no eager fallback.  A backward pass that is itself captured needs leaves whose gradients no live eager graph reaches
(engine.GraphedTrainer shows how).
"""
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _seqlib
from ._lib import SSNeuronError, _require_hip

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _operand(t, name, dev, dtype, shape):
    """A tensor of this device, type and shape, or the reason why not."""
    if isinstance(t, torch.Tensor) and t.device == dev and t.dtype is dtype and t.shape == shape:
        return
    _require_hip(t, name)
    if t.device != dev:
        raise SSNeuronError(f'{name} is on {t.device}, expected {dev}')
    if t.dtype != dtype:
        raise SSNeuronError(f'{name}: expected {dtype}, got {t.dtype}')
    raise SSNeuronError(f'{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}')


def _last_contiguous(t):
    return t if t.stride(-1) == 1 or t.is_contiguous() else t.contiguous()


# ----------------------------------------------------------------------------------------------------------------------------------------------------------
# leaky attention
# ----------------------------------------------------------------------------------------------------------------------------------------------------------
def _attention_operands(q, k, v, log_decay, state, lengths, lead):
    _require_hip(q, 'q')
    dt, dev = q.dtype, q.device
    if dt not in _FLOATS:
        raise SSNeuronError(f'q: expected float32, float16 or bfloat16, got {dt}')
    if q.dim() != lead + 2 or k.dim() != lead + 2 or v.dim() != lead + 2:
        raise SSNeuronError(f'q, k, v: expected {lead + 2} axes ([{"T, " if lead == 2 else ""}B, heads, D]), got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}')
    qs, vs = q.shape, v.shape
    B, H, Dk = qs[-3:]
    Hk, Dv = vs[-2:]
    head = qs[:lead]
    _operand(k, 'k', dev, dt, (*head, Hk, Dk))
    _operand(v, 'v', dev, dt, (*head, Hk, Dv))
    if H < 1 or Hk < 1 or H % Hk:
        raise SSNeuronError(f'{H} query heads cannot share {Hk} key / value heads')
    if not (1 <= Dk <= _seqlib.MAX_HEAD_DIM and 1 <= Dv <= _seqlib.MAX_HEAD_DIM):
        raise SSNeuronError(f'head sizes {Dk} and {Dv}: 1 .. {_seqlib.MAX_HEAD_DIM} are implemented')
    if B * H > 65535:
        raise SSNeuronError(f'B * heads = {B * H}: at most 65535 states in one call')
    _operand(log_decay, 'log_decay', dev, torch.float32, (H,))
    if state is not None:
        _operand(state, 'state', dev, torch.float32, (B, H, Dk, Dv))
    if lengths is not None:
        _operand(lengths, 'lengths', dev, torch.int32, (B,))
    return B, H, Hk, Dk, Dv


class _LeakyAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, state, log_decay, scale, lengths):
        ctx.set_materialize_grads(False)
        q, k, v = _last_contiguous(q), _last_contiguous(k), _last_contiguous(v)
        B, H, Dk = q.shape[1:]
        Dv = v.shape[3]
        if state is not None:
            state = state.contiguous()
        out = torch.empty((q.shape[0], B, H, Dv), dtype=q.dtype, device=q.device)
        last = torch.empty((B, H, Dk, Dv), dtype=torch.float32, device=q.device)
        states = _seqlib.leaky(q, k, v, out, log_decay, scale, lengths, state, last)
        if any(ctx.needs_input_grad):
            ctx.save_for_backward(q, k, v, state, log_decay, lengths, states)
            ctx.scale = scale
        return out, last

    @staticmethod
    def backward(ctx, g, g_last):
        return _attention_grads_once(ctx, g, g_last) if torch.is_grad_enabled() else _attention_grads(ctx, g, g_last)


def _attention_grads(ctx, g, g_last):
    q, k, v, state, log_decay, lengths, states = ctx.saved_tensors
    need_q, need_k, need_v, need_s = ctx.needs_input_grad[:4]
    g = torch.zeros((*q.shape[:3], v.shape[3]), dtype=q.dtype, device=q.device) if g is None else _last_contiguous(g)
    if g_last is not None:
        g_last = g_last.contiguous()
    g_q, g_k, g_v = (torch.empty(t.shape, dtype=t.dtype, device=t.device) if need else None for t, need in ((q, need_q), (k, need_k), (v, need_v or need_s)))
    g_s = torch.empty(state.shape, dtype=torch.float32, device=q.device) if need_s else None
    _seqlib.leaky_bwd(q, k, v, g, g_q, g_k, g_v, log_decay, ctx.scale, lengths, state, g_last, g_s, states)
    return g_q, g_k, g_v if need_v else None, g_s, None, None, None


_attention_grads_once = once_differentiable(_attention_grads)        # under create_graph: a second derivative is refused, not silently zero


def leaky_attention(q_seq: torch.Tensor, k_seq: torch.Tensor, v_seq: torch.Tensor, log_decay: torch.Tensor, scale: Optional[float] = None,
                    state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None, return_state: bool = False):
    """Linear attention with a decay per head over a sequence:

        S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T,     o_t = scale * q_t^T S_t

    q_seq [T, B, H, Dk], k_seq [T, B, Hk, Dk], v_seq [T, B, Hk, Dv] in one of float32 / float16 / bfloat16 with any strides (a last axis that is not
    contiguous is copied); H is a multiple of Hk and query head h reads key / value head h // (H // Hk).  Dk, Dv <= 256.  log_decay fp32 [H], <= 0: the log of
    lambda (1 - 1 / tau of a leaky integrator; -inf forgets at once).  scale: Dk ** -0.5 by default.
    state: fp32 [B, H, Dk, Dv], S before the first step (None: zero).  lengths: int32 [B] on the device, the valid steps of each stream (clamped to 0 .. T);
    rows behind them are not read, their outputs and gradients are zero.
    Returns o_seq [T, B, H, Dv]; with return_state also the state after the last valid step (fp32).  States, sums and decays are fp32.  Gradients: q, k, v and
    state, from both results."""
    B, H, Hk, Dk, Dv = _attention_operands(q_seq, k_seq, v_seq, log_decay, state, lengths, 2)
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise SSNeuronError('log_decay: the decay of a head is a constant of the layer (as tau of a LIFNode); it has no gradient — pass log_decay.detach()')
    scale = Dk ** -0.5 if scale is None else float(scale)
    T = q_seq.shape[0]
    if T == 0 or B == 0:                                   # no step: nothing to launch
        out = q_seq.new_zeros((T, B, H, Dv))
        last = torch.zeros((B, H, Dk, Dv), dtype=torch.float32, device=q_seq.device) if state is None else state.clone()
    else:
        out, last = _LeakyAttention.apply(q_seq, k_seq, v_seq, state, log_decay.contiguous(), scale, None if lengths is None else lengths.contiguous())
    return (out, last) if return_state else out


def leaky_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor,
                         scale: Optional[float] = None) -> torch.Tensor:
    """One time step of `leaky_attention`: q [B, H, Dk], k [B, Hk, Dk], v [B, Hk, Dv]; `state` (fp32 [B, H, Dk, Dv], contiguous) is updated IN PLACE.
    Returns o [B, H, Dv].  No gradients (use leaky_attention with T = 1)."""
    B, H, Hk, Dk, Dv = _attention_operands(q, k, v, log_decay, state, None, 1)
    if not state.is_contiguous():
        raise SSNeuronError('state: tensor must be contiguous (it is updated in place)')
    out = torch.empty((B, H, Dv), dtype=q.dtype, device=q.device)
    if B:
        _seqlib.leaky(_last_contiguous(q), _last_contiguous(k), _last_contiguous(v), out, log_decay.contiguous(), Dk ** -0.5 if scale is None else float(scale),
                      s_in=state, s_out=state)
        if not state.is_inference():
            torch.autograd.graph.increment_version(state)  # an autograd graph that saved this state must notice
    return out


# ----------------------------------------------------------------------------------------------------------------------------------------------------------
# add + root-mean-square norm
# ----------------------------------------------------------------------------------------------------------------------------------------------------------
def _norm_operands(x, weight, residual, eps):
    _require_hip(x, 'x')
    shape = x.shape
    if x.dtype not in _FLOATS:
        raise SSNeuronError(f'x: expected float32, float16 or bfloat16, got {x.dtype}')
    if len(shape) < 1 or not 1 <= shape[-1] <= _seqlib.MAX_NORM_WIDTH:
        raise SSNeuronError(f'x: shape {tuple(shape)}; rows of 1 .. {_seqlib.MAX_NORM_WIDTH} values are implemented')
    _operand(weight, 'weight', x.device, torch.float32, shape[-1:])
    if residual is not None:
        _operand(residual, 'residual', x.device, x.dtype, shape)
    if not float(eps) >= 0.:
        raise SSNeuronError(f'eps: expected a number >= 0, got {eps}')


def _rows(t):
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


class _AddRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        ctx.set_materialize_grads(False)
        need = any(ctx.needs_input_grad)
        rows = _rows(x)
        if need and residual is None:
            rows = rows.contiguous()                       # kept for the backward
        weight = weight.contiguous()
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        total = torch.empty_like(y) if residual is not None else None
        rstd = torch.empty(rows.shape[0], dtype=torch.float32, device=x.device) if need else None
        if rows.shape[0]:
            _seqlib.rms_norm_fwd(rows, None if residual is None else _rows(residual), weight, y, total, rstd, eps)
        if need:
            ctx.save_for_backward(rows if residual is None else total, weight, rstd)
            ctx.shape = x.shape
        return (y, total) if residual is not None else y

    @staticmethod
    def backward(ctx, g_y, g_sum=None):
        return _norm_grads_once(ctx, g_y, g_sum) if torch.is_grad_enabled() else _norm_grads(ctx, g_y, g_sum)


def _norm_grads(ctx, g_y, g_sum):
    h, weight, rstd = ctx.saved_tensors
    need_x, need_r, need_w, _ = ctx.needs_input_grad
    g_h = torch.empty(ctx.shape, dtype=h.dtype, device=h.device)
    g_w = torch.empty_like(weight) if need_w else None
    if rstd.shape[0]:
        _seqlib.rms_norm_bwd(None if g_y is None else g_y.contiguous(), None if g_sum is None else g_sum.contiguous(), _rows(h), weight, rstd, g_h, g_w)
    elif need_w:
        g_w.zero_()
    return g_h if need_x else None, g_h if need_r else None, g_w, None


_norm_grads_once = once_differentiable(_norm_grads)


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """h = x + residual, kept in x's type;  y = h / sqrt(mean(h^2) + eps) * weight over the last axis.  Returns (y, h); without a residual h is x itself.

    x, residual: [..., C] in float32 / float16 / bfloat16, C <= 16384; weight fp32 [C].  Sums are fp32; y is rounded once.  Gradients: x, residual, weight."""
    _norm_operands(x, weight, residual, eps)
    if residual is None:
        return _AddRMSNorm.apply(x, None, weight, float(eps)), x
    return _AddRMSNorm.apply(x, residual, weight, float(eps))


def add_rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """`add_rms_norm` handed on in 8 bits: returns (codes int8 [..., C], scales fp32 [...], h) with codes * scales the norm; the largest value of a row has the
    code +-127, ties go to the even code.  A row of zeros has scale 0; a row with a NaN or an infinity has codes 0 and scale NaN.  No gradients."""
    _norm_operands(x, weight, residual, eps)
    shape, dev = x.shape, x.device
    rows = _rows(x)
    codes = torch.empty(shape, dtype=torch.int8, device=dev)
    scales = torch.empty(shape[:-1], dtype=torch.float32, device=dev)
    total = torch.empty(shape, dtype=x.dtype, device=dev) if residual is not None else None
    if rows.shape[0]:
        _seqlib.rms_norm_int8(rows, None if residual is None else _rows(residual), weight.contiguous(), codes, scales, total, float(eps))
    return codes, scales, x if residual is None else total


def dequantize_int8(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that 8-bit codes [..., C] with a scale per row [...] stand for."""
    _require_hip(codes, 'codes')
    shape = codes.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise SSNeuronError(f'codes: expected [..., C], got {tuple(shape)}')
    _operand(codes, 'codes', codes.device, torch.int8, shape)
    _operand(scales, 'scales', codes.device, torch.float32, shape[:-1])
    if dtype not in _FLOATS:
        raise SSNeuronError(f'dtype: expected float32, float16 or bfloat16, got {dtype}')
    out = torch.empty(shape, dtype=dtype, device=codes.device)
    if out.numel():
        _seqlib.dequant_int8(codes.contiguous(), scales.contiguous(), out)
    return out


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

    codes int8 [..., K] (spike counts are codes of scale 1), scales fp32 [...], weight int8 [N, K], weight_scale fp32 [N], bias fp32 [N]; K < 131072.  Scaled in
    fp32, rounded once to out_dtype (float32 / float16 / bfloat16).  No gradients."""
    _require_hip(codes, 'codes')
    shape, dev = codes.shape, codes.device
    if len(shape) < 1 or weight.dim() != 2:
        raise SSNeuronError(f'codes [..., K], weight [N, K]: got {tuple(shape)}, {tuple(weight.shape)}')
    N, K = weight.shape
    lead = shape[:-1]
    _operand(codes, 'codes', dev, torch.int8, (*lead, K))
    _operand(scales, 'scales', dev, torch.float32, lead)
    _operand(weight, 'weight', dev, torch.int8, (N, K))
    _operand(weight_scale, 'weight_scale', dev, torch.float32, (N,))
    if bias is not None:
        _operand(bias, 'bias', dev, torch.float32, (N,))
    if not 1 <= K <= _seqlib.MAX_INT8_K or N < 1:
        raise SSNeuronError(f'weight: [N, K] = [{N}, {K}]; N >= 1 and 1 <= K <= {_seqlib.MAX_INT8_K} (sums stay within 32 bits) are implemented')
    if out_dtype not in _FLOATS:
        raise SSNeuronError(f'out_dtype: expected float32, float16 or bfloat16, got {out_dtype}')
    if (scales.requires_grad or weight_scale.requires_grad or (bias is not None and bias.requires_grad)) and torch.is_grad_enabled():
        raise SSNeuronError('int8_linear has no gradient: call it under torch.no_grad() or detach scales and bias')
    out = torch.empty((*lead, N), dtype=out_dtype, device=dev)
    if out.numel():
        _seqlib.int8_linear(_rows(codes), scales.contiguous(), _rows(weight), weight_scale.contiguous(), None if bias is None else bias.contiguous(), out)
    return out
