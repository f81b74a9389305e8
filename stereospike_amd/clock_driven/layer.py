"""`layer.Dropout` is only type-checked by the reference (SNN_models.py:26: `isinstance(m, layer.Dropout)` ->
`m.mask.detach_()`); no shipped model instantiates it.  Kept so that check has a class to test against.

`layer.LeakyAttention`, `layer.AddRMSNorm` and `layer.Int8Linear` are the layers of the sequence operators (stereospike_amd.sequence): the first keeps its
state between calls as a neuron node keeps its membrane (`functional.reset_net`, `functional.detach_net`)."""
from typing import Optional

import torch
import torch.nn as nn

from .. import sequence
from .._lib import SSNeuronError


class Dropout(nn.Module):
    """Dropout whose mask is drawn once and kept until reset() (time-invariant mask across steps)."""

    def __init__(self, p: float = 0.5):
        super().__init__()
        assert 0. <= p < 1.
        self.p = p
        self.mask = None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not self.training:
            return x
        if self.mask is None:
            self.mask = (torch.rand_like(x) > self.p).to(x) / (1. - self.p)
        return x * self.mask

    def reset(self):
        self.mask = None


class LeakyAttention(nn.Module):
    """Linear attention with a leak per head, stateful like a neuron node: `layer(q, k, v)` is one time step, `layer.forward_sequence(q_seq, k_seq, v_seq)` a
    whole [T, B, heads, D] sequence; the state `s` (fp32 [B, heads, Dk, Dv]) is carried from call to call until reset().

    tau: the heads' time constants in steps (lambda = 1 - 1 / tau, as in a LIFNode; inf never forgets): a list of `heads` numbers, or None for 2 .. 1024
    spread evenly over their logarithms.  scale: of the queries, Dk ** -0.5 by default."""

    def __init__(self, heads: int, tau=None, scale: Optional[float] = None):
        super().__init__()
        if tau is None:
            tau = 2. * 512. ** (torch.arange(heads, dtype=torch.float64) / max(1, heads - 1))
        tau = torch.as_tensor(tau, dtype=torch.float64)
        assert tau.shape == (heads,) and bool((tau >= 1.).all()), 'tau: one number >= 1 for each head'
        self.heads, self.scale = heads, scale
        self.register_buffer('log_decay', torch.log1p(-1. / tau).float())
        self.s = None

    def reset(self):
        self.s = None

    def detach(self):
        if self.s is not None:
            self.s = self.s.detach()

    def forward_sequence(self, q_seq, k_seq, v_seq, lengths: Optional[torch.Tensor] = None):
        """lengths: int32 [B], the valid steps of each stream; the state of a stream stops at its last valid step."""
        out, self.s = sequence.leaky_attention(q_seq, k_seq, v_seq, self.log_decay, self.scale, self._state(q_seq.shape[-3:], v_seq), lengths, True)
        return out

    def _state(self, shape, v):
        """The state, if it fits queries of this shape [B, heads, Dk]."""
        if self.s is not None and tuple(self.s.shape) != (*shape, v.shape[-1]):
            raise SSNeuronError(f'state shape {tuple(self.s.shape)} does not fit queries {tuple(shape)} and values of {v.shape[-1]}; '
                                f'call functional.reset_net(net) when the batch shape changes')
        return self.s

    def forward(self, q, k, v):
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, self.s)):
            return self.forward_sequence(q[None], k[None], v[None])[0]
        if self._state(q.shape, v) is None:
            self.s = torch.zeros((*q.shape, v.shape[-1]), dtype=torch.float32, device=q.device)
        elif self.s.requires_grad:                         # a training pass left it: its graph keeps its own tensor, the steps from here on are no part of it
            self.s = self.s.detach().clone()
        return sequence.leaky_attention_step(q, k, v, self.log_decay, self.s, self.scale)

    def extra_repr(self):
        return f'heads={self.heads}, scale={self.scale}'


class AddRMSNorm(nn.Module):
    """Residual addition + root-mean-square norm: `layer(x, residual)` -> (norm, sum); `layer.forward_int8(x, residual)` -> (codes, scales, sum)."""

    def __init__(self, width: int, eps: float = 1e-6):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(width))

    def forward(self, x, residual: Optional[torch.Tensor] = None):
        return sequence.add_rms_norm(x, self.weight, residual, self.eps)

    def forward_int8(self, x, residual: Optional[torch.Tensor] = None):
        return sequence.add_rms_norm_int8(x, self.weight, residual, self.eps)

    def extra_repr(self):
        return f'{self.weight.numel()}, eps={self.eps}'


class Int8Linear(nn.Module):
    """An nn.Linear with its weight in 8 bits and a scale per output channel, for inference: `layer(codes, scales)`; spike counts go in as int8 with
    scales = None (their own value)."""

    def __init__(self, linear: nn.Linear, out_dtype: torch.dtype = torch.float32):
        super().__init__()
        codes, scale = sequence.quantize_channels(linear.weight)
        self.out_dtype = out_dtype
        self.register_buffer('weight', codes)
        self.register_buffer('weight_scale', scale)
        self.register_buffer('bias', None if linear.bias is None else linear.bias.detach().float().clone())

    def forward(self, codes, scales: Optional[torch.Tensor] = None):
        if scales is None:
            scales = torch.ones(codes.shape[:-1], dtype=torch.float32, device=codes.device)
        return sequence.int8_linear(codes, scales, self.weight, self.weight_scale, self.bias, self.out_dtype)

    def extra_repr(self):
        return f'in_features={self.weight.shape[1]}, out_features={self.weight.shape[0]}, bias={self.bias is not None}'
