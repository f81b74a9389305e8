"""Cases of the sequence operators (stereospike_amd.sequence): leaky attention over a sequence and for one step, the root-mean-square norm with the
residual's addition (16 / 32-bit output with its gradients, or 8-bit output with scales), and the 8-bit integer product with scales.

A case is a dict of plain values; `prepare` makes a user's tensors for it, `run` is one pass, `exact` the definition in 64 bits, `work` what a pass cannot
do without.  With `own` false `run` computes the plain form in elementary torch operations; with `own` true it makes the framework's calls."""
import math

import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
BYTES = {'f32': 4, 'bf16': 2, 'f16': 2}


# ----------------------------------------------------------------------------------------------------------------------------------------------------------
# the cases
# ----------------------------------------------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a prompt of event tokens read in one pass by a wide sequence layer, the state kept for the steps that follow
        dict(name='attention prompt bf16', op='attention', dtype='bf16', train=False, T=4096, B=4, H=16, Hk=16, Dk=128, Dv=128, ragged=False, state=False),
        # one long recording, few heads: the time axis alone has to fill the card
        dict(name='attention long f16', op='attention', dtype='f16', train=False, T=16384, B=1, H=8, Hk=8, Dk=64, Dv=64, ragged=False, state=True),
        # a training step's forward and backward
        dict(name='attention train bf16', op='attention', dtype='bf16', train=True, T=2048, B=4, H=16, Hk=16, Dk=128, Dv=128, ragged=False, state=False),
        # a padded training batch in the framework's default precision, odd sizes, two query heads to a key head, a carried state
        dict(name='attention train f32 ragged', op='attention', dtype='f32', train=True, T=777, B=6, H=8, Hk=4, Dk=80, Dv=96, ragged=True, state=True),
        # one time step of one stream (the single-step call): latency
        dict(name='step one stream', op='step', dtype='f32', B=1, H=8, Hk=8, Dk=64, Dv=64),
        # one time step of many streams: every state is read and written
        dict(name='step many streams', op='step', dtype='bf16', B=512, H=16, Hk=16, Dk=128, Dv=128),
        # the bottleneck's rows (T = 5, B = 16, 17 x 22 positions, 512 channels), forward and backward
        dict(name='norm train bf16', op='norm', dtype='bf16', train=True, rows=29920, C=512, residual=True),
        # wide rows handed on in 8 bits
        dict(name='norm int8 wide', op='norm8', dtype='bf16', rows=16384, C=4096, residual=True),
        # one row: latency
        dict(name='norm int8 one row', op='norm8', dtype='f32', rows=1, C=512, residual=True),
        # the bottleneck's 3 x 3 convolution as a product: spike counts against 8-bit weights
        dict(name='product bottleneck', op='product', out='bf16', M=29920, N=512, K=4608, bias=False, spikes=True),
        # a wide projection of many tokens
        dict(name='product wide', op='product', out='bf16', M=8192, N=8192, K=4096, bias=False, spikes=False),
        # the same projection for one token: the weight is read once
        dict(name='product one token', op='product', out='f32', M=1, N=8192, K=4096, bias=True, spikes=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width over its whole range: most are whole vectors of eight, as in real layers, the others any number."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.3 else max(8, n // 8 * 8)


def _cost(case):
    w = work(case)
    return max(w['bytes'] / 5e12, w['flops'] / 1e15)


def draw(rng):
    op = rng.choice(['attention', 'attention', 'step', 'norm', 'norm8', 'product', 'product'])
    dtype = rng.choice(['f32', 'bf16', 'f16'])
    if op == 'attention':
        train = rng.random() < 0.5
        group = rng.choice([1, 1, 2, 3])
        Hk = _log_int(rng, 1, 12)
        c = dict(op=op, dtype=dtype, train=train, T=_log_int(rng, 1, 8192), B=_log_int(rng, 1, 8), H=Hk * group, Hk=Hk, Dk=_width(rng, 8, 256),
                 Dv=_width(rng, 8, 256), ragged=rng.random() < 0.4, state=rng.random() < 0.5)
        top = max(_cost(x) for x in listed() if x['op'] == op and x['train'] == train)
        while _cost(c) > top or c['B'] * c['H'] * c['T'] ** 2 > 2 ** 30:
            c['T'] = c['T'] * 2 // 3
        return c
    if op == 'step':
        group = rng.choice([1, 1, 2, 4])
        Hk = _log_int(rng, 1, 16)
        c = dict(op=op, dtype=dtype, B=_log_int(rng, 1, 512), H=Hk * group, Hk=Hk, Dk=_width(rng, 8, 256), Dv=_width(rng, 8, 256))
        top = max(_cost(x) for x in listed() if x['op'] == op)
        while _cost(c) > top:
            c['B'] = c['B'] * 2 // 3
        return c
    if op in ('norm', 'norm8'):
        c = dict(op=op, dtype=dtype, rows=_log_int(rng, 1, 65536), C=_width(rng, 8, 16384), residual=rng.random() < 0.7)
        if op == 'norm':
            c['train'] = rng.random() < 0.6
        top = max(_cost(x) for x in listed() if x['op'] == op)
        while _cost(c) > top:
            c['rows'] = c['rows'] * 2 // 3
        return c
    K = _log_int(rng, 16, 16384)
    c = dict(op=op, out=rng.choice(['f32', 'bf16', 'f16']), M=_log_int(rng, 1, 32768), N=_width(rng, 8, 16384),
             K=K if rng.random() < 0.3 else max(16, K // 16 * 16), bias=rng.random() < 0.5, spikes=rng.random() < 0.3)
    top = max(_cost(x) for x in listed() if x['op'] == op)
    while _cost(c) > top:
        c['M'] = c['M'] * 2 // 3
    return c


def work(case):
    c = case
    if c['op'] == 'attention':
        e, t = BYTES[c['dtype']], c['T'] * c['B']
        qk, vo, st = t * c['Dk'], t * c['Dv'], c['B'] * c['H'] * c['Dk'] * c['Dv'] * 4
        tokens = qk * (c['H'] + c['Hk']) + vo * (c['Hk'] + c['H'])                   # q, k, v in, o out
        b, f = tokens * e + st * (2 if c['state'] else 1), 4.0 * t * c['H'] * c['Dk'] * c['Dv']
        if c['train']:                                                              # + d o in, d q, d k, d v out; four more products of a token with a state
            b += tokens * e + (st if c['state'] else 0)
            f += 10.0 * t * c['H'] * c['Dk'] * c['Dv']
        return dict(bytes=b, flops=f)
    if c['op'] == 'step':
        e, n = BYTES[c['dtype']], c['B']
        return dict(bytes=n * c['H'] * c['Dk'] * c['Dv'] * 8 + n * (c['H'] + c['Hk']) * (c['Dk'] + c['Dv']) * e, flops=4.0 * n * c['H'] * c['Dk'] * c['Dv'])
    if c['op'] == 'norm':
        n, e, r = c['rows'] * c['C'], BYTES[c['dtype']], 2 if c['residual'] else 0
        b, f = n * e * (2 + r) + 4 * c['C'], 5.0 * n                                # x (and the residual) in, the norm (and the sum) out
        if c['train']:
            b, f = b + n * e * (2 + r // 2) + 8 * c['C'], f + 9.0 * n               # its gradient (and the sum's) in, the input's out, the weight's out
        return dict(bytes=b, flops=f)
    if c['op'] == 'norm8':
        n, e = c['rows'] * c['C'], BYTES[c['dtype']]
        return dict(bytes=n * (e * (3 if c['residual'] else 1) + 1) + n * e + 4 * c['C'] + 4 * c['rows'], flops=7.0 * n)
    M, N, K = c['M'], c['N'], c['K']
    return dict(bytes=M * K + N * K + M * N * BYTES[c['out']] + 4 * (M + N * (2 if c['bias'] else 1)), flops=2.0 * M * N * K)


# ----------------------------------------------------------------------------------------------------------------------------------------------------------
# a user's tensors
# ----------------------------------------------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c, dev = case, torch.device('cuda')
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(shape, generator=g, device=dev) * std).to(dtype)

    s = dict(case=c)
    if c['op'] in ('attention', 'step'):
        dt, B, H, Hk, Dk, Dv = DTYPES[c['dtype']], c['B'], c['H'], c['Hk'], c['Dk'], c['Dv']
        lead = (c['T'], B) if c['op'] == 'attention' else (B,)
        s['q'], s['k'], s['v'] = normal(*lead, H, Dk, dtype=dt), normal(*lead, Hk, Dk, dtype=dt), normal(*lead, Hk, Dv, dtype=dt)
        # time constants from two steps to a thousand, spread over the heads: lambda = 1 - 1 / tau
        tau = 2.0 * 512.0 ** (torch.arange(H, device=dev, dtype=torch.float64) / max(1, H - 1))
        s['log_decay'] = torch.log1p(-1.0 / tau).float()
        s['scale'] = Dk ** -0.5
        if c['op'] == 'step':
            s['state'] = normal(B, H, Dk, Dv)
            return s
        s['state'] = normal(B, H, Dk, Dv) if c['state'] else None
        s['lengths'] = None
        if c['ragged']:
            n = torch.randint(0, c['T'] + 1, (B,), generator=g, device=dev, dtype=torch.int32)
            n[0] = c['T']
            s['lengths'] = n
        if c['train']:
            s['grad'] = normal(c['T'], B, H, Dv, dtype=dt)
            for name in ('q', 'k', 'v', 'state'):
                if s[name] is not None:
                    s[name].requires_grad_()
        return s
    if c['op'] in ('norm', 'norm8'):
        dt = DTYPES[c['dtype']]
        s['x'] = normal(c['rows'], c['C'], dtype=dt)
        s['residual'] = normal(c['rows'], c['C'], dtype=dt, std=2.0) if c['residual'] else None
        s['weight'] = 1.0 + normal(c['C'], std=0.1)
        s['eps'] = 1e-6
        if c.get('train'):
            s['grad'] = normal(c['rows'], c['C'], dtype=dt)
            s['grad_sum'] = normal(c['rows'], c['C'], dtype=dt) if c['residual'] else None
            for name in ('x', 'residual', 'weight'):
                if s[name] is not None:
                    s[name].requires_grad_()
        return s
    M, N, K = c['M'], c['N'], c['K']
    if c['spikes']:                                                                # spike counts 0 .. 3, mostly 0: their own value, scale 1
        s['a'] = torch.poisson(torch.full((M, K), 0.2, device=dev), generator=g).clamp_(max=3).to(torch.int8)
        s['a_scale'] = torch.ones(M, device=dev)
    else:
        s['a'] = normal(M, K, std=32.0).round_().clamp_(-127, 127).to(torch.int8)
        s['a_scale'] = torch.exp(normal(M, std=0.5)) / 32
    s['w'] = normal(N, K, std=32.0).round_().clamp_(-127, 127).to(torch.int8)
    s['w_scale'] = torch.exp(normal(N, std=0.5)) / 1024
    s['bias'] = normal(N) if c['bias'] else None
    return s


# ----------------------------------------------------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------------------------------------------------
def run(state):
    c = state['case']
    if own:
        return _OWN[c['op']](c, state)
    with torch.no_grad():
        return _PLAIN[c['op']](c, state)


def _own_attention(c, s):
    from stereospike_amd import sequence
    o, last = sequence.leaky_attention(s['q'], s['k'], s['v'], s['log_decay'], scale=s['scale'], state=s['state'], lengths=s['lengths'], return_state=True)
    out = dict(o=o.detach(), last=last.detach())
    if c['train']:
        wrt = [n for n in ('q', 'k', 'v', 'state') if s[n] is not None]
        for n, gr in zip(wrt, torch.autograd.grad(o, [s[n] for n in wrt], s['grad'])):
            out['d_' + n] = gr
    return out


def _own_step(c, s):
    from stereospike_amd import sequence
    o = sequence.leaky_attention_step(s['q'], s['k'], s['v'], s['log_decay'], s['state'], scale=s['scale'])
    return dict(o=o, state=s['state'])


def _own_norm(c, s):
    from stereospike_amd import sequence
    y, total = sequence.add_rms_norm(s['x'], s['weight'], residual=s['residual'], eps=s['eps'])
    out = dict(y=y.detach())
    if c['residual']:
        out['sum'] = total.detach()
    if c['train']:
        if c['residual']:
            dx, dr, dw = torch.autograd.grad([y, total], [s['x'], s['residual'], s['weight']], [s['grad'], s['grad_sum']])
            out.update(d_x=dx, d_residual=dr, d_weight=dw)
        else:
            dx, dw = torch.autograd.grad(y, [s['x'], s['weight']], s['grad'])
            out.update(d_x=dx, d_weight=dw)
    return out


def _own_norm8(c, s):
    from stereospike_amd import sequence
    y8, scale, total = sequence.add_rms_norm_int8(s['x'], s['weight'], residual=s['residual'], eps=s['eps'])
    out = dict(y=sequence.dequantize_int8(y8, scale, s['x'].dtype), scale=scale)
    if c['residual']:
        out['sum'] = total
    return out


def _own_product(c, s):
    from stereospike_amd import sequence
    return sequence.int8_linear(s['a'], s['a_scale'], s['w'], s['w_scale'], bias=s['bias'], out_dtype=DTYPES[c['out']])


_OWN = dict(attention=_own_attention, step=_own_step, norm=_own_norm, norm8=_own_norm8, product=_own_product)


# ---- the plain forms: 32 bits, rounded once at the end
def _heads_first(x, group=1):
    """[T, B, h, D] -> fp32 [B, h * group, T, D], each head `group` times in a row."""
    x = x.detach().float().permute(1, 2, 0, 3)
    return x.repeat_interleave(group, 1) if group > 1 else x.contiguous()


def _plain_attention(c, s):
    dt, group = s['q'].dtype, c['H'] // c['Hk']
    T, dev = c['T'], s['q'].device
    q, k, v = _heads_first(s['q']) * s['scale'], _heads_first(s['k'], group), _heads_first(s['v'], group)
    t = torch.arange(T, device=dev, dtype=torch.float32)
    n = torch.full((c['B'],), T, device=dev) if s['lengths'] is None else s['lengths']
    live = (t[None, :] < n[:, None]).float()[:, None, :, None]                       # [B, 1, T, 1]
    q, k, v = q * live, k * live, v * live
    g = s['log_decay'][:, None, None]
    gap = t[:, None] - t[None, :]
    decay = torch.exp(g * gap.clamp_min(0)) * (gap >= 0)                             # [H, T, T]
    P = torch.matmul(q, k.transpose(-1, -2)) * decay
    o = torch.matmul(P, v)
    since = torch.exp(g * (t[:, None] + 1))                                          # [H, T, 1]: from the first state to each step
    left = torch.exp(s['log_decay'][None, :, None] * (n[:, None, None] - 1 - t).clamp_min(0))[..., None] * live      # [B, H, T, 1]: from each step to the last
    whole = torch.exp(s['log_decay'][None, :] * n[:, None])[..., None, None]         # [B, H, 1, 1]
    last = torch.matmul((k * left).transpose(-1, -2), v)
    if s['state'] is not None:
        o = o + torch.matmul(q * since, s['state'].detach())
        last = last + whole * s['state'].detach()
    back = lambda x: x.permute(2, 0, 1, 3).to(dt)                                    # noqa: E731
    out = dict(o=back(o).contiguous(), last=last)
    if c['train']:
        do = _heads_first(s['grad']) * live
        dP = torch.matmul(do, v.transpose(-1, -2)) * decay
        dq = torch.matmul(dP, k)
        dk, dv = torch.matmul(dP.transpose(-1, -2), q), torch.matmul(P.transpose(-1, -2), do)
        if s['state'] is not None:
            dq = dq + torch.matmul(do * since, s['state'].detach().transpose(-1, -2))
            out['d_state'] = torch.matmul((q * since).transpose(-1, -2), do)
        shared = lambda x: x.reshape(c['B'], c['Hk'], group, T, -1).sum(2)           # noqa: E731
        out.update(d_q=back(dq * s['scale']).contiguous(), d_k=back(shared(dk)).contiguous(), d_v=back(shared(dv)).contiguous())
    return out


def _plain_step(c, s):
    group = c['H'] // c['Hk']
    q, k, v = s['q'].float() * s['scale'], s['k'].float().repeat_interleave(group, 1), s['v'].float().repeat_interleave(group, 1)
    s['state'].mul_(torch.exp(s['log_decay'])[None, :, None, None]).add_(k[..., :, None] * v[..., None, :])
    return dict(o=(q[..., :, None] * s['state']).sum(-2).to(s['q'].dtype), state=s['state'])


def _plain_norm(c, s):
    dt = s['x'].dtype
    total = s['x'] if s['residual'] is None else (s['x'].float() + s['residual'].float()).to(dt)
    h, w = total.float(), s['weight']
    rstd = torch.rsqrt((h * h).mean(-1, keepdim=True) + s['eps'])
    n = h * rstd
    out = dict(y=(n * w).to(dt))
    if c['residual']:
        out['sum'] = total.detach()
    if c['train']:
        gw = s['grad'].float() * w
        d = rstd * (gw - n * (gw * n).mean(-1, keepdim=True))
        out['d_weight'] = (s['grad'].float() * n).sum(0)
        if c['residual']:
            d = d + s['grad_sum'].float()
            out['d_residual'] = d.to(dt)
        out['d_x'] = d.to(dt)
    return out


def _plain_norm8(c, s):
    # in 64 bits from the product with the weight on: a value next to the border of two codes would change its code
    dt = s['x'].dtype
    total = s['x'] if s['residual'] is None else (s['x'].float() + s['residual'].float()).to(dt)
    h = total.double()
    rstd = torch.rsqrt((h * h).mean(-1, keepdim=True) + s['eps'])
    u = h * s['weight'].double()
    top = u.abs().amax(-1, keepdim=True)
    codes = torch.round(u * 127.0 / top.clamp_min(1e-300))
    scale = top * rstd / 127.0
    out = dict(y=(codes * scale).to(dt), scale=scale[:, 0].float())
    if c['residual']:
        out['sum'] = total
    return out


def _plain_product(c, s):
    y = torch.matmul(s['a'].float(), s['w'].float().t()) * s['a_scale'][:, None] * s['w_scale'][None, :]
    if s['bias'] is not None:
        y = y + s['bias']
    return y.to(DTYPES[c['out']])


_PLAIN = dict(attention=_plain_attention, step=_plain_step, norm=_plain_norm, norm8=_plain_norm8, product=_plain_product)


# ----------------------------------------------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ----------------------------------------------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    c = case
    if c['op'] == 'product' and 2.0 * c['M'] * c['N'] * c['K'] > 4e12:
        return None
    s = prepare(c, seed)
    s = {n: x.detach() if isinstance(x, torch.Tensor) else x for n, x in s.items()}
    with torch.no_grad():
        return _EXACT[c['op']](c, s)


def _exact_attention(c, s):
    """The recurrence itself, one token after the other."""
    T, B, H, Dk, Dv, r = c['T'], c['B'], c['H'], c['Dk'], c['Dv'], c['H'] // c['Hk']
    q, k, v = (s[n].double() for n in ('q', 'k', 'v'))
    n = torch.full((B,), T, device=q.device) if s['lengths'] is None else s['lengths']
    dead = torch.arange(T, device=q.device)[:, None] >= n[None, :]
    lam = s['log_decay'].double().exp()[None, :, None, None]
    head = torch.arange(H, device=q.device) // r
    first = s['state'].double() if s['state'] is not None else torch.zeros(B, H, Dk, Dv, device=q.device, dtype=torch.float64)
    S, o = first.clone(), torch.zeros(T, B, H, Dv, device=q.device, dtype=torch.float64)
    dq, do = torch.zeros_like(q), s['grad'].double() if c['train'] else None
    for t in range(T):
        new = torch.addcmul(S * lam, k[t][:, head, :, None], v[t][:, head, None, :])
        S = torch.where(dead[t][:, None, None, None], S, new) if c['ragged'] else new
        o[t] = torch.matmul(q[t][:, :, None, :], S)[:, :, 0] * s['scale']
        if c['train']:
            dq[t] = torch.matmul(S, do[t][..., None])[..., 0] * s['scale']
    o[dead] = 0
    out = dict(o=o, last=S)
    if c['train']:
        dq[dead] = 0
        R = torch.zeros_like(S)
        dk, dv = torch.zeros(T, B, H, Dk, device=q.device, dtype=torch.float64), torch.zeros_like(o)
        for t in reversed(range(T)):
            R = R * lam
            add = (q[t][..., :, None] * s['scale']) * do[t][..., None, :]
            R = R + (add.masked_fill(dead[t][:, None, None, None], 0) if c['ragged'] else add)
            dk[t] = torch.matmul(R, v[t][:, head, :, None])[..., 0]
            dv[t] = torch.matmul(k[t][:, head, None, :], R)[:, :, 0]
        dk[dead], dv[dead] = 0, 0
        out.update(d_q=dq, d_k=dk.reshape(T, B, c['Hk'], r, Dk).sum(3), d_v=dv.reshape(T, B, c['Hk'], r, Dv).sum(3))
        if s['state'] is not None:
            out['d_state'] = R * lam
    return out


def _exact_step(c, s):
    r, q, k, v = c['H'] // c['Hk'], s['q'].double(), s['k'].double(), s['v'].double()
    S = torch.empty_like(s['state'], dtype=torch.float64)
    o = torch.empty(c['B'], c['H'], c['Dv'], device=q.device, dtype=torch.float64)
    for h in range(c['H']):
        S[:, h] = s['state'][:, h].double() * math.exp(float(s['log_decay'][h])) + torch.einsum('bi,bj->bij', k[:, h // r], v[:, h // r])
        o[:, h] = torch.einsum('bi,bij->bj', q[:, h] * s['scale'], S[:, h])
    return dict(o=o, state=S)


def _exact_norm(c, s):
    x, w, C = s['x'].double(), s['weight'].double(), c['C']
    total = x if s['residual'] is None else (s['x'].float() + s['residual'].float()).to(s['x'].dtype).double()     # the sum is kept in the input's type
    size = torch.sqrt(total.square().sum(1) / C + s['eps'])[:, None]
    out = dict(y=total / size * w)
    if c['residual']:
        out['sum'] = x + s['residual'].double()
    if c['train']:
        g = s['grad'].double()
        along = (g * w * total).sum(1, keepdim=True) / C
        d = g * w / size - total * along / size ** 3
        out['d_weight'] = (g * total / size).sum(0)
        if c['residual']:
            d = d + s['grad_sum'].double()
            out['d_residual'] = d
        out['d_x'] = d
    return out


def _exact_norm8(c, s):
    total = s['x'].double() if s['residual'] is None else (s['x'].float() + s['residual'].float()).to(s['x'].dtype).double()
    y = total * s['weight'].double() / torch.sqrt(total.square().sum(1, keepdim=True) / c['C'] + s['eps'])
    scale = y.abs().max(1, keepdim=True).values / 127
    out = dict(y=torch.where(scale > 0, torch.round(y / scale), torch.zeros_like(y)) * scale, scale=scale[:, 0])
    if c['residual']:
        out['sum'] = s['x'].double() + s['residual'].double()
    return out


def _exact_product(c, s):
    y = torch.empty(c['M'], c['N'], device=s['a'].device, dtype=torch.float64)
    w = s['w'].double()
    for i in range(0, c['M'], 4096):
        y[i:i + 4096] = s['a'][i:i + 4096].double() @ w.t()
    y *= s['a_scale'].double()[:, None]
    y *= s['w_scale'].double()[None, :]
    return y if s['bias'] is None else y + s['bias'].double()


_EXACT = dict(attention=_exact_attention, step=_exact_step, norm=_exact_norm, norm8=_exact_norm8, product=_exact_product)
