"""MI355X suite of the sequence operators against plain 64-bit implementations.

Tolerances count roundings.  u = 2^-24 is half a step of fp32, HALF[dtype] half a step of the output's type.  A computed sum of products may be off by
(roundings a term passes through) * u * (the sum of the terms' magnitudes), so every comparison has the same sum with absolute values beside it."""
import math

import pytest
import torch
import torch.utils.checkpoint

from stereospike_amd import sequence
from stereospike_amd.clock_driven import functional, layer

pytestmark = pytest.mark.gpu
U = 2. ** -24
HALF = {torch.float32: 2. ** -24, torch.bfloat16: 2. ** -8, torch.float16: 2. ** -11}
# below its smallest normal number 2^-14 fp16 has steps of 2^-24: half of one, whatever the value (the other types' steps there are under 1e-38)
TINY = {torch.float32: 1e-30, torch.bfloat16: 1e-30, torch.float16: 2. ** -25 * 1.01}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
DEV = 'cuda'


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, std=1.):
    return (torch.randn(shape, generator=g) * std).to(dtype)


def within(got, want, room, what):
    got, want, room = got.detach().cpu().double(), want.detach().cpu().double(), room.detach().cpu().double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), f'{what}: not finite'
    off = (got - want).abs() - room
    assert (off <= 0).all(), f'{what}: {(off > 0).sum().item()} of {off.numel()} out of tolerance, worst by {off.max().item():.3g} (values up to {want.abs().max().item():.3g})'


# ----------------------------------------------------------------------------------------------------------------------------------------------------------
# leaky attention
# ----------------------------------------------------------------------------------------------------------------------------------------------------------
def leaky_ref(q, k, v, log_decay, scale, state=None, lengths=None):
    """The recurrence in fp64 on the CPU, differentiable: the definition."""
    T, B, H, Dk = q.shape
    r = H // k.shape[2]
    q, k, v = q.double().cpu(), k.double().cpu().repeat_interleave(r, 2), v.double().cpu().repeat_interleave(r, 2)
    lam = log_decay.double().cpu().exp()[:, None, None]
    S = torch.zeros(B, H, Dk, v.shape[3], dtype=torch.float64) if state is None else state.double().cpu()
    out = []
    for t in range(T):
        new = lam * S + k[t, :, :, :, None] * v[t, :, :, None, :]
        o = scale * torch.einsum('bhi,bhij->bhj', q[t], new)
        if lengths is not None:
            live = (t < lengths.cpu())[:, None, None]
            new, o = torch.where(live[..., None], new, S), torch.where(live, o, torch.zeros_like(o))
        S = new
        out.append(o)
    return torch.stack(out), S


def leaky_case(T, B, H, Hk, Dk, Dv, dtype, state, ragged, seed=0):
    g = gen(seed)
    q, k, v = normal(g, T, B, H, Dk, dtype=dtype), normal(g, T, B, Hk, Dk, dtype=dtype), normal(g, T, B, Hk, Dv, dtype=dtype)
    decay = torch.tensor([0., -1e-3, -0.05, -0.7, -20., -math.inf])[torch.arange(H) * 5 % 6]
    s = normal(g, B, H, Dk, Dv) if state else None
    n = torch.tensor([T, 0, 1, T - 1, T // 2 + 1, T + 5, -1])[torch.arange(B) % 7].to(torch.int32) if ragged else None
    return q, k, v, decay, s, n


def leaky_check(T, B, H, Hk, Dk, Dv, dtype, state, ragged, grads, seed=0):
    q, k, v, decay, s, n = leaky_case(T, B, H, Hk, Dk, Dv, dtype, state, ragged, seed)
    scale = Dk ** -0.5
    leaf = [t.clone().to(DEV).requires_grad_(grads) if t is not None else None for t in (q, k, v, s)]
    poison = [t.detach().clone() if t is not None else None for t in leaf[:3]]
    if ragged:                                             # what lies behind the last valid step is not looked at
        for t in poison:
            t[torch.arange(T, device=DEV)[:, None] >= n.to(DEV).clamp(0, T)[None, :]] = math.nan
    use = [t.requires_grad_(grads) for t in poison] + [leaf[3]]
    o, last = sequence.leaky_attention(use[0], use[1], use[2], decay.to(DEV), state=use[3], lengths=None if n is None else n.to(DEV), return_state=True)
    # every term passes through at most 2 roundings per step it leaks, the products, and the sum over Dk and the steps of a tile
    steps = 2 * T + Dk + Dv + 80
    sharp = HALF[dtype] if dtype != torch.float32 else U   # one rounding of the token-by-token weights, or of the state, to the operands' type
    ref = [t.double().requires_grad_(grads) if t is not None else None for t in (q, k, v, s)]
    want, want_last = leaky_ref(*ref[:3], decay, scale, ref[3], n)
    mag = [t.detach().abs().double().requires_grad_(grads) if t is not None else None for t in (q, k, v, s)]
    size, size_last = leaky_ref(*mag[:3], decay, scale, mag[3], n)
    within(o, want, size * (steps * U + sharp) + want.abs() * HALF[dtype] * 1.02 + TINY[dtype], 'o')
    within(last, want_last, size_last * (steps * U) + 1e-30, 'state')
    assert o.dtype == dtype and last.dtype == torch.float32
    if not grads:
        return
    g = gen(seed + 1)
    go, gl = normal(g, *o.shape, dtype=dtype), normal(g, *last.shape)
    used = go.to(DEV)
    if ragged:
        used = used.clone()
        used[torch.arange(T, device=DEV)[:, None] >= n.to(DEV).clamp(0, T)[None, :]] = math.nan
    wrt = [i for i in range(4) if use[i] is not None]
    got = torch.autograd.grad([o, last], [use[i] for i in wrt], [used, gl.to(DEV)])
    exp = torch.autograd.grad([want, want_last], [ref[i] for i in wrt], [go.double(), gl.double()])
    mags = torch.autograd.grad([size, size_last], [mag[i] for i in wrt], [go.double().abs(), gl.double().abs()])
    for i, a, b, m in zip(wrt, got, exp, mags):
        name = 'qkvs'[i]
        low = name != 's'
        within(a, b, m * (steps * U + (sharp if low else 0)) + (b.abs() * HALF[dtype] * 1.02 if low else 0) + TINY[dtype], 'gradient of ' + name)
        assert a.dtype == use[i].dtype


SHAPES = [(1, 1, 1, 1, 1, 1), (2, 1, 2, 1, 16, 16), (5, 3, 2, 2, 7, 9), (16, 2, 2, 2, 64, 64), (63, 2, 2, 2, 8, 24), (64, 1, 1, 1, 128, 128), (65, 7, 3, 1, 33, 17),
          (130, 2, 4, 2, 64, 64), (257, 1, 2, 2, 128, 128), (200, 2, 2, 1, 20, 256), (129, 1, 1, 1, 256, 80), (1100, 1, 2, 2, 48, 72)]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_leaky_attention(shape, dtype):
    leaky_check(*shape, dtype, state=False, ragged=False, grads=True)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape', [(3, 7, 2, 1, 8, 8), (70, 7, 2, 2, 24, 40), (200, 7, 4, 2, 64, 128)])
def test_leaky_attention_state_and_lengths(shape, dtype):
    leaky_check(*shape, dtype, state=True, ragged=True, grads=True)
    leaky_check(*shape, dtype, state=True, ragged=False, grads=True, seed=3)


def segments_of(dtype, T, B, H, Dk, Dv):
    """(segments, the lengths that they may have) of the forward pass, from the size of its workspace: a padded state for each but the last."""
    import ctypes
    from test_sequence_host import _desc, _lib
    code, size = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype], _lib().ss_seq_leaky_ws_floats
    size.argtypes, size.restype = [ctypes.c_void_p], ctypes.c_longlong
    pad = 64 if Dk <= 64 else 128 if Dk <= 128 else 256
    cols = 64 if Dv <= 64 or (code and Dk > 128) else 128
    n, left = divmod(size(ctypes.byref(_desc(dtype=code, out_dtype=code, T=T, B=B, H=H, DA=Dk, DC=Dv))), B * H * -(-Dv // cols) * cols * pad)
    chunks = -(-T // 32)
    assert left == 0
    return n + 1, [32 * c for c in range(1, chunks + 1) if -(-chunks // c) == n + 1]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape,few', [((400, 42, 2, 1, 24, 40), True), ((1100, 12, 2, 1, 24, 40), False), ((700, 12, 1, 1, 72, 136), False), ((600, 12, 1, 1, 136, 72), False)])
def test_leaky_attention_of_ragged_streams_in_segments(shape, few, dtype, monkeypatch):
    """Streams that end on a segment's border, one step before and one behind it, and in no segment at all; few segments (joined by the output pass) and many (by a
    scan), with a state, shared heads and all gradients."""
    T, B, H, Hk, Dk, Dv = shape
    n, seg = segments_of(dtype, T, B, H, Dk, Dv)
    assert 2 <= n <= 5 if few else n > 5 and len(seg) == 1, (n, seg)
    borders = [32 * c for c in range(1, -(-T // 32))] if few else [seg[0], n // 2 * seg[0], (n - 1) * seg[0]]
    lengths = torch.tensor([T, 0, 1, *(b + d for b in borders for d in (-1, 0, 1)), *[T] * B][:B], dtype=torch.int32)
    case = leaky_case
    monkeypatch.setitem(globals(), 'leaky_case', lambda *args: (*case(*args)[:5], lengths))
    leaky_check(*shape, dtype, state=True, ragged=True, grads=True)


@pytest.mark.parametrize('dtype', DTYPES)
def test_leaky_attention_long(dtype):
    leaky_check(5000, 1, 2, 2, 16, 24, dtype, state=True, ragged=False, grads=False)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('what', [math.nan, math.inf])
def test_what_is_not_finite_reaches_no_earlier_step(dtype, what):
    """A value that is not finite at step 37 of 100 (inside a tile): outputs and states before it are bit for bit those without it; the gradients behind a gradient
    that is not finite likewise."""
    q, k, v, decay, _, _ = (t.to(DEV) if t is not None else None for t in leaky_case(100, 2, 2, 2, 24, 40, dtype, False, False, seed=11))
    decay = torch.tensor([-0.01, -0.2], device=DEV)
    clean = sequence.leaky_attention(q, k, v, decay)
    for operand in range(3):
        use = [q.clone(), k.clone(), v.clone()]
        use[operand][37, 0, 1, 5] = what
        o = sequence.leaky_attention(*use, decay)
        assert torch.equal(o[:37], clean[:37]) and torch.equal(o[:, 1], clean[:, 1]) and torch.equal(o[:, 0, 0], clean[:, 0, 0])
        assert not torch.isfinite(o[37, 0, 1]).all()
        if operand == 0:                                                        # a query reads, and leaves nothing behind
            assert torch.equal(o[38:], clean[38:])
        else:
            assert not torch.isfinite(o[38, 0, 1]).all()
        if operand == 2:                                                        # a value's column is its own
            rest = torch.arange(40, device=DEV) != 5
            assert torch.equal(o[..., rest], clean[..., rest])
    use = [t.clone().requires_grad_() for t in (q, k, v)]
    g = normal(gen(12), 100, 2, 2, 40, dtype=dtype).to(DEV)
    o = sequence.leaky_attention(*use, decay)
    want = torch.autograd.grad(o, use, g, retain_graph=True)
    bad = g.clone()
    bad[37, 0, 1, 5] = what
    got = torch.autograd.grad(o, use, bad)
    assert torch.equal(got[0][:37], want[0][:37]) and torch.equal(got[0][38:], want[0][38:])
    for a, b in zip(got[1:], want[1:]):
        assert torch.equal(a[38:], b[38:]) and torch.equal(a[:, 1], b[:, 1])
        assert not torch.isfinite(a[37, 0, 1]).all()


@pytest.mark.parametrize('T', [7, 8, 9, 31, 32, 33])
@pytest.mark.parametrize('dtype', DTYPES)
def test_leaky_attention_around_a_tile(T, dtype):
    """The shortest call in tiles and its neighbours, a tile and one step less or more; widths one behind a multiple of 64."""
    leaky_check(T, 7, 2, 1, 65, 129, dtype, state=True, ragged=True, grads=True)


@pytest.mark.parametrize('shape', [(1, 7, 4, 2, 33, 65), (1, 2, 3, 1, 128, 64), (1, 1, 2, 2, 200, 7), (2, 7, 4, 2, 16, 16), (3, 1, 6, 2, 80, 96)])
@pytest.mark.parametrize('dtype', DTYPES)
def test_leaky_attention_of_few_steps(shape, dtype):
    """One step with shared heads, lengths of 0 and 1 and rows of any alignment, and its neighbours."""
    leaky_check(*shape, dtype, state=True, ragged=True, grads=True)
    leaky_check(*shape, dtype, state=False, ragged=False, grads=True, seed=2)


@pytest.mark.parametrize('T', [2, 9, 32])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_short_sequences_round_their_outputs_once(T, dtype):
    """Within one tile and without a state only the token-by-token weights lie between operands and outputs, and those have two terms of the operands' type: what is
    left of them is half a step of a half step, beside the fp32 roundings and the output's own."""
    for Dk, Dv in ((8, 24), (64, 64), (200, 31)):
        q, k, v, decay, _, _ = leaky_case(T, 3, 2, 1, Dk, Dv, dtype, False, False, seed=21)
        o = sequence.leaky_attention(q.to(DEV), k.to(DEV), v.to(DEV), decay.to(DEV))
        want, size = leaky_ref(q, k, v, decay, Dk ** -0.5)[0], leaky_ref(q.abs(), k.abs(), v.abs(), decay, Dk ** -0.5)[0]
        within(o, want, size * ((2 * T + Dk + 80) * U + HALF[dtype] ** 2) + want.abs() * HALF[dtype] * 1.02 + TINY[dtype], f'{Dk} x {Dv}')


@pytest.mark.parametrize('shape', [(40, 2, 2, 1, 64, 64), (70, 3, 4, 2, 24, 40), (300, 1, 2, 2, 128, 128), (90, 1, 2, 1, 192, 80), (130, 2, 2, 2, 200, 72)])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_sequences_of_many_tiles_round_their_outputs_once(shape, dtype):
    """Where the state carries the result, and in the gradients: it meets the query in two terms of the operands' type, so what is left of its rounding is half a step
    of a half step (and, for fp16, 2^-39 of the largest value of a state, scaled to fp16's upper end, at the lower end of that type's range), beside the fp32 roundings
    and the output's own."""
    T, B, H, Hk, Dk, Dv = shape
    q, k, v, decay, s, _ = leaky_case(*shape, dtype, True, False, seed=22)
    use = [t.to(DEV).requires_grad_() for t in (q, k, v, s)]
    o = sequence.leaky_attention(*use[:3], decay.to(DEV), state=use[3])
    go = normal(gen(23), *o.shape, dtype=dtype)
    got = (o, *torch.autograd.grad(o, use[:3], go.to(DEV)))

    def exact(f):
        leaf = [f(t).double().requires_grad_() for t in (q, k, v)]
        o = leaky_ref(*leaf, decay, Dk ** -0.5, f(s))[0]
        return (o.detach(), *torch.autograd.grad(o, leaf, f(go).double()))

    for name, a, b, m in zip(('o', 'gradient of q', 'gradient of k', 'gradient of v'), got, exact(lambda t: t), exact(torch.abs)):
        within(a, b, m * ((2 * T + Dk + Dv + 80) * U + HALF[dtype] ** 2) + b.abs() * HALF[dtype] * 1.02 + TINY[dtype], name)


@pytest.mark.parametrize('shape', [(70, 2, 2, 1, 160, 256), (70, 2, 2, 2, 256, 160), (40, 1, 2, 1, 130, 193), (600, 1, 2, 2, 96, 65), (600, 2, 2, 1, 192, 129), (70, 1, 2, 2, 32, 96)])
@pytest.mark.parametrize('dtype', DTYPES)
def test_leaky_attention_of_unequal_widths(shape, dtype):
    """Keys and values whose padded widths agree and whose column blocks do not, and the reverse."""
    leaky_check(*shape, dtype, state=True, ragged=False, grads=True)


@pytest.mark.parametrize('T', [1, 3, 40, 700])
@pytest.mark.parametrize('dtype', DTYPES)
def test_a_decay_that_is_not_a_number_stays_in_its_head(T, dtype):
    q, k, v, _, s, _ = (t.to(DEV) if t is not None else None for t in leaky_case(T, 2, 3, 3, 16, 24, dtype, True, False, seed=13))
    decay = torch.tensor([-0.1, math.nan, -0.01], device=DEV)
    o, last = sequence.leaky_attention(q, k, v, decay, state=s, return_state=True)
    clean, clean_last = sequence.leaky_attention(q, k, v, torch.tensor([-0.1, -0.3, -0.01], device=DEV), state=s, return_state=True)
    assert o[:, :, 1].isnan().all() and last[:, 1].isnan().all()
    assert torch.equal(o[:, :, ::2], clean[:, :, ::2]) and torch.equal(last[:, ::2], clean_last[:, ::2])
    if T == 1:
        o = sequence.leaky_attention_step(q[0], k[0], v[0], decay, s)
        assert o[:, 1].isnan().all() and s[:, 1].isnan().all() and torch.isfinite(s[:, ::2]).all()


@pytest.mark.parametrize('T', [1, 2, 7, 40])
@pytest.mark.parametrize('dtype', DTYPES)
def test_an_infinite_state_stays_in_its_place(T, dtype):
    """S leaks as S * lambda, so an infinity stays one; the other rows and columns of the head keep their values."""
    q, k, v, _, s, _ = (t.to(DEV) if t is not None else None for t in leaky_case(T, 2, 1, 1, 16, 24, dtype, True, False, seed=14))
    decay = torch.tensor([-0.05], device=DEV)
    clean, clean_last = sequence.leaky_attention(q, k, v, decay, state=s, return_state=True)
    bad = s.clone()
    bad[1, 0, 3, 5] = math.inf
    o, last = sequence.leaky_attention(q, k, v, decay, state=bad, return_state=True)
    hit = torch.zeros_like(last, dtype=torch.bool)
    hit[1, 0, 3, 5] = True
    assert (last[hit] == math.inf).all() and torch.equal(last[~hit], clean_last[~hit])
    hit = torch.zeros_like(o, dtype=torch.bool)
    hit[:, 1, 0, 5] = True
    assert torch.equal(o[hit], (q[:, 1, 0, 3].sign() * math.inf)) and torch.equal(o[~hit], clean[~hit])


def test_fp16_states_beyond_the_type():
    """States and token-by-token weights beyond fp16's largest number (65504), with outputs within it: scaled by powers of two.  An infinite value in a column, or
    an infinite query, leaves the other columns' and rows' scales alone."""
    q, k, v, _, _, _ = (t.to(DEV) if t is not None else None for t in leaky_case(100, 1, 2, 2, 24, 40, torch.float16, False, False, seed=15))
    decay = torch.tensor([0., -0.01], device=DEV)
    for q, v in ((q * 0.02, v * 1e4), (q * 3e3, v * 1e-3)):
        k = k * 30 if v.abs().max() < 1 else k
        clean, last = sequence.leaky_attention(q, k, v, decay, return_state=True)
        want, _ = leaky_ref(q, k, v, decay, 24 ** -0.5)
        size, _ = leaky_ref(q.abs(), k.abs(), v.abs(), decay, 24 ** -0.5)
        within(clean, want, size * (400 * U + HALF[torch.float16]) + want.abs() * HALF[torch.float16] * 1.02 + TINY[torch.float16], 'o')
        assert last.abs().max() > 65504 or (q.float() @ k.float().transpose(-1, -2)).abs().max() > 65504
        bad = v.clone()
        bad[37, 0, 1, 5] = math.inf
        rest = torch.arange(40, device=DEV) != 5
        assert torch.equal(sequence.leaky_attention(q, k, bad, decay)[..., rest], clean[..., rest])
        bad = q.clone()
        bad[37, 0, 1, 5] = math.inf
        rest = torch.arange(100, device=DEV) != 37
        assert torch.equal(sequence.leaky_attention(bad, k, v, decay)[rest], clean[rest])


def test_leaky_gradient_against_differences():
    """The map is linear in each operand: a central difference of the definition along a direction is its derivative, up to the definition's fp64."""
    q, k, v, decay, s, n = leaky_case(70, 3, 2, 1, 12, 10, torch.float32, True, True, seed=5)
    use = [t.to(DEV).requires_grad_() for t in (q, k, v, s)]
    o, last = sequence.leaky_attention(*use[:3], decay.to(DEV), state=use[3], lengths=n.to(DEV), return_state=True)
    g = gen(9)
    wo, wl = normal(g, *o.shape), normal(g, *last.shape)
    got = torch.autograd.grad([o, last], use, [wo.to(DEV), wl.to(DEV)])
    base = [t.double() for t in (q, k, v, s)]

    def loss(x):
        a, b = leaky_ref(*x[:3], decay, 12 ** -0.5, x[3], n)
        return (a * wo).sum() + (b * wl).sum()

    for i, grad in enumerate(got):
        d = normal(g, *base[i].shape).double()
        up, down = [list(base) for _ in range(2)]
        up[i], down[i] = base[i] + 0.5 * d, base[i] - 0.5 * d
        slope, along = loss(up) - loss(down), (grad.cpu().double() * d)
        # fp32 roundings of the gradient (300 of them at most), against the size of the terms
        assert abs(along.sum() - slope) <= 300 * U * 40 * along.abs().sum(), 'qkvs'[i]


@pytest.mark.parametrize('dtype', DTYPES)
def test_leaky_attention_strides(dtype):
    """Batch-major tensors, slices of one projection, rows off any alignment, expanded heads: what the contiguous copies give, within the
    roundings of the two kernel forms."""
    g, decay = gen(2), torch.tensor([-0.1, -0.01]).to(DEV)
    T, B, H, D = 75, 2, 2, 32
    x = normal(g, B, T, 3, H, D + 1, dtype=dtype).to(DEV)
    q, k, v = (x[:, :, i, :, 1:].transpose(0, 1) for i in range(3))
    want = sequence.leaky_attention(q.contiguous(), k.contiguous(), v.contiguous(), decay, return_state=True)
    got = sequence.leaky_attention(q, k, v, decay, return_state=True)
    size = leaky_ref(q.abs(), k.abs(), v.abs(), decay, D ** -0.5)
    for a, b, m in zip(got, want, size):
        within(a, b, m * (600 * U + 2 * HALF[dtype]) + 2 * TINY[dtype], 'strided')
    one = k[:, :, :1].expand(T, B, H, D)
    a, b = sequence.leaky_attention(q, one, v, decay), sequence.leaky_attention(q, one.contiguous(), v, decay)
    within(a, b, leaky_ref(q.abs(), one.abs(), v.abs(), decay, D ** -0.5)[0] * (600 * U + 2 * HALF[dtype]) + 2 * TINY[dtype], 'expanded')
    vt = normal(g, T, B, D, H, dtype=dtype).to(DEV).transpose(2, 3)              # a last axis that is not contiguous
    assert torch.equal(sequence.leaky_attention(q, k, vt, decay), sequence.leaky_attention(q, k, vt.contiguous(), decay))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape', [(1, 1, 1, 1, 1), (3, 4, 2, 64, 64), (2, 6, 3, 33, 17), (5, 2, 2, 128, 128), (2, 1, 1, 256, 200), (300, 2, 1, 16, 32)])
def test_step(shape, dtype):
    """Several single steps: the state is updated in place, each against the definition from the state that was there."""
    B, H, Hk, Dk, Dv = shape
    q, k, v, decay, s, _ = leaky_case(3, B, H, Hk, Dk, Dv, dtype, True, False, seed=7)
    state = s.to(DEV)
    for t in range(3):
        before = state.clone()
        o = sequence.leaky_attention_step(q[t].to(DEV), k[t].to(DEV), v[t].to(DEV), decay.to(DEV), state)
        want, last = leaky_ref(q[t:t + 1], k[t:t + 1], v[t:t + 1], decay, Dk ** -0.5, before)
        size, size_last = leaky_ref(q[t:t + 1].abs(), k[t:t + 1].abs(), v[t:t + 1].abs(), decay, Dk ** -0.5, before.abs())
        within(o, want[0], size[0] * (Dk + 8) * U + want[0].abs() * HALF[dtype] * 1.02 + TINY[dtype], 'o')
        within(state, last, size_last * 8 * U + 1e-30, 'state')


def test_step_continues_a_sequence():
    q, k, v, decay, s, _ = (t.to(DEV) if t is not None else None for t in leaky_case(90, 2, 3, 1, 40, 24, torch.float32, True, False, seed=8))
    want, want_last = sequence.leaky_attention(q, k, v, decay, state=s, return_state=True)
    _, state = sequence.leaky_attention(q[:87], k[:87], v[:87], decay, state=s, return_state=True)
    for t in range(87, 90):
        o = sequence.leaky_attention_step(q[t], k[t], v[t], decay, state)
    size, size_last = leaky_ref(q.abs(), k.abs(), v.abs(), decay, 40 ** -0.5, s.abs())
    within(o, want[-1], size[-1] * 2 * 400 * U, 'o')
    within(state, want_last, size_last * 2 * 400 * U, 'state')


def test_step_notices_autograd():
    q, k, v, decay, s, _ = (t.to(DEV) if t is not None else None for t in leaky_case(1, 1, 1, 1, 8, 8, torch.float32, True, False))
    q.requires_grad_()
    o = sequence.leaky_attention(q, k, v, decay, state=s)
    sequence.leaky_attention_step(q.detach()[0], k[0], v[0], decay, s)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        o.sum().backward()


# ----------------------------------------------------------------------------------------------------------------------------------------------------------
# add + root-mean-square norm
# ----------------------------------------------------------------------------------------------------------------------------------------------------------
WIDTHS = [1, 7, 8, 63, 64, 100, 512, 513, 1000, 1024, 2048, 4096, 5000, 8192, 16383, 16384]
# a sum of squares: at most 64 values in a row and 26 levels of threads; half of that in its root, and a few roundings after it
NORM_ROOM = 55 * U


def norm_case(rows, C, dtype, residual, seed=0):
    g = gen(seed)
    x, w = normal(g, rows, C, dtype=dtype), 1 + normal(g, C, std=0.2)
    return x, w, normal(g, rows, C, dtype=dtype, std=2.) if residual else None


def norm_ref(x, w, r, eps):
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    d = h.double()
    return h, d, (d.square().mean(-1, keepdim=True) + eps).rsqrt()


@pytest.mark.parametrize('residual', [True, False])
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('C', WIDTHS)
def test_norm_and_gradients(C, dtype, residual):
    for rows in (1, 5, 1030 if C <= 2048 else 6):
        x, w, r = norm_case(rows, C, dtype, residual, seed=C)
        use = [t.to(DEV).requires_grad_() if t is not None else None for t in (x, r, w)]
        y, h = sequence.add_rms_norm(use[0], use[2], use[1], eps=1e-5)
        hr, d, rstd = norm_ref(x, w, r, 1e-5)
        assert torch.equal(h.detach().cpu(), hr) and y.dtype == dtype
        n = d * rstd
        within(y, n * w.double(), (n * w.double()).abs() * (NORM_ROOM + HALF[dtype] * 1.01) + TINY[dtype], f'y {rows}')
        g = gen(rows)
        gy, gh = normal(g, rows, C, dtype=dtype), normal(g, rows, C, dtype=dtype)
        outs, gs = ([y, h], [gy.to(DEV), gh.to(DEV)]) if residual else ([y], [gy.to(DEV)])
        got = torch.autograd.grad(outs, [t for t in use if t is not None], gs)
        gw = gy.double() * w.double()
        dot, dot_size = (gw * n).mean(-1, keepdim=True), (gw * n).abs().mean(-1, keepdim=True)
        want = rstd * (gw - n * dot) + (gh.double() if residual else 0)
        size = rstd * (gw.abs() + n.abs() * dot_size) + (gh.double().abs() if residual else 0)
        for a in got[:-1]:
            within(a, want, size * 3 * NORM_ROOM + want.abs() * HALF[dtype] * 1.01 + TINY[dtype], f'gradient of h {rows}')
        # rows of a block one after the other, the blocks in 32 slices
        within(got[-1], (gy.double() * n).sum(0), (gy.double() * n).abs().sum(0) * (rows + 70 + 60) * U + 1e-30, f'gradient of the weight {rows}')


def test_norm_gradient_against_differences():
    x, w, r = (t.double() for t in norm_case(4, 40, torch.float32, True, seed=1))
    use = [t.float().to(DEV).requires_grad_() for t in (x, r, w)]
    y, h = sequence.add_rms_norm(use[0], use[2], use[1])
    g = gen(4)
    wy, wh = normal(g, 4, 40).double(), normal(g, 4, 40).double()
    got = torch.autograd.grad([y, h], use, [wy.float().to(DEV), wh.float().to(DEV)])

    def loss(x, r, w):
        d = x + r
        return ((d * (d.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w) * wy).sum() + (d * wh).sum()

    base, step = [x, r, w], 1e-5
    for i, grad in enumerate(got):
        d = normal(g, *base[i].shape).double()
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + step * d, base[i] - step * d
        along = grad.cpu().double() * d
        # fp32 roundings, the rounding of x + r (2^-24 of it), and the difference's own error: step^2 times a third derivative of order one per value
        assert abs(along.sum() - (loss(*up) - loss(*down)) / (2 * step)) <= (4 * NORM_ROOM + 1e-9) * 10 * along.abs().sum()


@pytest.mark.parametrize('dtype', DTYPES)
def test_norm_strided_rows_and_alignment(dtype):
    g = gen(3)
    big, w = normal(g, 9, 3, 130, dtype=dtype).to(DEV), (1 + normal(g, 128, std=0.1)).to(DEV)
    for cut in (slice(0, 128), slice(1, 129), slice(2, 130)):
        x, r = big[:, 0, cut], big[:, 2, cut]
        a, b = sequence.add_rms_norm(x, w, r), sequence.add_rms_norm(x.contiguous(), w, r.contiguous())
        assert torch.equal(a[1], b[1])
        within(a[0], b[0], b[0].double().abs() * (2 * NORM_ROOM + 2.02 * HALF[dtype]) + 2 * TINY[dtype], 'strided')
        c, d = sequence.add_rms_norm_int8(x, w, r), sequence.add_rms_norm_int8(x.contiguous(), w, r.contiguous())
        assert torch.equal(c[0], d[0]) and torch.equal(c[2], d[2])
    assert sequence.add_rms_norm(big[:, :, :128].reshape(3, 9, 128), w)[0].shape == (3, 9, 128)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_norm_range(dtype):
    """Values whose squares leave fp32's range on either side."""
    g = gen(6)
    for size in (1e25, 1e-25):
        x = (normal(g, 3, 200) * size).to(dtype)
        w = 1 + normal(g, 200, std=0.1)
        y, _ = sequence.add_rms_norm(x.to(DEV), w.to(DEV), eps=0.)
        _, d, rstd = norm_ref(x, w, None, 0.)
        want = d * rstd * w.double()
        within(y, want, want.abs() * (NORM_ROOM + HALF[dtype] * 1.01), f'y at {size}')
        codes, scales, _ = sequence.add_rms_norm_int8(x.to(DEV), w.to(DEV), eps=0.)
        u = d * w.double()
        assert torch.equal(codes.cpu().double(), torch.round(u * 127. / u.abs().amax(-1, keepdim=True)))
    zero = torch.zeros(2, 64, dtype=dtype, device=DEV)
    assert not sequence.add_rms_norm(zero, torch.ones(64, device=DEV))[0].any()


@pytest.mark.parametrize('residual', [True, False])
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('C', WIDTHS)
def test_norm_int8(C, dtype, residual):
    for rows in (1, 5, 1030 if C <= 2048 else 6):
        x, w, r = norm_case(rows, C, dtype, residual, seed=C + 1)
        codes, scales, h = sequence.add_rms_norm_int8(x.to(DEV), w.to(DEV), None if r is None else r.to(DEV))
        hr, d, rstd = norm_ref(x, w, r, 1e-6)
        assert torch.equal(h.cpu(), hr)
        u = d * w.double()
        top = u.abs().amax(-1, keepdim=True)
        assert codes.dtype == torch.int8 and torch.equal(codes.cpu().double(), torch.round(u * 127. / top.clamp_min(1e-300)))         # (a row of zeros has codes 0)
        want = (top * rstd / 127.)[:, 0]
        within(scales, want, want * NORM_ROOM, 'scales')
        back = sequence.dequantize_int8(codes, scales, dtype)
        values = codes.cpu().double() * scales.cpu().double()[:, None]
        within(back, values, values.abs() * (HALF[dtype] + U) * 1.01 + TINY[dtype], 'values')


@pytest.mark.parametrize('dtype', DTYPES)
def test_norm_int8_keeps_the_sum_in_the_graph(dtype):
    """h is handed on to the next layer's residual: its gradient reaches x and residual as an addition's does, with a residual as without."""
    x, w, r = (t.to(DEV) for t in norm_case(5, 72, dtype, True, seed=2))
    g = normal(gen(3), 5, 72, dtype=dtype).to(DEV)
    plain = sequence.add_rms_norm_int8(x, w, r)
    for need in ((True, True), (True, False), (False, True)):
        a, b, wl = x.clone().requires_grad_(need[0]), r.clone().requires_grad_(need[1]), w.clone().requires_grad_()
        codes, scales, h = sequence.add_rms_norm_int8(a, wl, b)
        for got, want in zip((codes, scales, h), plain):
            assert torch.equal(got, want)
        assert h.requires_grad and not scales.requires_grad
        for got in torch.autograd.grad(h, [t for t in (a, b) if t.requires_grad], g, retain_graph=True):
            assert torch.equal(got, g)
        h.sum().backward()
        assert wl.grad is None
    a = x.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(sequence.add_rms_norm_int8(a, w)[2], a, g)[0], g)
    assert torch.equal(torch.autograd.grad(sequence.add_rms_norm_int8(a, w, a)[2], a, g)[0], g + g)
    assert not sequence.add_rms_norm_int8(x, w.clone().requires_grad_(), r)[2].requires_grad


def test_norm_int8_ties_zeros_and_what_is_not_finite():
    x = torch.zeros(6, 64)
    x[0, 0], x[0, 1:8] = 127., torch.tensor([0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5])         # a code's step is 1: ties, to even
    x[1] = x[0] * 2. ** 40
    x[2, 0], x[2, 1:8] = -127., x[0, 1:8]
    x[4, 3], x[5, 3] = math.nan, -math.inf
    x[4, 5] = x[5, 5] = 1.
    for dtype in DTYPES:
        if dtype == torch.float16:
            x[1] = x[0] * 2. ** 8
        codes, scales, _ = sequence.add_rms_norm_int8(x.to(dtype).to(DEV), torch.ones(64, device=DEV))
        xd = x.to(dtype).double()
        want = torch.round(xd[:3] * 127 / xd[:3].abs().amax(-1, keepdim=True))
        assert torch.equal(codes[:3].cpu().double(), want)
        assert not codes[3:].any() and scales[3] == 0 and scales[4:].isnan().all() and scales[:3].isfinite().all()


@pytest.mark.parametrize('C', [5, 64, 1000, 1500, 5000])
def test_norm_int8_of_weights_that_are_not_finite(C):
    """h * weight that is not a number, from either side, shows in every row: codes 0, scale NaN, as where h holds one."""
    x, w, _ = norm_case(6, C, torch.float32, False, seed=C)
    x[3, C - 2] = 0.
    for at, bad in ((C - 1, math.nan), (C // 2, math.nan), (C - 2, math.inf), (0, -math.inf)):
        wb = w.clone()
        wb[at] = bad
        for dtype in DTYPES:
            codes, scales, _ = sequence.add_rms_norm_int8(x.to(dtype).to(DEV), wb.to(DEV))
            assert not codes.any() and scales.isnan().all(), (at, bad, dtype)
            assert sequence.dequantize_int8(codes, scales).isnan().all()


@pytest.mark.parametrize('C', [64, 1500])
@pytest.mark.parametrize('size', [1e25, 1e36])
def test_norm_int8_of_products_beyond_fp32(C, size):
    """Finite values whose products with the weight pass fp32's largest number: the norm is within it, so codes and scale are."""
    x, w, _ = norm_case(4, C, torch.float32, False, seed=C)
    x, w = x * size, w * 1e15
    codes, scales, _ = sequence.add_rms_norm_int8(x.to(DEV), w.to(DEV))
    d = x.double()
    u = d * w.double()
    top = u.abs().amax(-1, keepdim=True)
    assert top.max() > 3.5e38 and torch.equal(codes.cpu().double(), torch.round(u * 127. / top))
    want = (top * (d.square().mean(-1, keepdim=True) + 1e-6).rsqrt() / 127.)[:, 0]
    within(scales, want, want * NORM_ROOM, 'scales')


# ----------------------------------------------------------------------------------------------------------------------------------------------------------
# 8-bit integer product
# ----------------------------------------------------------------------------------------------------------------------------------------------------------
def product_case(M, N, K, bias, seed=0, full=False):
    g = gen(seed)
    lo, hi = (-128, 128)
    a, w = (torch.randint(lo, hi, s, generator=g, dtype=torch.int32).to(torch.int8) for s in ((M, K), (N, K)))
    return a, torch.rand(M, generator=g) + 0.01, w, torch.rand(N, generator=g) + 0.01, normal(g, N, std=1000.) if bias else None


def product_check(M, N, K, bias, out, seed=0):
    a, sa, w, sw, b = product_case(M, N, K, bias, seed)
    got = sequence.int8_linear(a.to(DEV), sa.to(DEV), w.to(DEV), sw.to(DEV), None if b is None else b.to(DEV), out)
    acc = a.double() @ w.double().t()
    y = acc * sa.double()[:, None] * sw.double()
    want = y if b is None else y + b.double()
    # what rounds beyond fp16's largest number, 65504 (from 65520 on), is an infinity there
    over = want.abs() > 65520 * (1 + 8 * U) if out == torch.float16 else torch.zeros_like(want, dtype=torch.bool)
    assert torch.equal(got.cpu().double()[over], want[over].sign() * math.inf)
    got, y, want = got.cpu().masked_fill(over, 0), y.masked_fill(over, 0), want.masked_fill(over, 0)
    # the integer to fp32, two scales, the bias; then the output's rounding
    within(got, want, y.abs() * 3.1 * U + want.abs() * (HALF[out] * 1.01 + U) + TINY[out], f'{M} x {N} x {K}')
    assert got.dtype == out


@pytest.mark.parametrize('K', [1, 15, 16, 17, 48, 64, 100, 128, 144, 1000, 4096])
@pytest.mark.parametrize('M', [1, 2, 5, 16, 17, 33, 64, 65, 130, 300])
def test_int8_linear(M, K):
    for N in (1, 8, 17, 64, 100, 257):
        product_check(M, N, K, bias=(M + N) % 2 == 0, out=DTYPES[(M + N + K) % 3], seed=M + N + K)


@pytest.mark.parametrize('shape', [(1, 8192, 512), (4, 2048, 4608), (700, 512, 4608), (513, 1025, 2064), (2100, 600, 320), (1100, 1300, 77), (66000, 8, 32)])
def test_int8_linear_larger(shape):
    a, sa, w, sw, b = product_case(*shape, True, seed=1)
    got = sequence.int8_linear(a.to(DEV), sa.to(DEV), w.to(DEV), sw.to(DEV), b.to(DEV))
    y = (a.to(DEV).double() @ w.to(DEV).double().t()) * sa.to(DEV).double()[:, None] * sw.to(DEV).double()
    want = y + b.to(DEV).double()
    within(got, want, y.abs() * 3.1 * U + want.abs() * 2 * U + 1e-30, str(shape))


@pytest.mark.parametrize('shape', [(3500, 3333, 400), (3500, 3333, 387), (3400, 3584, 640), (3329, 3329, 128), (3400, 3590, 1000)])
@pytest.mark.parametrize('out', DTYPES)
def test_int8_linear_in_tiles_of_256(shape, out):
    """At least 176 tiles of 256 x 256: several k steps and a partial one, rows copied to alignment, element stores, each type, with a bias and without."""
    M, N, K = shape
    assert -(-M // 256) * -(-N // 256) >= 176
    a, sa, w, sw, b = (t.to(DEV) for t in product_case(M, N, K, True, seed=K))
    y = (a.double() @ w.double().t()) * sa.double()[:, None] * (sw.double() / 512)
    for bias in (None, b / 512):
        got = sequence.int8_linear(a, sa, w, sw / 512, bias, out)
        want = y if bias is None else y + bias.double()
        if out == torch.float16:
            assert want.abs().max() < 65504
        within(got, want, y.abs() * 3.1 * U + want.abs() * (HALF[out] * 1.01 + U) + TINY[out], f'{shape}, bias {bias is not None}')


def test_int8_linear_extreme_sums_and_strides():
    K = 131071
    a, w = torch.full((3, K), -128, dtype=torch.int8, device=DEV), torch.full((2, K), -128, dtype=torch.int8, device=DEV)
    w[1] = 127
    got = sequence.int8_linear(a, torch.ones(3, device=DEV), w, torch.ones(2, device=DEV))
    want = torch.tensor([128. * 128 * K, -128. * 127 * K], dtype=torch.float64)
    within(got, want.expand(3, 2), want.abs().expand(3, 2) * 4 * U, 'extreme')
    g = gen(5)
    x = torch.randint(-128, 128, (40, 2, 300), generator=g, dtype=torch.int32).to(torch.int8).to(DEV)
    w = torch.randint(-128, 128, (33, 300), generator=g, dtype=torch.int32).to(torch.int8).to(DEV)
    s, sw = torch.rand(40, generator=g).to(DEV), torch.rand(33, generator=g).to(DEV)
    for cut in (slice(0, 256), slice(1, 257), slice(3, 290)):
        assert torch.equal(sequence.int8_linear(x[:, 1, cut], s, w[:, cut], sw), sequence.int8_linear(x[:, 1, cut].contiguous(), s, w[:, cut].contiguous(), sw))
    out = sequence.int8_linear(x[:, :, :256], torch.stack((s, s), 1), w[:, :256], sw)                     # leading axes are kept
    assert out.shape == (40, 2, 33) and torch.equal(out[:, 1], sequence.int8_linear(x[:, 1, :256], s, w[:, :256], sw))


# ----------------------------------------------------------------------------------------------------------------------------------------------------------
# together, streams, graphs
# ----------------------------------------------------------------------------------------------------------------------------------------------------------
class Block(torch.nn.Module):
    """A pre-norm sequence layer for serving: norm in 8 bits -> projections -> leaky attention -> projection; the sum is handed on."""

    def __init__(self, width, heads, dk, dv):
        super().__init__()
        self.norm, self.att = layer.AddRMSNorm(width), layer.LeakyAttention(heads)
        self.q, self.k = (layer.Int8Linear(torch.nn.Linear(width, heads * dk, bias=False), torch.bfloat16) for _ in range(2))
        self.v = layer.Int8Linear(torch.nn.Linear(width, heads * dv, bias=False), torch.bfloat16)
        self.norm_o, self.o = layer.AddRMSNorm(heads * dv), layer.Int8Linear(torch.nn.Linear(heads * dv, width), torch.bfloat16)
        self.heads, self.dk, self.dv = heads, dk, dv

    def forward_sequence(self, x, residual):
        c, s, h = self.norm.forward_int8(x, residual)
        q, k, v = self.q(c, s).unflatten(-1, (self.heads, self.dk)), self.k(c, s).unflatten(-1, (self.heads, self.dk)), self.v(c, s).unflatten(-1, (self.heads, self.dv))
        o = self.att.forward_sequence(q, k, v) if x.dim() == 3 else self.att(q, k, v)
        c, s, _ = self.norm_o.forward_int8(o.flatten(-2))
        return self.o(c, s), h


def test_block_sequence_equals_steps_and_the_definition():
    torch.manual_seed(0)
    T, B, W, H, D = 70, 2, 96, 3, 32
    block = Block(W, H, D, D).to(DEV)
    g = gen(1)
    x, r = normal(g, T, B, W, dtype=torch.bfloat16).to(DEV), normal(g, T, B, W, dtype=torch.bfloat16).to(DEV)
    with torch.no_grad():
        y, h = block.forward_sequence(x, r)
        last = block.att.s.clone()
        functional.reset_net(block)
        steps = torch.stack([block.forward_sequence(x[t], r[t])[0] for t in range(T)])
    # the norms, products and codes before the attention are the same numbers; the attention's outputs differ by the tile form's roundings (2 * 2^-8 of the
    # terms), which may move a code of the second norm by one: 1 / 127 of a row's largest value, against sums of 96 of them
    assert (y.float() - steps.float()).square().mean().sqrt() <= 0.02 * y.float().square().mean().sqrt()
    assert torch.allclose(last, block.att.s, rtol=1e-4, atol=1e-3)
    # the definition in fp64, with the same codes
    with torch.no_grad():
        c, s, _ = block.norm.forward_int8(x, r)
        n = c.cpu().double() * s.cpu().double()[..., None]
        lin = lambda l, z: z @ (l.weight.cpu().double() * l.weight_scale.cpu().double()[:, None]).t() + (0 if l.bias is None else l.bias.cpu().double())   # noqa: E731
        q, k, v = (lin(l, n).unflatten(-1, (H, D)) for l in (block.q, block.k, block.v))
        o = leaky_ref(q, k, v, block.att.log_decay, D ** -0.5)[0].flatten(-2)
        o = o / (o.square().mean(-1, keepdim=True) + 1e-6).sqrt()
        want = lin(block.o, o)
    # bf16 roundings of q, k, v, o and y (five halves of 2^-8) and the second norm's codes (uniform within half of 1/127 of the row's largest, about three
    # times its rms): 5 * 2^-9 + 3 / 127 / sqrt(12) of the rms
    assert (y.cpu().double() - want).square().mean().sqrt() <= 0.03 * want.square().mean().sqrt()


def test_training_block_gradients():
    """Norm -> projections -> leaky attention -> projection in fp32, its gradients against the definition's in fp64."""
    torch.manual_seed(1)
    T, B, W, H, D = 66, 2, 24, 2, 16
    g = gen(2)
    x, r = normal(g, T, B, W), normal(g, T, B, W)
    wq, wk, wv, wo = (normal(g, H * D, W, std=0.2) for _ in range(3)), None, None, normal(g, W, H * D, std=0.2)
    wq, wk, wv = tuple(wq)
    nw = 1 + normal(g, W, std=0.1)
    decay = torch.tensor([-0.02, -0.3])

    def run(x, r, nw, wq, wk, wv, wo, norm, att):
        n, h = norm(x, nw, r)
        q, k, v = ((n @ w.t()).unflatten(-1, (H, D)) for w in (wq, wk, wv))
        return att(q, k, v).flatten(-2) @ wo.t() + h

    leaves = (x, r, nw, wq, wk, wv, wo)
    ours = [t.to(DEV).requires_grad_() for t in leaves]
    y = run(*ours, sequence.add_rms_norm, lambda q, k, v: sequence.leaky_attention(q, k, v, decay.to(DEV)))
    ref = [t.double().requires_grad_() for t in leaves]
    norm64 = lambda x, w, r: ((x + r) * ((x + r).square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w, x + r)     # noqa: E731
    want = run(*ref, norm64, lambda q, k, v: leaky_ref(q, k, v, decay, D ** -0.5)[0])
    gy = normal(g, T, B, W)
    got, exp = torch.autograd.grad(y, ours, gy.to(DEV)), torch.autograd.grad(want, ref, gy.double())
    # chains of some 500 fp32 roundings, largely independent: 500 * u of the gradient's own norm is their worst case with a tenfold cancellation to spare
    for a, b in zip((y, *got), (want, *exp)):
        assert (a.cpu().double() - b).norm() <= 5000 * U * b.norm()


def test_nothing_to_do():
    """No step, no stream, no row: the shapes, and no launch."""
    q, g = torch.zeros(3, 2, 4, 8, device=DEV), torch.zeros(4, device=DEV)
    k, v = torch.zeros(3, 2, 2, 8, device=DEV), torch.zeros(3, 2, 2, 6, device=DEV)
    s = torch.ones(2, 4, 8, 6, device=DEV)
    o, last = sequence.leaky_attention(q[:0], k[:0], v[:0], g, state=s, return_state=True)
    assert o.shape == (0, 2, 4, 6) and torch.equal(last, s)
    assert sequence.leaky_attention(q[:, :0], k[:, :0], v[:, :0], g).shape == (3, 0, 4, 6)
    assert sequence.leaky_attention_step(q[0, :0], k[0, :0], v[0, :0], g, s[:0]).shape == (0, 4, 6)
    x, w = torch.zeros(3, 8, device=DEV, requires_grad=True), torch.ones(8, device=DEV, requires_grad=True)
    y, _ = sequence.add_rms_norm(x[:0], w)
    assert y.shape == (0, 8) and not torch.autograd.grad(y.sum(), w)[0].any()
    assert [t.shape for t in sequence.add_rms_norm_int8(x[:0], w, x[:0])] == [(0, 8), (0,), (0, 8)]
    c = torch.zeros(0, 8, dtype=torch.int8, device=DEV)
    assert sequence.int8_linear(c, torch.ones(0, device=DEV), torch.zeros(5, 8, dtype=torch.int8, device=DEV), torch.ones(5, device=DEV)).shape == (0, 5)
    assert sequence.dequantize_int8(c, torch.ones(0, device=DEV)).shape == (0, 8)


@pytest.mark.parametrize('dtype', DTYPES)
def test_gradients_of_nothing_to_do(dtype):
    """No step or no stream under autograd: gradients of the operands' shapes, the state's is the last state's."""
    q, k, v, decay, s, _ = (t.to(DEV) if t is not None else None for t in leaky_case(3, 2, 4, 2, 8, 6, dtype, True, False))
    for cut in ((slice(0, 0), slice(None)), (slice(None), slice(0, 0)), (slice(0, 0), slice(0, 0))):
        use = [t[cut].clone().requires_grad_() for t in (q, k, v)]
        state = s[cut[1]].clone().requires_grad_()
        o, last = sequence.leaky_attention(*use, decay, state=state, return_state=True)
        assert torch.equal(last, state) and o.shape == (*use[0].shape[:3], 6) and o.dtype == dtype
        g = torch.randn_like(last)
        got = torch.autograd.grad([o, last], [*use, state], [torch.ones_like(o), g], retain_graph=True)
        assert [t.shape for t in got[:3]] == [t.shape for t in use] and torch.equal(got[3], g)
        assert not torch.autograd.grad(o.sum(), state, retain_graph=True)[0].any()
        assert torch.autograd.grad(sequence.leaky_attention(*use, decay).sum(), use[1])[0].shape == use[1].shape


def test_refusals_on_the_device():
    """The library hands unfit operands back before it launches; the error names the operand."""
    q, g = torch.zeros(3, 2, 4, 8, device=DEV), torch.zeros(4, device=DEV)
    for bad, what in (((q, q[:2], q, g), 'k: expected shape'), ((q, q.half(), q, g), 'k: expected'), ((q, q, q.cpu(), g), 'v'), ((q, q, q, g[:2]), 'log_decay'),
                      ((q, q, q, g.clone().requires_grad_()), 'no gradient'), ((q, q, None, g), 'v')):
        with pytest.raises(sequence.SSNeuronError, match=what):
            sequence.leaky_attention(*bad)
    with pytest.raises(sequence.SSNeuronError, match='contiguous'):
        sequence.leaky_attention_step(q[0], q[0], q[0], g, torch.zeros(2, 4, 8, 8, device=DEV).transpose(2, 3))
    with pytest.raises(sequence.SSNeuronError, match='weight'):
        sequence.add_rms_norm(q, torch.ones(8, device=DEV).half())
    with pytest.raises(sequence.SSNeuronError, match='scales'):
        sequence.int8_linear(q.to(torch.int8), torch.ones(3, device=DEV), torch.zeros(5, 8, dtype=torch.int8, device=DEV), torch.ones(5, device=DEV))


def test_a_product_of_too_many_outputs_is_refused_by_name_on_the_device():
    a, s = torch.zeros(1, 16, dtype=torch.int8, device=DEV).expand(2 ** 19, 16), torch.ones(1, device=DEV).expand(2 ** 19)
    with pytest.raises(sequence.SSNeuronError, match='524288 rows by 524288 channels'):
        sequence.int8_linear(a, s, a, s)


def test_tracers_and_forward_mode_are_refused_on_the_device():
    q, g = torch.randn(3, 2, 2, 8, device=DEV), torch.zeros(2, device=DEV)
    x, c, one = torch.randn(3, 8, device=DEV), torch.zeros(3, 8, dtype=torch.int8, device=DEV), torch.ones(3, device=DEV)
    w, sw, ones = torch.zeros(5, 8, dtype=torch.int8, device=DEV), torch.ones(5, device=DEV), torch.ones(8, device=DEV)
    s = torch.zeros(2, 2, 8, 8, device=DEV)
    for call, t in ((lambda t: sequence.leaky_attention(q, t, q, g), q), (lambda t: sequence.leaky_attention(q, q, q, t), g), (lambda t: sequence.leaky_attention(q, q, q, g, state=t), s),
                    (lambda t: sequence.leaky_attention_step(t, q[0], q[0], g, s.clone()), q[0]), (lambda t: sequence.add_rms_norm(t, ones)[0], x),
                    (lambda t: sequence.add_rms_norm(x, ones, t)[1], x), (lambda t: sequence.add_rms_norm_int8(x, ones, t)[2], x),
                    (lambda t: sequence.dequantize_int8(c, t), one), (lambda t: sequence.int8_linear(c, one, w, sw, t), sw)):
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(sequence.SSNeuronError, match='no forward-mode'):
                call(torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(sequence.SSNeuronError, match='cannot be traced'):
            torch.jit.trace(call, (t,))
        with pytest.raises(sequence.SSNeuronError, match='cannot be traced'):
            torch.fx.experimental.proxy_tensor.make_fx(call)(t)
        call(t)                                            # and nothing of it stays behind


def test_values_of_codes_under_autograd_are_refused_on_the_device():
    c, s = torch.ones(3, 8, dtype=torch.int8, device=DEV), torch.ones(3, device=DEV, requires_grad=True)
    with pytest.raises(sequence.SSNeuronError, match='dequantize_int8 has no gradient'):
        sequence.dequantize_int8(c, s)
    with torch.no_grad():
        assert torch.equal(sequence.dequantize_int8(c, s), c.float())


def test_gradients_are_not_differentiated_again():
    q = torch.randn(4, 1, 1, 8, device=DEV, requires_grad=True)
    o = sequence.leaky_attention(q, q, q, torch.zeros(1, device=DEV))
    first, = torch.autograd.grad(o.square().sum(), q, create_graph=True)
    plain, = torch.autograd.grad(sequence.leaky_attention(q, q, q, torch.zeros(1, device=DEV)).square().sum(), q)
    assert torch.equal(first, plain)
    with pytest.raises(RuntimeError, match='differentiate twice'):
        first.sum().backward()
    w = torch.ones(8, device=DEV, requires_grad=True)
    y, _ = sequence.add_rms_norm(q, w)
    first, = torch.autograd.grad(y.square().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match='differentiate twice'):
        first.sum().backward()


def test_other_stream_and_repeat():
    """On a side stream, and twice on the same inputs: the same bits."""
    q, k, v, decay, s, _ = (t.to(DEV) if t is not None else None for t in leaky_case(300, 2, 4, 2, 64, 64, torch.bfloat16, True, False))
    use = [t.requires_grad_() for t in (q, k, v)]
    g = normal(gen(1), 300, 2, 4, 64, dtype=torch.bfloat16).to(DEV)

    def once():
        o = sequence.leaky_attention(*use, decay, state=s)
        return (o, *torch.autograd.grad(o, use, g))

    want = once()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = once()
    side.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_captured_calls_replay():
    """A serving step (norm, product, attention step) and a prompt in two graphs, replayed in turn with eager work between: every replay is the eager result."""
    torch.manual_seed(2)
    block = Block(64, 2, 32, 32).to(DEV)
    g = gen(3)
    xs, rs = normal(g, 4, 3, 64, dtype=torch.bfloat16).to(DEV), normal(g, 4, 3, 64, dtype=torch.bfloat16).to(DEV)
    ps, pr = normal(g, 100, 3, 64, dtype=torch.bfloat16).to(DEV), normal(g, 100, 3, 64, dtype=torch.bfloat16).to(DEV)
    x, r, px, pres = xs[0].clone(), rs[0].clone(), ps.clone(), pr.clone()
    state = torch.zeros(3, 2, 32, 32, device=DEV)

    def step():
        block.att.s = state
        return block.forward_sequence(x, r)[0]

    def prompt():
        block.att.s = None
        y = block.forward_sequence(px, pres)[0]
        return y, block.att.s

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        step(), prompt()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    gs, gp = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.no_grad():
        with torch.cuda.graph(gs):
            ys = step()
        with torch.cuda.graph(gp):
            yp, sp = prompt()
        state.zero_()
        eager_state = torch.zeros_like(state)
        for t in range(4):
            x.copy_(xs[t]), r.copy_(rs[t]), px.copy_(ps.roll(t, 0)), pres.copy_(pr.roll(t, 0))
            gp.replay()
            gs.replay()
            torch.cuda.synchronize()
            block.att.s = eager_state
            want = block.forward_sequence(xs[t], rs[t])[0]
            assert torch.equal(ys, want) and torch.equal(state, eager_state)
            wp, ws = prompt()
            assert torch.equal(yp, wp) and torch.equal(sp, ws)


def test_captured_gradients_replay():
    """Attention -> add + norm and all their gradients in one graph, on leaves of its own; replayed with eager passes between: the eager result each time."""
    g = gen(16)
    T, B, H, D = 90, 2, 4, 32
    sets = [[normal(g, T, B, n, D, dtype=torch.bfloat16).to(DEV) for n in (H, 2, 2, H, H)] + [normal(g, B, H, D, D).to(DEV) for _ in range(2)] for _ in range(3)]
    data, w, decay = [t.clone() for t in sets[0]], (1 + normal(g, D, std=0.1)).to(DEV), torch.tensor([-0.01, -0.1, -0.5, 0.], device=DEV)

    def run(q, k, v, gy, gh, s, gl):
        q, k, v, s, wl = (t.detach().requires_grad_() for t in (q, k, v, s, w))
        o, last = sequence.leaky_attention(q, k, v, decay, state=s, return_state=True)
        y, h = sequence.add_rms_norm(o, wl, q)
        return (y.detach(), h.detach(), last.detach(), *torch.autograd.grad([y, h, last], [q, k, v, s, wl], [gy, gh, gl]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*data)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(*data)
    for new in (*sets, *sets[:2]):
        for a, b in zip(data, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, run(*new)):
            assert torch.equal(a, b)


def test_captured_gradients_beside_a_living_eager_graph():
    """A training step captured on aliases of its leaves while an eager graph of the leaves themselves lives: each replay, and the eager backward after it, is right."""
    g = gen(20)
    q, k, v = (normal(g, 40, 2, 2, 32).to(DEV).requires_grad_() for _ in range(3))
    w, decay = (1 + normal(g, 32, std=0.1)).to(DEV).requires_grad_(), torch.tensor([-0.1, -0.01], device=DEV)
    go = normal(g, 40, 2, 2, 32).to(DEV)

    def run(q, k, v, w):
        return sequence.add_rms_norm(sequence.leaky_attention(q, k, v, decay), w)[0]

    eager = run(q, k, v, w)

    def step():
        use = [t.detach().requires_grad_() for t in (q, k, v, w)]
        return torch.autograd.grad(run(*use), use, go)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    want = torch.autograd.grad(eager, (q, k, v, w), go, retain_graph=True)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    for a, b in zip(torch.autograd.grad(eager, (q, k, v, w), go), want):
        assert torch.equal(a, b)


# ----------------------------------------------------------------------------------------------------------------------------------------------------------
# offsets that pass 32 bits: what the same values give in a small tensor
# ----------------------------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', DTYPES)
def test_far_steps_of_attention(dtype):
    T, D, step = 36, 64, 1 << 26
    far = torch.empty(T * step, dtype=dtype, device=DEV)
    q, k, v, go = (far.as_strided((T, 2, 1, D), (step, step // 2, D, 1), 8 * D * i) for i in range(4))
    g = gen(17)
    for t in (q, k, v, go):
        t.copy_(normal(g, T, 2, 1, D))
    decay, near = torch.tensor([-0.05], device=DEV), [t.contiguous() for t in (q, k, v, go)]

    def run(q, k, v, go):
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        o = sequence.leaky_attention(q, k, v, decay)
        return (o.detach(), *torch.autograd.grad(o, (q, k, v), go))

    for a, b in zip(run(q, k, v, go), run(*near)):
        assert torch.equal(a, b)
    for a, b in zip(run(q[::7], k[::7], v[::7], go[::7]), run(*(t[::7] for t in near))):
        assert torch.equal(a, b)


def test_far_states_of_steps():
    B, H, D = 200, 170, 256
    q, k, v = (normal(gen(i), B, H, D, dtype=torch.bfloat16).to(DEV) for i in range(3))
    state, decay = torch.empty(B, H, D, D, device=DEV), torch.full((H,), -0.1, device=DEV)
    state[-1] = normal(gen(3), H, D, D).to(DEV)
    last = state[-1:].clone()
    o = sequence.leaky_attention_step(q, k, v, decay, state)
    assert torch.equal(o[-1:], sequence.leaky_attention_step(q[-1:], k[-1:], v[-1:], decay, last)) and torch.equal(state[-1:], last)


def test_far_rows_of_norm_and_product():
    g = torch.Generator(device=DEV).manual_seed(18)
    M, K = 540000, 4096
    x = torch.empty(M, K, dtype=torch.bfloat16, device=DEV)
    x[-100:] = torch.randn(100, K, generator=g, device=DEV)
    x[:-100] = x[-100:].repeat(5399, 1)
    w = torch.rand(K, generator=g, device=DEV)
    y, h = sequence.add_rms_norm(x, w, x)
    ye, he = sequence.add_rms_norm(x[-100:], w, x[-100:])
    assert torch.equal(y[-100:], ye) and torch.equal(h[-100:], he) and torch.equal(y[:100], ye)
    del y, h
    c, s, h = sequence.add_rms_norm_int8(x, w)
    ce, se, _ = sequence.add_rms_norm_int8(x[-100:], w)
    assert torch.equal(c[-100:], ce) and torch.equal(s[-100:], se)
    d = sequence.dequantize_int8(c, s, torch.bfloat16)
    assert torch.equal(d[-100:], sequence.dequantize_int8(ce, se, torch.bfloat16))
    del d, x, h
    wc = torch.randint(-128, 128, (24, K), generator=g, device=DEV, dtype=torch.int32).to(torch.int8)
    ws = torch.rand(24, generator=g, device=DEV)
    out, few = sequence.int8_linear(c, s, wc, ws), sequence.int8_linear(ce, se, wc, ws)
    assert torch.equal(out[-100:], few) and torch.equal(out[:100], few)
    del c, out
    c = torch.randint(-128, 128, (70000, 16), generator=g, device=DEV, dtype=torch.int32).to(torch.int8)                # an output beyond 32 bits
    wc = torch.randint(-128, 128, (32768, 16), generator=g, device=DEV, dtype=torch.int32).to(torch.int8)
    s, ws = torch.rand(70000, generator=g, device=DEV), torch.rand(32768, generator=g, device=DEV)
    out = sequence.int8_linear(c, s, wc, ws, out_dtype=torch.bfloat16)
    assert torch.equal(out[-50:], sequence.int8_linear(c[-50:], s[-50:], wc, ws, out_dtype=torch.bfloat16))


def test_one_row_expanded():
    """Rows that are all the same memory (a stride of 0)."""
    g = gen(19)
    x, w = normal(g, 1, 64).to(DEV), torch.ones(64, device=DEV)
    for a, b in zip(sequence.add_rms_norm(x.expand(70, 64), w, x.expand(70, 64)), sequence.add_rms_norm(x, w, x)):
        assert torch.equal(a, b.expand(70, 64))
    c, s, _ = sequence.add_rms_norm_int8(x.expand(70, 64), w)
    one, s1, _ = sequence.add_rms_norm_int8(x, w)
    assert torch.equal(c, one.expand(70, 64)) and torch.equal(s, s1.expand(70))
    wc = torch.randint(-128, 128, (5, 64), generator=g, dtype=torch.int32).to(torch.int8).to(DEV)
    want = sequence.int8_linear(one, s1, wc, torch.ones(5, device=DEV))
    assert torch.equal(sequence.int8_linear(one.expand(70, 64), s1.expand(70), wc, torch.ones(5, device=DEV)), want.expand(70, 5))
    assert torch.equal(sequence.int8_linear(one, s1, wc[:1].expand(5, 64), torch.ones(5, device=DEV)), want[:, :1].expand(1, 5))


def test_layer_protocol_on_the_device():
    att = layer.LeakyAttention(2, tau=[2., 50.]).to(DEV)
    q, k, v, _, _, _ = (t.to(DEV) if t is not None else None for t in leaky_case(6, 2, 2, 2, 16, 16, torch.float32, False, False))
    want = sequence.leaky_attention(q, k, v, att.log_decay)
    size = leaky_ref(q.abs(), k.abs(), v.abs(), att.log_decay, 0.25)[0]
    first = att.forward_sequence(q[:3], k[:3], v[:3])
    rest = torch.stack([att(q[t], k[t], v[t]) for t in range(3, 6)])
    within(torch.cat((first, rest)), want, size * 200 * U, 'steps after a sequence')
    functional.reset_net(att)
    x = q.clone().requires_grad_()
    out = torch.stack([att(x[t], k[t], v[t]) for t in range(6)])                 # single steps under autograd: back through time
    assert torch.allclose(torch.autograd.grad(out.sum(), x)[0], torch.autograd.grad(sequence.leaky_attention(x, k, v, att.log_decay).sum(), x)[0], rtol=1e-4, atol=1e-4)
    functional.detach_net(att)
    with pytest.raises(sequence.SSNeuronError, match='reset_net'):
        att(q[0, :1], k[0, :1], v[0, :1])


def test_steps_without_gradients_after_a_training_pass():
    """Steps under no_grad leave the training graph's own state alone, and what is trained after them does not reach behind them."""
    att = layer.LeakyAttention(2, tau=[2., 50.]).to(DEV)
    q, k, v, _, _, _ = (t.to(DEV) if t is not None else None for t in leaky_case(6, 2, 2, 2, 16, 16, torch.float32, False, False))
    first = [t[:3].clone().requires_grad_() for t in (q, k, v)]
    o = att.forward_sequence(*first)
    trained = att.s
    before = trained.detach().clone()
    with torch.no_grad():
        att(q[3], k[3], v[3])
        att(q[4], k[4], v[4])
    assert not att.s.requires_grad and torch.equal(trained, before)
    start = att.s.clone()
    last = [t[5:].clone().requires_grad_() for t in (q, k, v)]
    o2 = att.forward_sequence(*last)
    assert torch.equal(o2, sequence.leaky_attention(*(t.detach() for t in last), att.log_decay, state=start))
    assert all(g is None for g in torch.autograd.grad(o2.sum(), first, retain_graph=True, allow_unused=True))
    got = torch.autograd.grad((o.sum(), trained.sum()), first)                   # the pass before is differentiated as if nothing had come after it
    use = [t.detach().requires_grad_() for t in first]
    want = torch.autograd.grad([t.sum() for t in sequence.leaky_attention(*use, att.log_decay, return_state=True)], use)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_a_step_under_autograd_is_refused_on_the_device():
    q, k, v, decay, s, _ = (t.to(DEV) if t is not None else None for t in leaky_case(1, 2, 2, 2, 16, 16, torch.float32, True, False))
    before = s.clone()
    with pytest.raises(sequence.SSNeuronError, match='step has no gradient'):
        sequence.leaky_attention_step(q[0], k[0].clone().requires_grad_(), v[0], decay, s)
    with torch.no_grad(), pytest.raises(sequence.SSNeuronError, match='state: it is updated in place'):
        sequence.leaky_attention_step(q[0], k[0], v[0], decay, s.clone().requires_grad_())
    with pytest.raises(sequence.SSNeuronError, match='state is on'):
        sequence.leaky_attention_step(q[0], k[0], v[0], decay, None)
    assert torch.equal(s, before)
    with torch.no_grad():                                  # without gradients enabled the operands may require one
        o = sequence.leaky_attention_step(q[0].clone().requires_grad_(), k[0], v[0], decay, s)
    assert not o.requires_grad and torch.equal(o, sequence.leaky_attention_step(q[0], k[0], v[0], decay, before))


def test_layer_of_no_steps():
    """A sequence of no steps leaves the state as it is and gives no outputs, as the function does."""
    att = layer.LeakyAttention(2).to(DEV)
    q, k, v, _, _, _ = (t.to(DEV) if t is not None else None for t in leaky_case(3, 2, 2, 1, 16, 24, torch.bfloat16, False, False))
    assert att.forward_sequence(q[:0], k[:0], v[:0]).shape == (0, 2, 2, 24) and not att.s.any() and att.s.shape == (2, 2, 16, 24)
    att.forward_sequence(q, k, v)
    s = att.s.clone()
    assert att.forward_sequence(q[:0], k[:0], v[:0]).shape == (0, 2, 2, 24) and torch.equal(att.s, s)
    with pytest.raises(sequence.SSNeuronError, match='reset_net'):
        att.forward_sequence(q[:0, :1], k[:0, :1], v[:0, :1])
    for bad in (q[0], q[None]):
        with pytest.raises(sequence.SSNeuronError):
            att.forward_sequence(bad, k, v)


@pytest.mark.parametrize('dtype', DTYPES)
def test_gradients_under_checkpointing_and_saved_tensor_hooks(dtype):
    """What the backward pass needs is saved as tensors are: recomputed (checkpoint) or kept on the host meanwhile, the gradients are bit for bit those without."""
    g = gen(24)
    q, k, v = (normal(g, 300, 2, h, 64, dtype=dtype).to(DEV).transpose(0, 1).contiguous().transpose(0, 1).requires_grad_() for h in (4, 2, 2))
    s, w = normal(g, 2, 4, 64, 64).to(DEV).requires_grad_(), (1 + normal(g, 64, std=0.1)).to(DEV).requires_grad_()
    decay, n = torch.tensor([-0.1, -0.01, -0.5, 0.], device=DEV), torch.tensor([300, 120], dtype=torch.int32, device=DEV)
    leaves = (q, k, v, s, w)

    def run(q, k, v, s, w):
        o, last = sequence.leaky_attention(q, k, v, decay, state=s, lengths=n, return_state=True)
        y, h = sequence.add_rms_norm(o, w, q)
        return y, sequence.add_rms_norm_int8(y, w, h)[2], last

    def grads(outs):
        return torch.autograd.grad(sum(t.float().square().sum() for t in outs), leaves)

    want = grads(run(*leaves))
    with torch.autograd.graph.save_on_cpu():
        kept = run(*leaves)
    for got in (grads(torch.utils.checkpoint.checkpoint(run, *leaves, use_reentrant=False)), grads(kept)):
        for a, b in zip(got, want):
            assert torch.equal(a, b)
