"""CPU suite of the sequence operators: the library's exports and refusals, the Python checks, the layers' state protocol, weight quantisation."""
import ctypes
import math
import os
import re
import subprocess

import pytest
import torch

from stereospike_amd import _seqlib, sequence
from stereospike_amd._lib import SSNeuronError
from stereospike_amd.clock_driven import functional, layer

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


p, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float


class LeakyDesc(ctypes.Structure):
    """struct ss_seq_leaky_desc (include/ss_sequence.h)."""
    _fields_ = ([('size', ctypes.c_uint), ('dtype', i32), ('out_dtype', i32)] + [(n, i32) for n in ('T', 'B', 'H', 'DA', 'DC', 'reverse')] +
                [('b_scale', f32), ('o_scale', f32)] + [(n, p) for n in ('a', 'b', 'c', 'out')] + [(f'{n}_{s}', i64) for n in 'abco' for s in 'tbh'] +
                [(f'{n}_group', i32) for n in 'abc'] + [(n, p) for n in ('log_decay', 'lengths', 's_in', 's_out')] +
                [(n, i32) for n in ('s_in_row', 's_in_col', 's_out_row', 's_out_col')] + [('ws', p)])


class LeakyBwdDesc(ctypes.Structure):
    """struct ss_seq_leaky_bwd_desc (include/ss_sequence.h)."""
    _fields_ = ([('size', ctypes.c_uint)] + [(n, i32) for n in ('dtype', 'T', 'B', 'H', 'Hk', 'Dk', 'Dv')] + [('scale', f32)] + [(n, p) for n in 'qkvg'] +
                [(f'{n}_{s}', i64) for n in 'qkvg' for s in 'tbh'] + [(n, p) for n in ('g_q', 'g_k', 'g_v', 'log_decay', 'lengths', 's_in', 'g_last', 'g_s', 'states', 'ws')])


def _lib():
    L = ctypes.CDLL(_seqlib.LIB_PATH)
    for name, args in (('ss_seq_leaky', [p, p]), ('ss_seq_leaky_bwd', [p, p]), ('ss_seq_group_sum', [p, p, i64, i32, i32, i32, p]),
                       ('ss_seq_rms_norm_fwd', [p, i64, p, i64, p, p, p, p, i64, i32, f32, i32, p]), ('ss_seq_rms_norm_bwd', [p, p, p, p, p, p, p, p, i64, i32, i32, p]),
                       ('ss_seq_rms_norm_int8', [p, i64, p, i64, p, p, p, p, i64, i32, f32, i32, p]), ('ss_seq_dequant_int8', [p, p, p, i64, i32, i32, p]),
                       ('ss_seq_int8_linear', [p, i64, p, p, i64, p, p, p, i64, i32, i32, i32, p, p])):
        getattr(L, name).argtypes = args
    return L


def test_header_binding_and_library_agree():
    src = re.sub(r'/\*.*?\*/', '', open(os.path.join(ROOT, 'include', 'ss_sequence.h')).read(), flags=re.S)
    declared = set(re.findall(r'\b(?:int|long long)\s+(ss_seq_[a-z0-9_]+)\s*\(', src))
    L = _lib()
    for name in declared:
        assert hasattr(L, name), name
    out = subprocess.check_output(['nm', '-D', '--defined-only', _seqlib.LIB_PATH]).decode()
    assert declared <= {l.split()[-1] for l in out.splitlines() if ' T ' in l}
    assert L.ss_seq_abi_version() == _seqlib.ABI_VERSION == _seqlib.ops().abi_version()
    assert b'gfx950' in open(_seqlib.LIB_PATH, 'rb').read()


def test_product_fails_loudly_on_cpu_tensors():
    q = torch.zeros(2, 1, 1, 8)
    with pytest.raises(SSNeuronError, match='no CPU fallback'):
        sequence.leaky_attention(q, q, q, torch.zeros(1))
    with pytest.raises(SSNeuronError, match='no CPU fallback'):
        sequence.leaky_attention_step(q[0], q[0], q[0], torch.zeros(1), torch.zeros(1, 1, 8, 8))
    with pytest.raises(SSNeuronError, match='no CPU fallback'):
        sequence.add_rms_norm(q, torch.ones(8))
    with pytest.raises(SSNeuronError, match='no CPU fallback'):
        sequence.add_rms_norm_int8(q, torch.ones(8))
    with pytest.raises(SSNeuronError, match='no CPU fallback'):
        sequence.dequantize_int8(q.to(torch.int8), torch.ones(2, 1, 1))
    with pytest.raises(SSNeuronError, match='no CPU fallback'):
        sequence.int8_linear(q.to(torch.int8), torch.ones(2, 1, 1), torch.zeros(3, 8, dtype=torch.int8), torch.ones(3))


def test_library_missing(monkeypatch):
    monkeypatch.setattr(_seqlib, '_ops', None)
    monkeypatch.setattr(_seqlib, 'LIB_PATH', '/nonexistent/libss_sequence.so')
    with pytest.raises(SSNeuronError, match='not built'):
        sequence.add_rms_norm(torch.zeros(1, 8), torch.ones(8))


def _desc(**kw):
    d = LeakyDesc(size=ctypes.sizeof(LeakyDesc), T=1, B=1, H=1, DA=8, DC=8, a_group=1, b_group=1, c_group=1, a=256, b=256, c=256, out=256,
                          log_decay=256, b_scale=1., o_scale=1.)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize('bad', [dict(size=8), dict(T=0), dict(B=0), dict(H=0), dict(DA=0), dict(DA=257), dict(DC=0), dict(DC=257), dict(dtype=3), dict(dtype=1, out_dtype=2),
                                 dict(a_group=0), dict(b_group=2), dict(c_group=2), dict(a=0), dict(b=0), dict(c=0), dict(out=0), dict(log_decay=0), dict(B=70000), dict(T=2, s_in=512, s_out=512)])
def test_leaky_entry_refuses(bad):
    """Refused on the host, before any HIP call (the pointers are never read)."""
    assert _lib().ss_seq_leaky(ctypes.byref(_desc(**bad)), None) == -22


@pytest.mark.parametrize('bad', [dict(size=8), dict(T=0), dict(Hk=0), dict(Hk=3), dict(Dk=0), dict(Dk=257), dict(Dv=0), dict(Dv=257), dict(dtype=3), dict(B=70000), dict(q=0),
                                 dict(k=0), dict(v=0), dict(g=0), dict(log_decay=0), dict(g_v=0, g_s=256), dict(T=4096, states=0), dict(T=4096, ws=0)])
def test_leaky_bwd_entry_refuses(bad):
    d = LeakyBwdDesc(size=ctypes.sizeof(LeakyBwdDesc), T=4, B=1, H=4, Hk=2, Dk=8, Dv=8, q=256, k=256, v=256, g=256, g_q=256, g_k=256, g_v=256, log_decay=256,
                     states=256, ws=256, scale=1.)
    for k, v in bad.items():
        setattr(d, k, v)
    assert _lib().ss_seq_leaky_bwd(ctypes.byref(d), None) == -22


def test_other_entries_refuse():
    L = _lib()
    assert L.ss_seq_leaky(None, None) == -22
    assert L.ss_seq_group_sum(None, None, 1, 1, 1, 0, None) == -22
    ok = (256, 8, None, 0, 256, 256, None, None, 4, 8, 1e-6, 0, None)
    for at, value in ((0, None), (4, None), (5, None), (8, -1), (9, 0), (9, 16385), (10, -1.), (10, math.nan), (11, 3), (2, 256)):       # (residual without a sum)
        bad = list(ok)
        bad[at] = value
        assert L.ss_seq_rms_norm_fwd(*bad) == -22, (at, value)
    assert L.ss_seq_rms_norm_fwd(None, 0, None, 0, None, None, None, None, 0, 8, 1e-6, 0, None) == 0          # no rows: nothing to do
    assert L.ss_seq_rms_norm_int8(256, 8, None, 0, 256, None, 256, None, 4, 8, 1e-6, 0, None) == -22
    assert L.ss_seq_rms_norm_bwd(None, None, None, None, None, None, None, None, 4, 8, 0, None) == -22
    assert L.ss_seq_rms_norm_bwd(None, None, 256, 256, 256, 256, 256, None, 4, 8, 0, None) == -22             # a weight gradient without its workspace
    assert L.ss_seq_dequant_int8(None, None, None, 4, 8, 0, None) == -22
    for M, N, K, dt in ((-1, 8, 8, 0), (1, 0, 8, 0), (1, 8, 0, 0), (1, 8, 131072, 0), (1, 8, 8, 5)):
        assert L.ss_seq_int8_linear(256, K, 256, 256, K, 256, None, 256, M, N, K, dt, None, None) == -22
    assert L.ss_seq_int8_linear(None, 8, 256, 256, 8, 256, None, 256, 1, 8, 8, 0, None, None) == -22


def test_leaky_entry_refuses_a_state_in_place_of_its_transpose():
    same = dict(T=1, s_in=512, s_out=512, s_in_row=8, s_in_col=1)
    for bad in (dict(s_out_row=1, s_out_col=8), dict(s_out_row=16, s_out_col=1)):
        assert _lib().ss_seq_leaky(ctypes.byref(_desc(**same, **bad)), None) == -22


def test_product_entry_refuses_more_than_a_grid_holds():
    L = _lib()
    for M, N in ((2 ** 27 + 1, 8), (8, 2 ** 27 + 1), (2 ** 27, 2 ** 27), (2 ** 19, 2 ** 19)):
        assert L.ss_seq_int8_linear(256, 16, 256, 256, 16, 256, None, 256, M, N, 16, 0, 256, None) == -22


def test_limits_agree():
    """The three places that know a limit: the Python checks, the library's, and the C entries' own."""
    src = open(os.path.join(ROOT, 'stereospike_amd', 'csrc', 'ss_seq_torch.cpp')).read()
    mine = {n: int(v) << int(by or 0) for n, v, by in re.findall(r'\b(kMax\w+) = (\d+)(?: << (\d+))?', src)}
    assert mine == dict(kMaxHead=_seqlib.MAX_HEAD_DIM, kMaxWidth=_seqlib.MAX_NORM_WIDTH, kMaxK=_seqlib.MAX_INT8_K, kMaxStates=_seqlib.MAX_STATES,
                        kMaxSteps=_seqlib.MAX_STEPS, kMaxSide=_seqlib.MAX_SIDE, kMaxTiles=_seqlib.MAX_TILES)
    L, null = _lib(), None
    L.ss_seq_leaky_ws_floats.argtypes, L.ss_seq_leaky_ws_floats.restype = [p], i64
    # inside every limit a workspace is asked for, behind one nothing is (and the entry refuses)
    inside = dict(T=65536, B=1, H=1, DA=_seqlib.MAX_HEAD_DIM, DC=_seqlib.MAX_HEAD_DIM)
    assert L.ss_seq_leaky_ws_floats(ctypes.byref(_desc(**inside))) > 0
    for behind in (dict(DA=_seqlib.MAX_HEAD_DIM + 1), dict(DC=_seqlib.MAX_HEAD_DIM + 1), dict(T=_seqlib.MAX_STEPS + 1), dict(B=_seqlib.MAX_STATES + 1)):
        assert L.ss_seq_leaky_ws_floats(ctypes.byref(_desc(**{**inside, **behind}))) == 0
        assert L.ss_seq_leaky(ctypes.byref(_desc(**{**inside, **behind})), null) == -22
    L.ss_seq_rms_norm_ws_floats.argtypes, L.ss_seq_rms_norm_ws_floats.restype = [i64, i32, i32], i64
    assert L.ss_seq_rms_norm_ws_floats(2, _seqlib.MAX_NORM_WIDTH, 0) > 0 and L.ss_seq_rms_norm_ws_floats(2, _seqlib.MAX_NORM_WIDTH + 1, 0) == 0
    for M, N, K, rc in ((0, _seqlib.MAX_SIDE, 16, 0), (_seqlib.MAX_SIDE + 1, 1, 16, -22), (1, _seqlib.MAX_SIDE + 1, 16, -22), (0, 8, _seqlib.MAX_INT8_K, 0), (0, 8, _seqlib.MAX_INT8_K + 1, -22),
                        (128 * 4096, 128 * (_seqlib.MAX_TILES // 4096), 16, -22)):
        assert L.ss_seq_int8_linear(256, K, 256, 256, K, 256, null, 256, M, N, K, 0, null, null) == rc, (M, N, K)


@pytest.fixture
def anywhere(monkeypatch):
    """The reasons of a refusal behind the device check, on CPU tensors (which the library hands back before it launches anything)."""
    monkeypatch.setattr(sequence, '_require_hip', lambda t, name: None)


def _qkv(T=3, B=2, H=4, Hk=2, Dk=8, Dv=6, dtype=torch.float32):
    return torch.zeros(T, B, H, Dk, dtype=dtype), torch.zeros(T, B, Hk, Dk, dtype=dtype), torch.zeros(T, B, Hk, Dv, dtype=dtype)


def test_attention_refusals(anywhere):
    q, k, v = _qkv()
    g, i32 = torch.zeros(4), torch.int32
    for args, kw, what in (((q.double(), k, v, g), {}, 'q: expected float32'), ((q[0], k, v, g), {}, '4 axes'), ((q, k.half(), v, g), {}, 'k: expected'),
                           ((q, k[:2], v, g), {}, 'k: expected shape'), ((q, k, v[:, :1], g), {}, 'v: expected shape'), ((q[:, :, :3], k, v, g[:3]), {}, 'cannot share'),
                           ((q, k, v, g[:2]), {}, 'log_decay'), ((q, k, v, g.double()), {}, 'log_decay'),
                           ((q, k, v, torch.zeros(4, requires_grad=True)), {}, 'no gradient'),
                           ((q, k, v, g), dict(state=torch.zeros(2, 4, 6, 8)), 'state: expected shape'),
                           ((q, k, v, g), dict(state=torch.zeros(2, 4, 8, 6, dtype=torch.float16)), 'state: expected torch.float32'),
                           ((q, k, v, g), dict(lengths=torch.zeros(2)), 'lengths: expected torch.int32'), ((q, k, v, g), dict(lengths=torch.zeros(3, dtype=i32)), 'lengths')):
        with pytest.raises(SSNeuronError, match=what):
            sequence.leaky_attention(*args, **kw)
    with pytest.raises(SSNeuronError, match='head sizes'):
        sequence.leaky_attention(*_qkv(Dk=257), g)
    with pytest.raises(SSNeuronError, match='at most 65535'):
        sequence.leaky_attention(*_qkv(T=1, B=16384, Dk=1, Dv=1), g)
    s = torch.zeros(2, 4, 8, 6)
    with pytest.raises(SSNeuronError, match='state: tensor must be contiguous'):
        sequence.leaky_attention_step(q[0], k[0], v[0], g, torch.zeros(2, 4, 6, 8).transpose(2, 3))
    with pytest.raises(SSNeuronError, match='3 axes'):
        sequence.leaky_attention_step(q, k, v, g, s)


def test_a_product_of_too_many_outputs_is_refused_by_name(anywhere):
    a, s = torch.zeros(1, 16, dtype=torch.int8).expand(2 ** 19, 16), torch.ones(1).expand(2 ** 19)
    with pytest.raises(SSNeuronError, match='524288 rows by 524288 channels'):
        sequence.int8_linear(a, s, a, s)


def test_a_step_under_autograd_is_refused(anywhere):
    """It has no gradient: operands that require one while gradients are enabled, or a state (updated in place) that does, would lose it without a word."""
    q, k, v = (t[0] for t in _qkv())
    g, s = torch.zeros(4), torch.zeros(2, 4, 8, 6)
    for i in range(3):
        use = [q, k, v]
        use[i] = use[i].clone().requires_grad_()
        with pytest.raises(SSNeuronError, match='step has no gradient'):
            sequence.leaky_attention_step(*use, g, s)
    with pytest.raises(SSNeuronError, match='step has no gradient'):
        sequence.leaky_attention_step(q, k, v, g.clone().requires_grad_(), s)
    for state in (s.clone().requires_grad_(), s.clone().requires_grad_() * 2):
        with pytest.raises(SSNeuronError, match='state: it is updated in place'):
            sequence.leaky_attention_step(q, k, v, g, state)
        with torch.no_grad(), pytest.raises(SSNeuronError, match='state: it is updated in place'):
            sequence.leaky_attention_step(q, k, v, g, state)


def test_norm_and_product_refusals(anywhere):
    x, w = torch.zeros(3, 8), torch.ones(8)
    for args, kw, what in (((x.double(), w), {}, 'x: expected'), ((x, w[:4]), {}, 'weight'), ((x, w.half()), {}, 'weight'), ((x, w), dict(residual=x.half()), 'residual'),
                           ((x, w), dict(residual=x[:2]), 'residual'), ((x, w), dict(eps=-1.), 'eps'), ((torch.zeros(1, 16385), torch.ones(16385)), {}, 'rows of')):
        with pytest.raises(SSNeuronError, match=what):
            sequence.add_rms_norm(*args, **kw)
        with pytest.raises(SSNeuronError, match=what):
            sequence.add_rms_norm_int8(*args, **kw)
    a, sa, b, sb = torch.zeros(3, 8, dtype=torch.int8), torch.ones(3), torch.zeros(5, 8, dtype=torch.int8), torch.ones(5)
    for args, kw, what in (((a.float(), sa, b, sb), {}, 'codes'), ((a[:, :4], sa, b, sb), {}, 'codes'), ((a, sa[:2], b, sb), {}, 'scales'), ((a, sa, b.float(), sb), {}, 'weight'),
                           ((a, sa, b, sb[:4]), {}, 'weight_scale'), ((a, sa, b, sb), dict(bias=torch.ones(4)), 'bias'), ((a, sa, b, sb), dict(out_dtype=torch.int32), 'out_dtype'),
                           ((a, sa, b[0], sb), {}, 'weight'), ((a, sa.requires_grad_(), b, sb), {}, 'no gradient')):
        with pytest.raises(SSNeuronError, match=what):
            sequence.int8_linear(*args, **kw)
    with pytest.raises(SSNeuronError, match='K <= 131071'):
        sequence.int8_linear(torch.zeros(1, 131072, dtype=torch.int8), torch.ones(1), torch.zeros(1, 131072, dtype=torch.int8), torch.ones(1))
    with pytest.raises(SSNeuronError, match='scales'):
        sequence.dequantize_int8(a, torch.ones(2))
    with pytest.raises(SSNeuronError, match='dtype'):
        sequence.dequantize_int8(a, torch.ones(3), torch.float64)


def test_values_of_codes_under_autograd_are_refused(anywhere):
    with pytest.raises(SSNeuronError, match='dequantize_int8 has no gradient'):
        sequence.dequantize_int8(torch.zeros(3, 8, dtype=torch.int8), torch.ones(3, requires_grad=True))


def test_quantize_channels():
    torch.manual_seed(0)
    w = torch.randn(5, 40)
    w[3] = 0
    codes, scale = sequence.quantize_channels(w)
    assert codes.dtype == torch.int8 and codes.abs().max() == 127 and scale[3] == 0 and not codes[3].any()
    # half a code's step, and the scale's own rounding (2^-24) over 127 codes
    assert ((codes * scale[:, None]).double() - w.double()).abs().le(scale[:, None].double() * (0.5 + 127 * 2. ** -23)).all()
    with pytest.raises(SSNeuronError, match='weight'):
        sequence.quantize_channels(torch.zeros(3, dtype=torch.float32))


def test_layers_keep_the_state_protocol():
    att = layer.LeakyAttention(4)
    tau = 1. / -torch.expm1(att.log_decay.double())
    assert torch.allclose(tau, 2. * 512. ** (torch.arange(4).double() / 3), rtol=1e-4)        # tau = 1 / (1 - lambda): 1024 times the rounding of log lambda
    att.s = torch.ones(1, 4, 2, 2, requires_grad=True) * 2
    functional.detach_net(att)
    assert not att.s.requires_grad
    functional.reset_net(att)
    assert att.s is None
    assert layer.LeakyAttention(2, tau=[1., math.inf]).log_decay.tolist() == [-math.inf, 0.]
    with pytest.raises(AssertionError):
        layer.LeakyAttention(2, tau=[0.5, 2.])
    lin = torch.nn.Linear(6, 3)
    q = layer.Int8Linear(lin)
    assert set(q.state_dict()) == {'weight', 'weight_scale', 'bias'} and q.weight.dtype == torch.int8
    assert layer.Int8Linear(torch.nn.Linear(6, 3, bias=False)).bias is None
    assert list(layer.AddRMSNorm(7).state_dict()) == ['weight']


def _every_call():
    """(name, call of one floating operand, that operand) for each entry point."""
    q, g, s = torch.randn(3, 2, 2, 8), torch.zeros(2), torch.zeros(2, 2, 8, 8)
    x, c, one = torch.randn(3, 8), torch.zeros(3, 8, dtype=torch.int8), torch.ones(3)
    w, sw = torch.zeros(5, 8, dtype=torch.int8), torch.ones(5)
    return [('leaky_attention', lambda t: sequence.leaky_attention(t, q, q, g), q), ('leaky_attention', lambda t: sequence.leaky_attention(q, q, t, g), q),
            ('leaky_attention', lambda t: sequence.leaky_attention(q, q, q, t), g), ('leaky_attention', lambda t: sequence.leaky_attention(q, q, q, g, state=t), s),
            ('leaky_attention_step', lambda t: sequence.leaky_attention_step(q[0], t, q[0], g, s), q[0]),
            ('leaky_attention_step', lambda t: sequence.leaky_attention_step(q[0], q[0], q[0], g, t), s),
            ('add_rms_norm', lambda t: sequence.add_rms_norm(t, torch.ones(8))[0], x), ('add_rms_norm', lambda t: sequence.add_rms_norm(x, t, x)[0], torch.ones(8)),
            ('add_rms_norm', lambda t: sequence.add_rms_norm(x, torch.ones(8), t)[0], x), ('add_rms_norm_int8', lambda t: sequence.add_rms_norm_int8(x, torch.ones(8), t), x),
            ('dequantize_int8', lambda t: sequence.dequantize_int8(c, t), one), ('int8_linear', lambda t: sequence.int8_linear(c, t, w, sw), one),
            ('int8_linear', lambda t: sequence.int8_linear(c, one, w, sw, t), sw)]


@pytest.mark.parametrize('i', range(len(_every_call())))
def test_tracers_and_forward_mode_are_refused(anywhere, i):
    """A trace would hold the outputs' allocation without the launch, and an output would have no tangent."""
    name, call, t = _every_call()[i]
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(SSNeuronError, match=f'{name} has no forward-mode'):
            call(torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)))
    with pytest.raises(SSNeuronError, match=f'{name} cannot be traced'):
        torch.jit.trace(call, (t,))
    with pytest.raises(SSNeuronError, match=f'{name} cannot be traced'):
        torch.fx.experimental.proxy_tensor.make_fx(call)(t)
