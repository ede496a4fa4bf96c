"""CPU checks of the position operators: bucket borders, refusals (status codes before anything touches a device) and the
float64 reference's gradients against differences."""

import ctypes
import math

import pytest
import torch

from substation_b200 import _lib, ops
from tests import position_reference as ref


# ---- buckets ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('n,far,both', [(32, 128, True), (32, 128, False), (2, 2, False), (4, 7, True), (320, 800, True), (256, 832, False),
                                        (16, 9, False), (64, 64, False)])
def test_bucket_borders_against_logarithms(n, far, both):
    b = ops.relative_buckets(n, far, both)
    d = n // 2 if both else n
    exact = d // 2
    assert len(b) == n and len(b.starts) == d and b.starts[0] == 0
    for x in range(0, 2 * far):
        if x < exact:
            want = x
        else:
            y = math.log(x / exact) / math.log(far / exact) * (d - exact)
            if abs(y - round(y)) < 1e-9:
                y = round(y)               # a border that is a distance itself
            want = min(d - 1, exact + math.floor(y))
        assert b.bucket(-x) == want, x
        assert b.bucket(x) == ((want + d if x else 0) if both else 0), x


def test_bucket_borders_that_are_distances():
    b = ops.relative_buckets(32, 128, True)
    assert b.starts[8::2] == (8, 16, 32, 64) and b.bucket(-16) == 10 and b.bucket(-15) == 9


def test_bucket_refusals():
    for args in ((1, 128, False), (2, 128, True), (33, 128, True), (32, 8, True), (32, 16, False)):
        with pytest.raises(ValueError):
            ops.relative_buckets(*args)
    assert ops.relative_buckets(32, 128) is ops.relative_buckets(32, 128)
    assert ops.relative_buckets(32, 10 ** 9).bucket(-10 ** 8) == 15     # (far borders are searched, not counted to)
    for starts in ([0, -1], [0, 1 << 31]):
        with pytest.raises(ValueError):
            ops.RelativeBuckets(starts)


# ---- refusals --------------------------------------------------------------------------------------------------------
def _t(sizes, strides=None, ptr=0x10000):
    t = _lib.SbTensor()
    t.ptr, t.ndim = ptr, len(sizes)
    run = 1
    for i in reversed(range(len(sizes))):
        t.size[i] = sizes[i]
        t.stride[i] = run if strides is None else strides[i]
        run *= sizes[i]
    return t


def _norm_call(**kw):
    a = dict(q=_t([64, 4, 2, 8]), k=_t([64, 2, 2, 8]), qg=_t([64]), kg=_t([64]), pos=_t([2, 8]), qo=_t([64, 4, 2, 8], ptr=0x90000),
             ko=_t([64, 2, 2, 8], ptr=0xa0000), base=1e4, rotary=64, pairing=0, eps=1e-6, rot=True)
    a.update(kw)
    r = _lib.SbRotation()
    r.base, r.rotary, r.pairing, r.eps = a['base'], a['rotary'], a['pairing'], a['eps']
    opt = lambda t: None if t is None else ctypes.byref(t)
    lib = _lib.load()
    st = lib.sb_query_key_norm_rotation(None, opt(a['q']), opt(a['k']), opt(a['qg']), opt(a['kg']), opt(a['pos']), opt(a['qo']),
                                        opt(a['ko']), ctypes.byref(r) if a['rot'] else None)
    return st, lib.sb_last_error().decode()


@pytest.mark.parametrize('kw,status,fragment', [
    (dict(q=None), 1, 'null tensor'),
    (dict(kg=None), 1, 'together or not at all'),
    (dict(k=None), 1, 'together or not at all'),
    (dict(qg=_t([32])), 1, 'extent mismatch'),
    (dict(qg=_t([64], [2])), 3, 'contiguous'),
    (dict(k=_t([64, 2, 2, 9])), 1, 'extent mismatch'),
    (dict(k=_t([64, 0, 2, 8]), ko=_t([64, 0, 2, 8])), 1, 'no heads'),
    (dict(pos=_t([8, 2])), 1, 'extent mismatch'),
    (dict(qo=_t([64, 4, 2, 7])), 1, 'extent mismatch'),
    (dict(qo=_t([64, 4, 2, 8], [1, 0, 64, 128])), 1, 'zero stride'),
    (dict(qo=_t([64, 4, 2, 8], [1, 64, 256, 512])), 1, "its input's place"),
    (dict(rotary=3), 1, 'even'),
    (dict(rotary=66), 1, 'even'),
    (dict(rotary=-2), 1, 'even'),
    (dict(pairing=2), 1, 'pairing'),
    (dict(base=0.0), 1, 'base'),
    (dict(base=math.inf), 1, 'base'),
    (dict(eps=-1.0), 1, 'eps'),
    (dict(eps=math.nan), 1, 'eps'),
    (dict(rot=False), 1, 'null rotation'),
    (dict(q=_t([320, 4, 2, 8]), qo=_t([320, 4, 2, 8]), qg=_t([320]), k=None, kg=None, ko=None), 3, 'at most 256'),
    (dict(q=_t([64, 4, 65536, 65536], [0] * 4), k=None, kg=None, ko=None), 3, 'tokens'),
    (dict(q=_t([64, 4, 32768, 32769], [0] * 4), k=None, kg=None, ko=None), 3, 'tokens'),
])
def test_norm_refusals(kw, status, fragment):
    st, text = _norm_call(**kw)
    assert st == status and fragment in text, (st, text)


def test_attention_output_in_an_inputs_place():
    for name in ('q', 'k', 'v'):
        st, text = _attention_call(**{name: _t([64, 4, 2, 8] if name == 'q' else [64, 2, 2, 12], ptr=0x90000)})
        assert st == 1 and 'place' in text


def test_norm_backward_refusals():
    lib = _lib.load()
    r = _lib.SbRotation()
    r.base, r.rotary, r.pairing, r.eps = 1e4, 64, 0, 1e-6
    x, o, g, pos = _t([64, 4, 2, 8]), _t([64, 4, 2, 8], ptr=0x90000), _t([64]), _t([2, 8])
    need = lib.sb_query_key_norm_scratch_bytes()

    def call(scratch, n, dq=o, dout=x):
        b = ctypes.byref
        return lib.sb_backward_query_key_norm_rotation(None, scratch, n, b(dout), None, b(x), None, b(g), None, b(pos), b(dq), None,
                                                       b(g), None, b(r)), lib.sb_last_error().decode()
    for args, status, text in (((None, need), 1, 'scratch'), ((0x1000, need - 1), 1, 'scratch'), ((0x1008, need), 5, 'aligned')):
        st, msg = call(*args)
        assert st == status and text in msg
    assert call(0x1000, need, dq=_t([64, 4, 2, 9]))[0] == 1
    assert call(0x1000, need, dout=_t([64, 4, 1, 8]))[0] == 1


def _attention_call(backward=False, **kw):
    a = dict(q=_t([64, 4, 2, 8]), k=_t([64, 2, 2, 12]), v=_t([64, 2, 2, 12]), table=_t([8, 4]), starts=[0, 1, 2, 4], n=None, both=1,
             out=_t([64, 4, 2, 8], ptr=0x90000), lse=_t([4, 2, 8]), scale=1.0, lengths=None, first=None, dtable=_t([8, 4], ptr=0xa0000),
             dout=_t([64, 4, 2, 8]), dq=_t([64, 4, 2, 8], ptr=0xb0000), dk=_t([64, 2, 2, 12], ptr=0xc0000),
             dv=_t([64, 2, 2, 12], ptr=0xd0000), scratch=0x1000, room=1 << 40, span=True)
    a.update(kw)
    bias = _lib.SbRelativeBias()
    starts = (ctypes.c_int32 * max(1, len(a['starts'])))(*a['starts'])
    bias.table = ctypes.pointer(a['table']) if a['table'] is not None else None
    bias.n, bias.bidirectional = len(a['starts']) if a['n'] is None else a['n'], a['both']
    bias.starts = ctypes.cast(starts, ctypes.POINTER(ctypes.c_int32))
    span = _lib.SbAttentionSpan()
    span.scale, span.causal, span.lengths, span.first = a['scale'], 0, a['lengths'], a['first']
    opt = lambda t: None if t is None else ctypes.byref(t)
    lib = _lib.load()
    sp = ctypes.byref(span) if a['span'] else None
    if backward:
        st = lib.sb_backward_relative_attention(None, a['scratch'], a['room'], opt(a['dout']), opt(a['q']), opt(a['k']), opt(a['v']),
                                                ctypes.byref(bias), opt(a['out']), opt(a['lse']), opt(a['dq']), opt(a['dk']),
                                                opt(a['dv']), opt(a['dtable']), sp)
    else:
        st = lib.sb_relative_attention(None, a['scratch'], a['room'], opt(a['q']), opt(a['k']), opt(a['v']), ctypes.byref(bias),
                                       opt(a['out']), opt(a['lse']), sp)
    return st, lib.sb_last_error().decode()


@pytest.mark.parametrize('backward', [False, True])
@pytest.mark.parametrize('kw,status,fragment', [
    (dict(q=None), 1, 'null tensor'),
    (dict(v=_t([64, 2, 2, 11])), 1, 'extent mismatch'),
    (dict(k=_t([32, 2, 2, 12]), v=_t([32, 2, 2, 12])), 1, 'extent mismatch'),
    (dict(k=_t([64, 2, 3, 12]), v=_t([64, 2, 3, 12])), 1, 'extent mismatch'),
    (dict(k=_t([64, 3, 2, 12]), v=_t([64, 3, 2, 12])), 1, 'multiple'),
    (dict(k=_t([64, 2, 2, 0]), v=_t([64, 2, 2, 0])), 1, 'positive'),
    (dict(q=_t([64, 4, 2, 0])), 1, 'positive'),
    (dict(q=_t([136, 4, 2, 8]), k=_t([136, 2, 2, 12]), v=_t([136, 2, 2, 12])), 3, 'at most 128'),
    (dict(table=None), 1, 'null'),
    (dict(table=_t([8, 3])), 1, '[buckets, heads]'),
    (dict(table=_t([4, 4])), 1, '[buckets, heads]'),
    (dict(both=0), 1, '[buckets, heads]'),
    (dict(n=0), 1, 'at least one'),
    (dict(starts=[0] * 513, table=_t([1026, 4])), 3, 'at most 512'),
    (dict(starts=[1, 2, 3, 4]), 1, 'distance 0'),
    (dict(starts=[0, 3, 2, 4]), 1, 'decrease'),
    (dict(starts=[0, 1, 2, 833]), 3, 'at most 832'),
    (dict(out=_t([64, 4, 2, 9])), 1, 'extent mismatch'),
    (dict(lse=_t([4, 2, 9])), 1, 'extent mismatch'),
    (dict(q=_t([64, 65536, 2, 8]), out=_t([64, 65536, 2, 8], ptr=0x90000), dout=_t([64, 65536, 2, 8]), table=_t([8, 65536])), 3, '65535'),
    (dict(k=_t([64, 2, 2, (1 << 28) + 1]), v=_t([64, 2, 2, (1 << 28) + 1])), 3, 'too many'),
    (dict(scale=math.nan), 1, 'finite'),
    (dict(scale=-1.0), 1, 'negative'),
    (dict(lengths=0x1002), 5, 'int32'),
    (dict(first=0x1001), 5, 'int32'),
    (dict(span=False), 1, 'null span'),
])
def test_attention_refusals(backward, kw, status, fragment):
    st, text = _attention_call(backward, **kw)
    assert st == status and fragment in text, (st, text)


@pytest.mark.parametrize('kw,status,fragment', [
    (dict(lse=None), 1, 'lse'),
    (dict(dtable=_t([8, 5], ptr=0xa0000)), 1, 'extent mismatch'),
    (dict(dq=_t([64, 4, 2, 8])), 1, 'place'),
    (dict(dv=_t([64, 2, 2, 12], ptr=0x90000)), 1, 'place'),
    (dict(dtable=_t([8, 4], [0, 1], ptr=0xa0000)), 1, 'zero stride'),
    (dict(dk=_t([64, 2, 2, 12], [1, 64, 0, 128], ptr=0xc0000)), 1, 'zero stride'),
    (dict(dout=_t([64, 4, 2, 9])), 1, 'extent mismatch'),
    (dict(scratch=None), 1, 'scratch'),
    (dict(room=16), 1, 'scratch'),
    (dict(scratch=0x1004), 5, 'aligned'),
])
def test_attention_backward_refusals(kw, status, fragment):
    st, text = _attention_call(True, **kw)
    assert st == status and fragment in text, (st, text)


def test_python_refusals():
    x, g, pos = torch.zeros(64, 4, 2, 8).half(), torch.zeros(64).half(), torch.zeros(2, 8, dtype=torch.int32)
    with pytest.raises(ValueError, match='CUDA'):
        ops.query_key_norm_rotation(x, None, g, None, pos, x, None)
    with pytest.raises(ValueError, match='CUDA'):
        ops.relative_attention(x, x, x, torch.zeros(32, 4).half(), x, buckets=ops.relative_buckets(), scale=1.0)


# ---- the reference itself --------------------------------------------------------------------------------------------
def test_reference_gradients_against_differences():
    torch.manual_seed(0)
    b = ops.relative_buckets(8, 6, True)
    q, k, v = (torch.randn(*s, dtype=torch.float64) for s in ((6, 4, 2, 7), (6, 2, 2, 9), (6, 2, 2, 9)))
    table, dout = torch.randn(8, 4, dtype=torch.float64), torch.randn(6, 4, 2, 7, dtype=torch.float64)
    how = dict(scale=0.4, lengths=torch.tensor([9, 5], dtype=torch.int32), first=torch.tensor([1, -2], dtype=torch.int32))
    for causal in (False, True):
        r, _ = ref.attention(q, k, v, table, b, causal=causal, dout=dout, **how)
        args = {'q': q, 'k': k, 'v': v, 'table': table}
        for name in args:
            d = torch.randn_like(args[name])
            f = [(ref.attention(**{**args, name: args[name] + e * d}, buckets=b, causal=causal, **how)[0]['out'] * dout).sum()
                 for e in (1e-5, -1e-5)]
            got = (r['d' + name] * d).sum()
            assert abs((f[0] - f[1]) / 2e-5 - got) <= 1e-7 * (1 + abs(got)), (name, causal)
    x, gain, pos = torch.randn(10, 3, 2, 4, dtype=torch.float64), torch.randn(10, dtype=torch.float64), torch.tensor([[5, -3, 0, 77]] * 2)
    w = torch.randn_like(x)
    for pairing in ('halves', 'adjacent'):
        how = (pos, 100.0, 6, pairing, 1e-3)
        dx, dgain, _ = ref.norm_backward(w, x, gain, *how)
        for name, grad in (('x', dx), ('gain', dgain)):
            d = torch.randn_like(grad)
            f = [(ref.norm_forward(x + e * d if name == 'x' else x, gain + e * d if name == 'gain' else gain, *how) * w).sum()
                 for e in (1e-5, -1e-5)]
            got = (grad * d).sum()
            assert abs((f[0] - f[1]) / 2e-5 - got) <= 1e-7 * (1 + abs(got)), (name, pairing)
