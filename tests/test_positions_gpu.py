"""Position operators on the GPU against float64: types, head layouts, lengths from one token on, odd sizes, strides, masks
that leave rows empty, what stands behind a sequence's end, streams, graphs.  Tolerances are half a step of the storage type
per rounding plus 32-bit arithmetic; ``tests/position_reference.py`` derives them for attention."""

import pytest
import torch

from tests import position_reference as ref

pytestmark = pytest.mark.gpu

DEV = 'cuda:0'
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
BOTH = [torch.float16, torch.bfloat16]


def _ops():
    from substation_b200 import ops
    return ops


def _make(shape, order, dtype, gen, scale=1.0, pad=0, fill=None):
    """Tensor of logical extents ``shape`` = [P,H,B,J], stored in ``order`` (a permutation of 'PHBJ', outermost first) with
    ``pad`` unused elements behind each innermost row."""
    at = ['PHBJ'.index(c) for c in order]
    ext = [shape[i] for i in at]
    full = torch.empty(*ext[:-1], ext[-1] + pad, dtype=dtype, device=DEV)
    if fill is None:
        full.copy_(torch.randn(full.shape, generator=gen, device=DEV) * scale)
    else:
        full.fill_(fill)
    t = full[..., :ext[-1]]
    return t.permute([order.index(c) for c in 'PHBJ'])


def _nan(shape, order, dtype, pad=0):
    return _make(shape, order, dtype, None, fill=float('nan'), pad=pad)


def _within(got, want, bound, what):
    got = got.double()
    assert torch.isfinite(got).all(), f'{what}: not finite (unwritten?)'
    worst = ((got - want).abs() - bound).max().item()
    assert worst <= 0, f'{what}: {worst:.3e} beyond its bound, off by {(got - want).abs().max().item():.3e}'


# ---- norms and rotation ----------------------------------------------------------------------------------------------
# ten 32-bit roundings at most, two units in the last place of sine and cosine and their angle's conversion to 32 bits: below
# 2e-6 of the largest element that a pair may hold, which the row's largest bounds
NORM_F32 = 2e-6

NORM_CASES = [
    # P, H, G, B, J, order of q, order of k, rotary, pairing
    (64, 16, 16, 2, 37, 'BJHP', 'BJHP', 64, 'halves'),
    (64, 4, 2, 1, 1, 'BJHP', 'BJHP', 64, 'adjacent'),
    (128, 8, 1, 3, 50, 'BJHP', 'BJHP', 64, 'halves'),
    (32, 3, 3, 2, 65, 'BHJP', 'BJHP', 32, 'adjacent'),
    (16, 5, 2, 4, 9, 'BJHP', 'JBHP', 16, 'halves'),
    (256, 2, 1, 2, 33, 'BJHP', 'BHJP', 256, 'halves'),
    (80, 12, 4, 2, 40, 'BJHP', 'BJHP', 80, 'halves'),
    (80, 6, 3, 2, 33, 'BJHP', 'BHJP', 40, 'halves'),        # pairs that no two pieces hold
    (31, 5, 2, 3, 20, 'BJHP', 'BJHP', 30, 'adjacent'),
    (130, 3, 9, 2, 41, 'BJHP', 'BHJP', 66, 'halves'),
    (90, 4, 2, 2, 150, 'PHBJ', 'BHPJ', 90, 'adjacent'),     # tokens in twos, sixteen warps
    (2, 9600, 20000, 1, 2, 'PHBJ', 'PHBJ', 2, 'halves'),    # more heads than rows of partial sums for eight of them each
    (2, 9600, 20000, 1, 2, 'BJHP', 'BJHP', 2, 'halves'),
    (96, 4, 4, 2, 21, 'BJHP', 'BJHP', 32, 'adjacent'),
    (64, 12, 12, 3, 24, 'PHBJ', 'PHBJ', 32, 'adjacent'),
    (64, 12, 4, 3, 25, 'PHBJ', 'BJHP', 64, 'halves'),
    (128, 2, 2, 2, 200, 'PHBJ', 'HPBJ', 128, 'halves'),
    (64, 2, 2, 2, 64, 'HBPJ', 'JHPB', 48, 'halves'),
    (65, 2, 1, 2, 7, 'BJHP', 'PHBJ', 64, 'adjacent'),
    (1, 2, 2, 3, 5, 'BJHP', 'BJHP', 0, 'halves'),
    (72, 3, 1, 1, 300, 'BJHP', 'BJHP', 36, 'halves'),
    (64, 2, 2, 70, 1, 'BJHP', 'BJHP', 0, 'halves'),
    (64, 32, 8, 1, 1000, 'BJHP', 'BJHP', 64, 'halves'),
]


def _norm_inputs(case, dtype, pad=0):
    P, H, G, B, J, oq, ok, rotary, pairing = case
    gen = torch.Generator(device=DEV).manual_seed(P * 7 + H + J)
    q, k = _make((P, H, B, J), oq, dtype, gen, 3.0, pad), _make((P, G, B, J), ok, dtype, gen, 0.2, pad)
    qg, kg = (1 + 0.3 * torch.randn(2, P, generator=gen, device=DEV)).to(dtype)
    pos = torch.randint(-5000, 1 << 21, (B, J), generator=gen, device=DEV, dtype=torch.int32)
    return gen, q, k, qg, kg, pos, dict(base=10000.0, rotary=rotary, pairing=pairing, eps=1e-6)


@pytest.mark.parametrize('dtype', BOTH)
@pytest.mark.parametrize('case', NORM_CASES)
def test_norm_rotation(case, dtype):
    ops = _ops()
    P, H, G, B, J, oq, ok = case[:7]
    gen, q, k, qg, kg, pos, how = _norm_inputs(case, dtype)
    qo, ko = _nan((P, H, B, J), oq, dtype), _nan((P, G, B, J), ok, dtype)
    ops.query_key_norm_rotation(q, k, qg, kg, pos, qo, ko, **how)
    for x, gain, got, name in ((q, qg, qo, 'q'), (k, kg, ko, 'k')):
        want = ref.norm_forward(x, gain, pos, **how)
        _within(got, want, HALF[dtype] * 1.01 * want.abs() + NORM_F32 * want.abs().amax(0, keepdim=True) + ref.SMALL, name)


@pytest.mark.parametrize('dtype', BOTH)
@pytest.mark.parametrize('case', NORM_CASES)
def test_norm_rotation_backward(case, dtype):
    ops = _ops()
    P, H, G, B, J, oq, ok = case[:7]
    gen, q, k, qg, kg, pos, how = _norm_inputs(case, dtype)
    gq, gk = _make((P, H, B, J), ok, dtype, gen), _make((P, G, B, J), oq, dtype, gen)      # gradients in other orders
    dq, dk = _nan((P, H, B, J), oq, dtype), _nan((P, G, B, J), ok, dtype)
    dqg, dkg = torch.full((2, P), float('nan'), dtype=dtype, device=DEV)
    ops.backward_query_key_norm_rotation(gq, gk, q, k, qg, kg, pos, dq, dk, dqg, dkg, **how)
    again = [torch.empty_like(t) for t in (dq, dk, dqg, dkg)]
    ops.backward_query_key_norm_rotation(gq, gk, q, k, qg, kg, pos, *again, **how)
    for a, b in zip((dq, dk, dqg, dkg), again):
        assert torch.equal(a, b)
    for x, gain, g, got, gotg, name in ((q, qg, gq, dq, dqg, 'dq'), (k, kg, gk, dk, dkg, 'dk')):
        dx, dgain, mass = ref.norm_backward(g, x, gain, pos, **how)
        # dx is a difference of two terms, each at most as large as r * |g gain|: what 32 bits lose counts against those
        r = 1 / (x.double().square().mean(0, keepdim=True) + how['eps']).sqrt()
        w = r * (g.double().abs().amax(0, keepdim=True) * gain.double().abs().max()) * 2
        n = (x.double() * r).abs().amax(0, keepdim=True)
        _within(got, dx, HALF[dtype] * 1.01 * dx.abs() + NORM_F32 * (1 + n * n) * w + ref.SMALL, name)
        _within(gotg, dgain, HALF[dtype] * 1.01 * dgain.abs() + 1e-5 * mass + ref.SMALL, name + '_gain')


def test_norm_without_keys_in_place_and_with_shared_positions():
    ops = _ops()
    gen = torch.Generator(device=DEV).manual_seed(3)
    for order, P in (('BJHP', 64), ('PHBJ', 64), ('BJHP', 72)):
        q, k = _make((P, 6, 2, 40), order, torch.bfloat16, gen), _make((P, 2, 2, 40), order, torch.bfloat16, gen)
        gain = torch.ones(P, device=DEV).bfloat16()
        pos = torch.arange(40, device=DEV, dtype=torch.int32).expand(2, 40)
        a, b = torch.empty_like(q), torch.empty_like(k)
        ops.query_key_norm_rotation(q, k, gain, gain, pos, a, b)
        c = torch.empty_like(q)
        ops.query_key_norm_rotation(q, None, gain, None, pos, c, None)
        assert torch.equal(a, c)
        da, db, ga, gb = torch.empty_like(q), torch.empty_like(k), torch.empty_like(gain), torch.empty_like(gain)
        gq, gk = torch.randn_like(q), torch.randn_like(k)
        ops.backward_query_key_norm_rotation(gq, gk, q, k, gain, gain, pos, da, db, ga, gb)
        dc, gc = torch.empty_like(q), torch.empty_like(gain)
        ops.backward_query_key_norm_rotation(gq, None, q, None, gain, None, pos, dc, None, gc, None)
        assert torch.equal(da, dc)
        assert torch.allclose(ga.float(), gc.float(), rtol=2 * 2.0 ** -8, atol=1e-4)
        ops.backward_query_key_norm_rotation(gq, gk, q, k, gain, gain, pos, gq, gk, ga, gb)     # in place of the incoming gradients
        assert torch.equal(gq, da) and torch.equal(gk, db)
        ops.query_key_norm_rotation(q, k, gain, gain, pos, q, k)                                # and of the inputs
        assert torch.equal(q, a) and torch.equal(k, b)


def test_norm_of_zeros_and_of_nothing():
    ops = _ops()
    q = torch.zeros(2, 5, 3, 64, device=DEV).half().permute(3, 2, 0, 1)
    gain = torch.ones(64, device=DEV).half()
    pos = torch.zeros(2, 5, dtype=torch.int32, device=DEV)
    out = torch.full_like(q, float('nan'))
    ops.query_key_norm_rotation(q, None, gain, None, pos, out, None)
    assert (out == 0).all()
    e, dg = q[..., :0], torch.full_like(gain, float('nan'))
    ops.query_key_norm_rotation(e, None, gain, None, pos[:, :0], out[..., :0], None)
    ops.backward_query_key_norm_rotation(e, None, e, None, gain, None, pos[:, :0], out[..., :0], None, dg, None)
    assert (dg == 0).all()


def test_norm_leaves_what_lies_between_rows():
    ops = _ops()
    gen = torch.Generator(device=DEV).manual_seed(5)
    for order, pad in (('BJHP', 8), ('BJHP', 3), ('PHBJ', 5)):
        q = _make((64, 3, 2, 21), order, torch.float16, gen, pad=pad)
        full = torch.full((q.untyped_storage().size() // 2,), 7.0, dtype=torch.float16, device=DEV)
        out = full.as_strided(q.shape, q.stride())
        gain = torch.ones(64, device=DEV).half()
        pos = torch.arange(42, device=DEV, dtype=torch.int32).view(2, 21)
        mark = torch.ones_like(full, dtype=torch.bool)
        mark.as_strided(q.shape, q.stride()).fill_(False)
        ops.query_key_norm_rotation(q, None, gain, None, pos, out, None)
        assert (full[mark] == 7).all() and mark.sum() > 0


# ---- attention -------------------------------------------------------------------------------------------------------
ATTENTION_CASES = [
    # P, H, G, B, J, K, order, buckets, far, both, causal, lengths, first
    (64, 4, 4, 2, 128, 128, 'BJHP', 32, 128, True, False, None, None),
    (64, 2, 2, 2, 300, 300, 'BJHP', 32, 128, True, False, [300, 171], None),
    (64, 2, 2, 3, 100, 200, 'BJHP', 32, 128, True, False, [0, 200, 1], None),
    (128, 4, 2, 2, 257, 257, 'BJHP', 32, 128, False, True, None, None),
    (128, 2, 1, 1, 64, 640, 'BJHP', 64, 512, True, False, None, [500]),
    (32, 6, 2, 2, 65, 129, 'BHJP', 16, 20, True, True, [129, 60], [64, -30]),
    (80, 3, 3, 2, 77, 77, 'BJHP', 320, 800, True, False, None, None),
    (64, 8, 8, 2, 64, 64, 'PHBJ', 32, 128, True, False, None, None),
    (64, 4, 2, 2, 51, 83, 'PHBJ', 32, 128, True, False, [83, 20], None),
    (40, 2, 2, 1, 33, 47, 'JBHP', 8, 30, False, False, None, None),
    (7, 2, 1, 2, 19, 23, 'BJHP', 8, 16, True, True, None, None),
    (64, 1, 1, 1, 1000, 1000, 'BJHP', 320, 800, True, False, [937], None),
    (64, 1, 1, 1, 1, 1, 'BJHP', 32, 128, True, False, None, None),
    (64, 2, 1, 2, 700, 20, 'BJHP', 32, 128, False, True, None, [0, -400]),
    (128, 2, 2, 1, 513, 130, 'BJHP', 2, 2, False, False, None, None),
    # few queries against a cache
    (64, 16, 16, 3, 1, 77, 'BJHP', 32, 128, False, True, [77, 5, 40], [76, 4, 39]),
    (128, 32, 8, 2, 1, 2000, 'BJHP', 32, 128, False, True, [2000, 1311], [1999, 1310]),
    (128, 8, 1, 4, 2, 513, 'BHJP', 32, 128, False, True, [513, 0, 2, 300], [511, -2, 0, 298]),
    (64, 4, 4, 1, 5, 5000, 'BJHP', 320, 800, True, False, None, [4995]),
    (80, 4, 2, 2, 3, 333, 'PHBJ', 32, 128, True, False, None, [100, 330]),
    (24, 2, 2, 2, 4, 70, 'BJHP', 32, 128, False, True, [70, 9], [66, 5]),
    (64, 24, 1, 2, 1, 700, 'BJHP', 64, 512, False, True, [700, 699], [699, 698]),
    # many queries, few heads and long keys: split along the keys as well
    (64, 2, 1, 1, 150, 1100, 'BJHP', 32, 128, True, False, [1090], [900]),
    (128, 2, 2, 2, 40, 2100, 'BJHP', 32, 128, False, True, [2100, 700], [2060, 500]),
    (40, 3, 3, 1, 333, 1300, 'PHBJ', 16, 64, True, True, None, [967]),
    # many single tokens, and as many again with shared keys
    (64, 4, 4, 50, 1, 70, 'BJHP', 32, 128, False, True, None, [69] * 50),
    (64, 8, 4, 50, 3, 90, 'BJHP', 32, 128, True, False, list(range(41, 91)), [20] * 50),
    # as many buckets as there may be, up to the last distance
    (64, 2, 2, 1, 900, 900, 'BJHP', 512, 832, False, True, None, None),
    (128, 4, 4, 1, 2, 1700, 'BJHP', 1024, 832, True, False, None, [850]),
    (128, 2, 2, 1, 150, 1000, 'BJHP', 512, 832, True, False, None, [850]),
]


def _attention_inputs(case, dtype, pad=0, junk=False):
    P, H, G, B, J, K, order, n, far, both, causal, lengths, first = case
    gen = torch.Generator(device=DEV).manual_seed(P + 3 * H + J + K)
    q = _make((P, H, B, J), order, dtype, gen, 1.0, pad)
    k, v = (_make((P, G, B, K), order, dtype, gen, 1.0, pad) for _ in range(2))
    table = torch.randn(n, H, generator=gen, device=DEV).to(dtype)
    lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    first = None if first is None else torch.tensor(first, dtype=torch.int32, device=DEV)
    if junk and lengths is not None:      # what stands behind a sequence's end must not matter
        for b in range(B):
            n0 = int(lengths[b])
            k[:, :, b, n0:] = float('nan')
            v[:, :, b, n0:] = float('inf')
    how = dict(buckets=_ops().relative_buckets(n, far, both), scale=P ** -0.5, causal=causal, lengths=lengths, first=first)
    return gen, q, k, v, table, how


@pytest.mark.parametrize('dtype', BOTH)
@pytest.mark.parametrize('case', ATTENTION_CASES)
def test_attention(case, dtype):
    ops = _ops()
    P, H, G, B, J, K, order = case[:7]
    gen, q, k, v, table, how = _attention_inputs(case, dtype, junk=True)
    out, lse = _nan((P, H, B, J), order, dtype), torch.full((H, B, J), float('nan'), device=DEV)
    ops.relative_attention(q, k, v, table, out, lse, **how)
    want, bound = ref.attention(q, k, v, table, half=HALF[dtype], **how)
    _within(out, want['out'], bound['out'], 'out')
    empty = want['lse'].isinf()
    assert torch.equal(lse.isinf(), empty) and (out.permute(1, 2, 3, 0)[empty] == 0).all()
    assert ((lse - want['lse'])[~empty].abs() <= 1e-5 * (1 + want['lse'][~empty].abs())).all()
    bare = _nan((P, H, B, J), order, dtype)
    ops.relative_attention(q, k, v, table, bare, **how)
    assert torch.equal(bare, out)


@pytest.mark.parametrize('dtype', BOTH)
@pytest.mark.parametrize('case', ATTENTION_CASES)
def test_attention_backward(case, dtype):
    ops = _ops()
    P, H, G, B, J, K, order, n = case[:8]
    gen, q, k, v, table, how = _attention_inputs(case, dtype, junk=True)
    out, lse = torch.empty_like(q), torch.empty(H, B, J, device=DEV)
    ops.relative_attention(q, k, v, table, out, lse, **how)
    dout = _make((P, H, B, J), 'BJHP', dtype, gen)
    got = {}
    for _ in range(2):
        last = got
        got = {'dq': _nan((P, H, B, J), order, dtype), 'dk': _nan((P, G, B, K), order, dtype), 'dv': _nan((P, G, B, K), 'BJHP', dtype),
               'dtable': torch.full((n, H), float('nan'), dtype=dtype, device=DEV)}
        ops.backward_relative_attention(dout, q, k, v, table, out, lse, *got.values(), **how)
        assert all(torch.equal(last[x], got[x]) for x in last)
    want, bound = ref.attention(q, k, v, table, half=HALF[dtype], dout=dout, out_used=out, **how)
    for name in got:
        _within(got[name], want[name], bound[name], name)
        if how['lengths'] is not None and name in ('dk', 'dv'):
            for b in range(B):
                assert (got[name][:, :, b, int(how['lengths'][b]):] == 0).all()
    # the bounds above add up; roundings do not: overall the results are nearer (the tolerance of the other parity tests)
    for name in got:
        size = want[name].norm()
        if size > 1e-3 * bound[name].norm() and K > 1:
            stray = 3 * want['dtable_stray'] if name == 'dtable' else 0.0        # (three standard deviations, see the reference)
            assert (got[name].double() - want[name]).norm() <= 1e-2 * size + stray, name


@pytest.mark.parametrize('dtype', BOTH)
@pytest.mark.parametrize('J', [1, 150])
def test_hidden_buckets_and_large_biases(dtype, J):
    """Entries of -inf (and bfloat16's lowest value) hide their keys, a row may lose all of them; finite ones of any size count."""
    ops = _ops()
    gen = torch.Generator(device=DEV).manual_seed(9)
    B, H, K, P = 2, 4, 300, 64
    q, k, v = (_make((P, H, B, n), 'BJHP', dtype, gen) for n in (J, K, K))
    b = ops.relative_buckets(8, 20, True)
    table = torch.randn(8, H, generator=gen, device=DEV)
    table[:4, 0] = -float('inf')                       # head 0 sees nothing at or before the query
    table[:, 1] = -float('inf')                        # head 1 sees nothing at all
    table[7, 2] = torch.finfo(dtype).min               # head 2: the far keys behind the query are as good as hidden
    table[3, 3] = 300.0                                # head 3: far keys before the query outweigh everything
    table = table.to(dtype)
    first = torch.tensor([0, K - J], dtype=torch.int32, device=DEV)
    how = dict(buckets=b, scale=0.125, first=first)
    out, lse = _nan((P, H, B, J), 'BJHP', dtype), torch.empty(H, B, J, device=DEV)
    ops.relative_attention(q, k, v, table, out, lse, **how)
    dout = _make((P, H, B, J), 'BJHP', dtype, gen)
    got = {'dq': torch.empty_like(q), 'dk': torch.empty_like(k), 'dv': torch.empty_like(v), 'dtable': torch.empty_like(table)}
    ops.backward_relative_attention(dout, q, k, v, table, out, lse, *got.values(), **how)
    want, bound = ref.attention(q, k, v, table, half=HALF[dtype], dout=dout, out_used=out, **how)
    _within(out, want['out'], bound['out'] + 1e-4 * want['out'].abs().max(), 'out')     # (300 in 32 bits: 2e-5 of an exponent)
    assert (out[:, 1] == 0).all() and lse[1].isinf().all()
    for name in got:
        _within(got[name], want[name], bound[name] * 1.05 + 1e-4, name)


def test_attention_of_broadcast_keys_and_odd_strides():
    """Keys and values shared by the batch (stride 0), rows that start off the 16-byte grid, and a cache longer than what is
    read of it."""
    ops = _ops()
    gen = torch.Generator(device=DEV).manual_seed(4)
    b = ops.relative_buckets(32, 128, True)
    for J in (3, 140):
        base = torch.randn(1, 260, 2, 64, generator=gen, device=DEV).half()
        k = base.expand(3, 260, 2, 64).permute(3, 2, 0, 1)
        odd = torch.randn(3 * 260 * 2 * 67 + 1, generator=gen, device=DEV).half()
        v = odd[1:].view(3, 260, 2, 67)[..., :64].permute(3, 2, 0, 1)
        q = torch.randn(3, J, 2, 64, generator=gen, device=DEV).half().permute(3, 2, 0, 1)
        table = torch.randn(2, 32, generator=gen, device=DEV).half().t()
        out, lse = torch.empty_like(q), torch.empty(3, J, 2, device=DEV).permute(2, 0, 1)
        ops.relative_attention(q, k, v, table, out, lse, buckets=b, scale=0.125)
        dout = torch.randn(64, 3, 2, J, generator=gen, device=DEV).half().permute(0, 2, 1, 3)
        got = {'dq': torch.empty_like(q), 'dk': torch.empty(3, 260, 2, 64, device=DEV).half().permute(3, 2, 0, 1),
               'dv': torch.empty(3, 260, 2, 64, device=DEV).half().permute(3, 2, 0, 1), 'dtable': torch.empty_like(table)}
        ops.backward_relative_attention(dout, q, k, v, table, out, lse, *got.values(), buckets=b, scale=0.125)
        want, bound = ref.attention(q, k, v, table, b, 0.125, dout=dout, out_used=out, half=HALF[torch.float16])
        _within(out, want['out'], bound['out'], 'out')
        for name in got:
            _within(got[name], want[name], bound[name], name)


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements: the last sample's rows lie behind that."""
    ops = _ops()
    B, K, G, P = 5, 4096, 1024, 128
    need = 2 * B * K * G * P * 2
    if torch.cuda.mem_get_info()[0] < 2 * need:
        pytest.skip('not enough device memory')
    k = torch.zeros(B, K, G, P, dtype=torch.float16, device=DEV)
    v = torch.zeros(B, K, G, P, dtype=torch.float16, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(2)
    k[-1] = torch.randn(K, G, P, generator=gen, device=DEV)
    v[-1] = torch.randn(K, G, P, generator=gen, device=DEV)
    b = ops.relative_buckets(32, 128, False)
    table = torch.randn(32, G, generator=gen, device=DEV).half()
    for J in (1, 130):
        q = torch.randn(B, J, G, P, generator=gen, device=DEV).half().permute(3, 2, 0, 1)
        out = torch.empty_like(q)
        lengths = torch.tensor([1, 1, 1, 1, K], dtype=torch.int32, device=DEV)
        first = torch.tensor([0, 0, 0, 0, K - J], dtype=torch.int32, device=DEV)
        ops.relative_attention(q, k.permute(3, 2, 0, 1), v.permute(3, 2, 0, 1), table, out, buckets=b, scale=0.1, causal=True,
                               lengths=lengths, first=first)
        heads = [0, 500, G - 1]
        pick = lambda t: t.permute(3, 2, 0, 1)[:, heads, -1:]
        want, bound = ref.attention(q[:, heads, -1:], pick(k), pick(v), table[:, heads], b, 0.1, causal=True, first=first[-1:],
                                    half=HALF[torch.float16])
        _within(out[:, heads, -1:], want['out'], bound['out'], 'out')
        assert (out[:, :, :-1] == 0).all()


# ---- together --------------------------------------------------------------------------------------------------------
def _layer(ops, t, how, rot):
    """Norms and rotation, attention, and all gradients back to the projections."""
    qn, kn = torch.empty_like(t['q']), torch.empty_like(t['k'])
    ops.query_key_norm_rotation(t['q'], t['k'], t['qg'], t['kg'], t['pos'], qn, kn, **rot)
    out, lse = torch.empty_like(qn), torch.empty(qn.shape[1:], device=DEV)
    ops.relative_attention(qn, kn, t['v'], t['table'], out, lse, **how)
    dqn, dkn, dv, dtable = (torch.empty_like(x) for x in (qn, kn, t['v'], t['table']))
    ops.backward_relative_attention(t['dout'], qn, kn, t['v'], t['table'], out, lse, dqn, dkn, dv, dtable, **how)
    dqg, dkg = torch.empty_like(t['qg']), torch.empty_like(t['kg'])
    ops.backward_query_key_norm_rotation(dqn, dkn, t['q'], t['k'], t['qg'], t['kg'], t['pos'], dqn, dkn, dqg, dkg, **rot)
    return {'out': out, 'dq': dqn, 'dk': dkn, 'dv': dv, 'dtable': dtable, 'dq_gain': dqg, 'dk_gain': dkg}


def _layer_inputs(dtype, B=3, J=200, H=4, G=2, P=64, seed=1, order='BJHP'):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    t = {'q': _make((P, H, B, J), order, dtype, gen), 'k': _make((P, G, B, J), order, dtype, gen), 'v': _make((P, G, B, J), order, dtype, gen),
         'dout': _make((P, H, B, J), order, dtype, gen), 'qg': (1 + 0.2 * torch.randn(P, generator=gen, device=DEV)).to(dtype),
         'kg': (1 + 0.2 * torch.randn(P, generator=gen, device=DEV)).to(dtype), 'table': torch.randn(32, H, generator=gen, device=DEV).to(dtype),
         'pos': torch.arange(J, dtype=torch.int32, device=DEV).expand(B, J)}
    how = dict(buckets=_ops().relative_buckets(), scale=P ** -0.5,
               lengths=torch.tensor([J, J // 2, 0][:B], dtype=torch.int32, device=DEV))
    return t, how, dict(rotary=P // 2)


@pytest.mark.parametrize('order', ['BJHP', 'PHBJ'])
@pytest.mark.parametrize('dtype', BOTH)
def test_norms_attention_and_gradients_together(dtype, order):
    ops = _ops()
    t, how, rot = _layer_inputs(dtype, order=order)
    got = _layer(ops, t, how, rot)
    full = dict(base=10000.0, rotary=32, pairing='halves', eps=1e-6)
    leaves = {n: t[n].double().detach().requires_grad_(True) for n in ('q', 'k', 'v', 'table', 'qg', 'kg')}
    qn, kn = (ref.norm_forward(leaves[x], leaves[x + 'g'], t['pos'], **full) for x in 'qk')
    out = ref.attention(qn, kn, leaves['v'], leaves['table'], **how)[0]['out']
    out.backward(t['dout'].double())
    want = {'out': out.detach(), 'dq': leaves['q'].grad, 'dk': leaves['k'].grad, 'dv': leaves['v'].grad, 'dtable': leaves['table'].grad,
            'dq_gain': leaves['qg'].grad, 'dk_gain': leaves['kg'].grad}
    # the normed queries and keys are rounded before the scores are taken: exponents move by about half a step times sqrt(P)/8,
    # and three roundings follow; twice the usual bound of 1e-2
    for name in want:
        off = (got[name].double() - want[name]).norm() / want[name].norm()
        assert off <= (2e-2 if dtype == torch.bfloat16 else 4e-3), (name, off.item())


def test_calls_on_two_streams_and_captured_ones():
    ops = _ops()
    sets = [_layer_inputs(torch.bfloat16, seed=s, J=j) for s, j in ((1, 200), (2, 131))]
    plain = [_layer(ops, *s[:1], s[1], s[2]) for s in sets]
    torch.cuda.synchronize()
    # side by side on two streams
    streams = [torch.cuda.Stream() for _ in sets]
    res = [None, None]
    for _ in range(3):
        for i, (s, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                res[i] = _layer(ops, s[0], s[1], s[2])
    torch.cuda.synchronize()
    for a, b in zip(plain, res):
        assert all(torch.equal(a[n], b[n]) for n in a)
    # captured from one stream, replayed on two at once
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_layer(ops, s[0], s[1], s[2]))
        graphs.append(g)
    for o in outs:
        for x in o.values():
            x.fill_(float('nan'))
    torch.cuda.synchronize()
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(plain, outs):
        assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize('P', [64, 128])
@pytest.mark.parametrize('behind', [0, 5, 15])
def test_few_queries_far_behind_the_last_key(P, behind):
    """The last key is just beyond the buckets' reach, the places behind it, up to a whole piece, would be within."""
    ops = _ops()
    gen = torch.Generator(device=DEV).manual_seed(behind)
    B, H, G, J, K = 3, 4, 2, 3, 300
    q, k, v = (_make((P, h, B, n), 'BJHP', torch.float16, gen) for h, n in ((H, J), (G, K), (G, K)))
    b = ops.relative_buckets(32, 128, True)
    table = torch.randn(32, H, generator=gen, device=DEV).half()
    lengths = torch.tensor([1, 257, 289], dtype=torch.int32, device=DEV)
    how = dict(buckets=b, scale=P ** -0.5, lengths=lengths, first=lengths - 1 + b.starts[-1] + behind)
    out, lse = _nan((P, H, B, J), 'BJHP', torch.float16), torch.empty(H, B, J, device=DEV)
    ops.relative_attention(q, k, v, table, out, lse, **how)
    want, bound = ref.attention(q, k, v, table, half=HALF[torch.float16], **how)
    _within(out, want['out'], bound['out'], 'out')
    assert ((lse - want['lse']).abs() <= 1e-5 * (1 + want['lse'].abs())).all()


@pytest.mark.parametrize('P,J,causal', [(64, 161, False), (128, 161, True), (64, 65, False), (128, 65, True)])
def test_gradients_are_the_same_each_time(P, J, causal):
    """Which CTA takes which item changes from call to call, and items of an odd number of tiles change what it does next."""
    ops = _ops()
    gen = torch.Generator(device=DEV).manual_seed(J)
    B, H = 24, 8
    q, k, v, dout = (_make((P, H, B, J), 'BJHP', torch.float16, gen) for _ in range(4))
    table = torch.randn(32, H, generator=gen, device=DEV).half()
    lengths = torch.arange(J - 2 * B, J, 2, dtype=torch.int32, device=DEV)
    how = dict(buckets=ops.relative_buckets(32, 64, True), scale=P ** -0.5, causal=causal, lengths=lengths)
    out, lse = torch.empty_like(q), torch.empty(H, B, J, device=DEV)
    ops.relative_attention(q, k, v, table, out, lse, **how)
    want = None
    for _ in range(60):
        got = [torch.empty_like(x) for x in (q, k, v, table)]
        ops.backward_relative_attention(dout, q, k, v, table, out, lse, *got, **how)
        want = want or got
        assert all(torch.equal(x, y) for x, y in zip(want, got))


def test_few_queries_agree_with_many():
    """The last queries of a causal sequence, one call for all or a call for the last ones against the cache."""
    ops = _ops()
    gen = torch.Generator(device=DEV).manual_seed(6)
    b = ops.relative_buckets(32, 128, False)
    for P, H, G, K in ((64, 4, 4, 700), (128, 8, 2, 515)):
        q, k, v = (_make((P, h, 2, K), 'BJHP', torch.bfloat16, gen) for h in (H, G, G))
        table = torch.randn(32, H, generator=gen, device=DEV).bfloat16()
        full = torch.empty_like(q)
        ops.relative_attention(q, k, v, table, full, buckets=b, scale=P ** -0.5, causal=True)
        for J in (1, 3, 16):
            few = torch.empty_like(q[..., -J:])
            ops.relative_attention(q[..., -J:], k, v, table, few, buckets=b, scale=P ** -0.5, causal=True,
                                   first=torch.full((2,), K - J, dtype=torch.int32, device=DEV))
            # both round exponentials and the result once: apart by at most four half steps of sum p |v| (about 1 here)
            assert (few.float() - full[..., -J:].float()).abs().max() <= 4 * HALF[torch.bfloat16] * v.abs().max()


def test_gpu_refusals():
    ops = _ops()
    t, how, rot = _layer_inputs(torch.float16)
    out = torch.empty_like(t['q'])
    call = lambda **kw: ops.relative_attention(**{**dict(q=t['q'], k=t['k'], v=t['v'], table=t['table'], out=out), **how, **kw})
    with pytest.raises(TypeError):
        call(k=t['k'].bfloat16())
    with pytest.raises(TypeError):
        call(lengths=torch.zeros(3, device=DEV))
    with pytest.raises(ValueError):
        call(lengths=torch.zeros(2, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        call(lengths=torch.zeros(6, dtype=torch.int32, device=DEV)[::2])
    with pytest.raises(TypeError):
        call(lse=torch.zeros(4, 3, 200, device=DEV).half())
    with pytest.raises(TypeError):
        call(q=t['q'].float(), out=out.float())
    with pytest.raises(ValueError):
        call(lengths=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ops.SubstationError):
        call(table=t['table'][:31])
    with pytest.raises(TypeError):
        ops.query_key_norm_rotation(t['q'], None, t['qg'], None, t['pos'].long(), out, None)
    with pytest.raises(KeyError):
        ops.query_key_norm_rotation(t['q'], None, t['qg'], None, t['pos'], out, None, pairing='thirds')
