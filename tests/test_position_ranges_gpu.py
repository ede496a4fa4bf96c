"""Position operators on the GPU at the ends of their ranges, against float64 and against themselves: NaN and infinity inside a
sequence, gradients of any size, caches of many small weights,
biases of any size, budgets of SMs, several rotations."""

import pytest
import torch

from tests import position_reference as ref
from tests.test_positions_gpu import BOTH, DEV, _make, _nan, _ops

pytestmark = pytest.mark.gpu


# ---- NaN and infinity inside a sequence --------------------------------------------------------------------------------
# P, H, G, J, K: one share of the keys, several shares, the tile kernel
NAN_CASES = [(64, 4, 2, 1, 90), (128, 8, 2, 2, 1500), (80, 2, 2, 3, 600), (64, 4, 2, 200, 333), (128, 2, 2, 140, 140)]


def _nan_inputs(case, dtype):
    P, H, G, J, K = case
    gen = torch.Generator(device=DEV).manual_seed(P + J + K)
    q, k, v = (_make((P, h, 2, n), 'BJHP', dtype, gen) for h, n in ((H, J), (G, K), (G, K)))
    table = torch.randn(32, H, generator=gen, device=DEV).to(dtype)
    how = dict(buckets=_ops().relative_buckets(32, 128, False), scale=P ** -0.5, causal=True,
               first=torch.full((2,), K - J, dtype=torch.int32, device=DEV))
    return gen, q, k, v, table, how


def _forward(q, k, v, table, how):
    out, lse = _nan(q.shape, 'BJHP', q.dtype).fill_(7.0), torch.full(q.shape[1:], 7.0, device=DEV)
    _ops().relative_attention(q, k, v, table, out, lse, **how)
    return out, lse


@pytest.mark.parametrize('dtype', BOTH)
@pytest.mark.parametrize('case', NAN_CASES)
@pytest.mark.parametrize('what', ['query', 'key', 'infinity'])
def test_nan_and_infinity_inside_a_sequence_show(case, dtype, what):
    """A score that is NaN, or infinite, gives a NaN output and log-sum-exp to the queries that meet it, as the formula does; it is
    not taken for a query that sees no key.  All other queries keep their bits."""
    P, H, G, J, K = case
    gen, q, k, v, table, how = _nan_inputs(case, dtype)
    q[0] = q[0].abs() + 0.5
    clean = _forward(q, k, v, table, how)
    hit = torch.zeros(H, 2, J, dtype=torch.bool, device=DEV)
    if what == 'query':
        q[P // 2, 1, 1, J - 1] = float('nan')
        hit[1, 1, J - 1] = True
    else:
        at = K - (J + 1) // 2                          # a key that some of the queries see and some do not
        k[0 if what == 'infinity' else P - 1, G - 1, 0, at] = float('inf' if what == 'infinity' else 'nan')
        hit[H // G * (G - 1):, 0, at - (K - J):] = True
    out, lse = _forward(q, k, v, table, how)
    assert hit.any() and not hit.all()
    assert torch.equal(lse.isnan(), hit), 'log-sum-exp'
    assert torch.equal(out.isnan(), hit.expand(P, H, 2, J)), 'output'
    assert torch.equal(lse[~hit], clean[1][~hit]) and torch.equal(out[:, ~hit], clean[0][:, ~hit])


@pytest.mark.parametrize('dtype', BOTH)
def test_gradients_of_a_query_that_is_nan(dtype):
    """Its own gradient is NaN, that of the other queries of its head and of the other heads is not."""
    for case in NAN_CASES:
        P, H, G, J, K = case
        gen, q, k, v, table, how = _nan_inputs(case, dtype)
        q[0, 1, 1, J - 1] = float('nan')
        out, lse = _forward(q, k, v, table, how)
        dout = _make(q.shape, 'BJHP', dtype, gen)
        dout[:, 1, 1, J - 1] = 1.0
        got = [torch.empty_like(x) for x in (q, k, v, table)]
        _ops().backward_relative_attention(dout, q, k, v, table, out, lse, *got, **how)
        hit = torch.zeros(P, H, 2, J, dtype=torch.bool, device=DEV)
        hit[:, 1, 1, J - 1] = True
        assert torch.equal(got[0].isnan(), hit), case
        assert got[1][:, 1 // (H // G), 1].isnan().all() and not got[1][:, :, 0].isnan().any(), case


# ---- gradients of any size ---------------------------------------------------------------------------------------------
F32 = 1e-5                # as in position_reference


def _gradients(q, k, v, table, buckets, scale, causal, dout, used, h):
    """float64 gradients, and for dq, dk and dv the variance that roundings give each element: a rounding to 16 bits is uniform
    within half a step, at most h |x| (or 2^-25, half of float16's smallest step), of variance (h x)^2 / 3, and roundings are
    independent of one another.  Exponentials and score gradients are rounded once, results once; 32-bit sums count with F32 of
    their terms' sizes.  What the rounded output adds through D is returned by itself: it is known."""
    P, H, B, J = q.shape
    G, K = k.shape[1], k.shape[3]
    rep = H // G
    q, k, v, g = q.double(), k.double(), v.double(), dout.double()
    kk, vv = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    rel = torch.arange(K, device=DEV) - torch.arange(J, device=DEV)[:, None]
    lookup = torch.tensor([buckets.bucket(r) for r in range(1 - J, K)], device=DEV)
    s = scale * torch.einsum('phbj,phbk->hbjk', q, kk) + table.double()[lookup[rel + J - 1]].permute(2, 0, 1)[:, None]
    if causal:
        s = s.masked_fill(rel > 0, -float('inf'))
    p = s.softmax(-1)
    out = torch.einsum('hbjk,phbk->phbj', p, vv)
    dp = torch.einsum('phbj,phbk->hbjk', g, vv)
    ds = p * (dp - (g * out).sum(0)[..., None])
    size = (g.abs() * out.abs()).sum(0)[..., None] + torch.einsum('phbj,phbk->hbjk', g.abs(), vv.abs())
    var = (h * ds) ** 2 / 3 + (F32 * p * size) ** 2
    via_d = -p * (g * (used.double() - out)).sum(0)[..., None]
    fold = lambda x: x.unflatten(1, (G, rep)).sum(2)
    end = lambda x: (h * x.abs()).clamp(min=2.0 ** -25) ** 2 / 3
    want, noise, known = {}, {}, {}
    to_q = lambda w, x: torch.einsum('hbjk,phbk->phbj', w, x)
    to_k = lambda w, x: fold(torch.einsum('hbjk,phbj->phbk', w, x))
    want['dq'], known['dq'] = scale * to_q(ds, kk), scale * to_q(via_d, kk)
    noise['dq'] = scale ** 2 * to_q(var, kk ** 2) + end(want['dq'])
    want['dk'], known['dk'] = scale * to_k(ds, q), scale * to_k(via_d, q)
    noise['dk'] = scale ** 2 * to_k(var, q ** 2) + end(want['dk'])
    want['dv'], known['dv'] = to_k(p, g), torch.zeros_like(v)
    noise['dv'] = to_k(((h * p) ** 2 / 3 + (F32 * p) ** 2), g ** 2) + end(want['dv'])
    return want, noise, known


def _check_gradients(P, H, G, B, J, K, causal, dtype, make_dout, vs=1.0, ks=1.0, mirror=False):
    ops = _ops()
    gen = torch.Generator(device=DEV).manual_seed(P + J + K)
    q, k, v = (_make((P, n, B, m), 'BJHP', dtype, gen, x) for n, m, x in ((H, J, 1.0), (G, K, ks), (G, K, vs)))
    if mirror:
        for x in (q, k, v):
            x[:, :, 1] = x[:, :, 0]
    table = (0.5 * torch.randn(32, H, generator=gen, device=DEV)).to(dtype)
    buckets = ops.relative_buckets(32, 128, not causal)
    out, lse = torch.empty_like(q), torch.empty(H, B, J, device=DEV)
    how = dict(buckets=buckets, scale=P ** -0.5, causal=causal)
    ops.relative_attention(q, k, v, table, out, lse, **how)
    dout = make_dout(torch.randn(B, J, H, P, generator=gen, device=DEV)).to(dtype).permute(3, 2, 0, 1)
    got = {'dq': _nan(q.shape, 'BJHP', dtype), 'dk': _nan(k.shape, 'BJHP', dtype), 'dv': _nan(v.shape, 'BJHP', dtype),
           'dtable': torch.full_like(table, float('nan'))}
    ops.backward_relative_attention(dout, q, k, v, table, out, lse, *got.values(), **how)
    h = torch.finfo(dtype).eps / 2
    want, noise, known = _gradients(q, k, v, table, dout=dout, used=out, h=h, **how)
    for name in want:
        held = want[name].abs() < torch.finfo(dtype).max               # (what is larger is infinite)
        assert got[name][held].isfinite().all(), name
        norm = lambda x: (x.square() * held).sum((0, 1, 3)).sqrt()     # of each sample
        off, may = norm((got[name].double() - want[name]).where(held, 0.0)), (noise[name] * held).sum((0, 1, 3)).sqrt()
        # hundreds of independent roundings at least: their norm is the expected one to a few percent, and the variances are upper ends
        assert (off <= 1.1 * may + norm(known[name])).all(), (name, off, may, norm(known[name]))
    full, bound = ref.attention(q, k, v, table, half=h, dout=dout, out_used=out, **how)
    assert ((got['dtable'].double() - full['dtable']).abs() <= bound['dtable']).all(), 'dtable'


@pytest.mark.parametrize('dtype', BOTH)
@pytest.mark.parametrize('size', [1.0, 1e-3, 1e-4, 1e-5, 300.0])
@pytest.mark.parametrize('P,H,G,B,J,K,causal', [(64, 2, 2, 1, 2048, 2048, False), (128, 2, 1, 2, 700, 1500, False), (64, 4, 2, 1, 1000, 1000, True),
                                                (64, 8, 8, 4, 128, 128, False), (48, 4, 4, 2, 100, 77, False)])
def test_gradients_of_any_size_keep_their_digits(P, H, G, B, J, K, causal, size, dtype):
    """Score gradients are products of a probability and an output's gradient, and far smaller than the results.  With 16-bit numbers
    of few exponent bits they must not fall among the smallest steps while results are far from those."""
    _check_gradients(P, H, G, B, J, K, causal, dtype, lambda g: g * size)


@pytest.mark.parametrize('dtype', BOTH)
def test_gradients_of_many_keys_keep_their_digits(dtype):
    """Probabilities of one in 65536 on their way into dv."""
    _check_gradients(64, 1, 1, 1, 128, 65536, False, dtype, lambda g: g)


@pytest.mark.parametrize('dtype', BOTH)
def test_gradients_of_samples_of_very_different_sizes(dtype):
    """One sample's gradients are ten thousand times those of the next one's."""
    _check_gradients(64, 2, 2, 4, 500, 500, False, dtype, lambda g: g * torch.tensor([30.0, 3e-3, 1.0, 1e-4], device=DEV)[:, None, None, None])


def test_score_gradients_beyond_what_16_bits_hold():
    """Output gradients as a large loss scale gives them: score gradients exceed 65504, their products with small keys do not.  The
    second sample has the opposite gradients, so that the table's stay representable."""
    sign = torch.tensor([1.0, -1.0], device=DEV)[:, None, None, None]
    for P, J, K in ((64, 6, 8), (64, 150, 8), (128, 6, 8)):
        _check_gradients(P, 2, 2, 2, J, K, False, torch.float16, lambda g: (g[:1] * 1.2e4).clamp(-5e4, 5e4) * sign * (1 if J < 100 else 0.3),
                         vs=8.0, ks=0.02, mirror=True)


def test_a_gradient_without_a_number_leaves_other_queries_theirs():
    """A row of dout that is infinite does not decide how the others are rounded."""
    ops = _ops()
    for P, J in ((64, 100), (64, 300), (128, 200)):
        gen = torch.Generator(device=DEV).manual_seed(J)
        q, k, v, dout = (_make((P, 2, 1, J), 'BJHP', torch.float16, gen) for _ in range(4))
        dout *= 1e-3
        table = torch.randn(32, 2, generator=gen, device=DEV).half()
        how = dict(buckets=ops.relative_buckets(), scale=P ** -0.5)
        out, lse = torch.empty_like(q), torch.empty(2, 1, J, device=DEV)
        ops.relative_attention(q, k, v, table, out, lse, **how)
        got = []
        for bad in (False, True):
            if bad:
                dout[:, 0, 0, 7] = float('inf')
            got.append([torch.empty_like(x) for x in (q, k, v, table)])
            ops.backward_relative_attention(dout, q, k, v, table, out, lse, *got[-1], **how)
        hit = torch.zeros(2, 1, J, dtype=torch.bool, device=DEV)
        hit[0, 0, 7] = True
        assert not got[1][0][:, hit].isfinite().any()
        a, b = (g[0][:, ~hit].double() for g in got)
        assert (a - b).norm() <= 2e-3 * a.norm()


# ---- long caches -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', BOTH)
@pytest.mark.parametrize('H,J', [(150, 1), (20, 130)])
def test_many_small_weights_count(dtype, H, J):
    """Four keys outweigh each of 131068 others by 2^26, together those have a weight of 2^-11, and all of the values.  One share of the
    keys, and the tile kernel."""
    ops = _ops()
    K, P = 1 << 17, 64
    q = torch.zeros(1, J, H, P, dtype=dtype, device=DEV).permute(3, 2, 0, 1)
    q[0] = 4.0
    k = torch.zeros(1, K, 1, P, dtype=dtype, device=DEV)
    k[0, 0:128:32, 0, 0] = 4.5
    v = torch.ones(1, K, 1, P, dtype=dtype, device=DEV)
    v[0, 0:128:32] = 0
    k, v = (x.permute(3, 2, 0, 1).expand(P, H, 1, K) for x in (k, v))
    table = torch.zeros(1, H, dtype=dtype, device=DEV)
    out, lse = torch.empty_like(q), torch.empty(H, 1, J, device=DEV)
    ops.relative_attention(q, k, v, table, out, lse, buckets=ops.RelativeBuckets([0], False), scale=1.0)
    few = (K - 4) * torch.tensor(-18.0, dtype=torch.float64).exp()
    want, h = (few / (4 + few)).item(), torch.finfo(dtype).eps / 2
    # exponentials are rounded once (all alike), the result once; float16 holds them in steps of 2^-31 of the largest in the tile
    # kernel, of 2^-39 elsewhere
    step = 0.0 if dtype is torch.bfloat16 else 2.0 ** -32 * K / 4 if J > 1 else 2.0 ** -40 * K / 4
    assert ((out.double() - want).abs() <= 2.02 * h * want + F32 * want + step).all(), (out.flatten()[0].item(), want)
    assert ((lse.double() - (18 + (4 + few).log())).abs() <= 1e-5 * 20).all()


# ---- biases of any size ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', BOTH)
@pytest.mark.parametrize('J', [1, 150])
def test_biases_up_to_the_largest(dtype, J):
    """The largest number of the type in one bucket: its keys share the row, and nothing is NaN.  What is above 2^127 counts as 2^127."""
    ops = _ops()
    gen = torch.Generator(device=DEV).manual_seed(J)
    P, H, K = 64, 3, 400
    q, k, v = (_make((P, H, 2, n), 'BJHP', dtype, gen) for n in (J, K, K))
    table = torch.randn(8, H, generator=gen, device=DEV).to(dtype)
    table[1, 0] = table[5, 1] = table[0, 2] = torch.finfo(dtype).max
    table[3, 2] = 0.75 * torch.finfo(dtype).max
    how = dict(buckets=ops.relative_buckets(8, 20, True), scale=0.125, first=torch.tensor([0, 200], dtype=torch.int32, device=DEV))
    out, lse = _forward(q, k, v, table, how)
    full = dict(how, table=table.double().clamp(max=2.0 ** 127))
    h = torch.finfo(dtype).eps / 2
    want, bound = ref.attention(q, k, v, half=h, **full)
    assert ((lse - want['lse']).abs() <= 1e-5 * (1 + want['lse'].abs())).all()
    # A score beside a bias of 2^104 or more is below half a step of their 32-bit sum, and whether it is rounded away depends on the
    # order of the sums: of such rows only that the keys with the largest bias share them, so that each feature lies between those
    # keys' least and largest value.  (65504 in 32 bits moves an exponent by half a step of that, 2^-9.)
    rel = torch.arange(K, device=DEV) - torch.arange(J, device=DEV)[:, None] - how['first'][:, None, None]            # [B,J,K]
    lookup = torch.tensor([how['buckets'].bucket(r) for r in range(-K - J, K + J)], device=DEV)
    bias = full['table'][lookup[rel + K + J]].permute(3, 0, 1, 2)                                                    # [H,B,J,K]
    top = bias.amax(-1, keepdim=True)
    huge = (top > 2.0 ** 100).squeeze(-1)
    shares = bias == top
    off = 2.02 * h * v.abs().max().double() + ref.SMALL
    for p in range(P):
        x = v[p].double()[:, :, None].expand(H, 2, J, K)
        least, most = x.masked_fill(~shares, torch.inf).amin(-1), x.masked_fill(~shares, -torch.inf).amax(-1)
        assert ((out[p] >= least - off) & (out[p] <= most + off))[huge].all()
    loose = 2.0 ** -8 * want['out'].abs().max() if dtype is torch.float16 else 0.0
    assert ((out.double() - want['out']).abs() <= bound['out'] + loose)[:, ~huge].all()
    dout = _make(q.shape, 'BJHP', dtype, gen)
    got = [torch.empty_like(x) for x in (q, k, v, table)]
    ops.backward_relative_attention(dout, q, k, v, table, out, lse, *got, **how)
    assert all(x.isfinite().all() for x in got)


# ---- a budget of SMs ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('P,H,G,B,J,K', [(64, 16, 16, 2, 1, 3000), (128, 16, 4, 8, 2, 900), (64, 8, 8, 2, 300, 300), (64, 6, 6, 30, 128, 128),
                                         (128, 8, 2, 2, 200, 257)])
def test_results_do_not_depend_on_the_sm_budget(P, H, G, B, J, K):
    """Outputs and gradients keep their bits; the gains' gradients, sums over a different number of rows, stay within rounding."""
    ops = _ops()
    gen = torch.Generator(device=DEV).manual_seed(K)
    q, k, v, dout = (_make((P, h, B, n), 'BJHP', torch.float16, gen) for h, n in ((H, J), (G, K), (G, K), (H, J)))
    table, gain = torch.randn(32, H, generator=gen, device=DEV).half(), (1 + 0.1 * torch.randn(P, generator=gen, device=DEV)).half()
    how = dict(buckets=ops.relative_buckets(), scale=P ** -0.5)
    pos = torch.arange(J, dtype=torch.int32, device=DEV).expand(B, J)

    def run():
        out, lse = _forward(q, k, v, table, how)
        got = [torch.empty_like(x) for x in (q, k, v, table)]
        ops.backward_relative_attention(dout, q, k, v, table, out, lse, *got, **how)
        y, dx, dg = torch.empty_like(q), torch.empty_like(q), torch.empty_like(gain)
        ops.query_key_norm_rotation(q, None, gain, None, pos, y, None)
        ops.backward_query_key_norm_rotation(dout, None, q, None, gain, None, pos, dx, None, dg, None)
        return [out, lse, y, dx] + got, dg
    try:
        seen = []
        for budget in (0, 136, 100, 3):
            ops.set_sm_budget(budget)
            seen.append(run())
    finally:
        ops.set_sm_budget(0)
    for got, dg in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got, seen[0][0]))
        assert (dg.float() - seen[0][1].float()).norm() <= 2e-3 * seen[0][1].float().norm()
    assert ops.device_error() == 0


# ---- two rotations in turn ---------------------------------------------------------------------------------------------
def test_alternating_rotations_cost_no_more_than_one():
    """Layers of local and of global attention have bases of their own.  Host time of a call, the least of many: frequencies are not
    worked out again (11 us a call for 64 features, 22 for 128)."""
    import time
    ops = _ops()
    q = torch.randn(1, 1, 1, 128, device=DEV).half().permute(3, 2, 0, 1)
    gain, pos, out = torch.ones(128, device=DEV).half(), torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.empty_like(q)

    def least(bases):
        best = 1e9
        for _ in range(400):
            torch.cuda.synchronize()
            t = time.perf_counter()
            for b in bases:
                ops.query_key_norm_rotation(q, None, gain, None, pos, out, None, base=b)
            best = min(best, time.perf_counter() - t)
        return best / len(bases)
    one, four = least([1e4] * 4), least([1e4, 1e6, 5e5, 500.0])
    assert four <= one + 4e-6, (one, four)


@pytest.mark.parametrize('dtype', BOTH)
def test_many_rotations_in_turn(dtype):
    """More rotations than are remembered, twice each, in one thread and in another beside it."""
    import threading
    ops = _ops()
    gen = torch.Generator(device=DEV).manual_seed(8)
    q = _make((64, 2, 2, 9), 'BJHP', dtype, gen)
    gain = torch.ones(64, device=DEV).to(dtype)
    pos = torch.randint(-5000, 1 << 21, (2, 9), generator=gen, device=DEV, dtype=torch.int32)
    rotations = [(b, r) for b in (100.0, 1e4, 1e6) for r in (0, 2, 32, 64)]
    wrong = []

    def turns():
        for base, rotary in 2 * rotations + rotations[::-1]:
            out = torch.empty_like(q)
            ops.query_key_norm_rotation(q, None, gain, None, pos, out, None, base=base, rotary=rotary)
            want = ref.norm_forward(q, gain, pos, base, rotary, 'halves', 1e-6)
            bound = torch.finfo(dtype).eps / 2 * 1.01 * want.abs() + 2e-6 * want.abs().amax(0, keepdim=True) + ref.SMALL
            if ((out.double() - want).abs() > bound).any():
                wrong.append((base, rotary))
    threads = [threading.Thread(target=turns) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize('dtype', BOTH)
@pytest.mark.parametrize('size,values', [(30.0, 1.0), (30.0, 8.0), (1000.0, 0.05)])
@pytest.mark.parametrize('P,H,G,B,J,K', [(64, 1, 1, 5, 3, 289), (80, 3, 3, 8, 2, 465), (128, 6, 2, 2, 1, 692), (64, 4, 4, 4, 5, 100)])
def test_gradients_of_keys_that_hardly_count(P, H, G, B, J, K, size, values, dtype):
    """Large output gradients, few queries and sharp softmaxes: keys of a weight of 1e-6 and less have gradients that are small beside the
    others' of their item, but not beside what the type holds."""
    ops = _ops()
    gen = torch.Generator(device=DEV).manual_seed(K)
    q, k, v, dout = (_make((P, h, B, n), 'BJHP', dtype, gen, x) for h, n, x in ((H, J, 2.0), (G, K, 2.0), (G, K, values), (H, J, size)))
    table = torch.randn(32, H, generator=gen, device=DEV).to(dtype)
    how = dict(buckets=ops.relative_buckets(), scale=P ** -0.5)
    out, lse = _forward(q, k, v, table, how)
    got = {n: torch.empty_like(x) for n, x in (('dq', q), ('dk', k), ('dv', v), ('dtable', table))}
    ops.backward_relative_attention(dout, q, k, v, table, out, lse, *got.values(), **how)
    want, bound = ref.attention(q, k, v, table, half=torch.finfo(dtype).eps / 2, dout=dout, out_used=out, **how)
    # float16's numbers spread over 2^40, from 2^-24 on: an item whose score gradients may be as large as N = |dout| (|v| + |out|) rounds
    # them in steps of 2^-24 times 2^-shift, and 2^-shift is below sqrt(2) 2 N / 2^15; the reference counts 2^-24
    N = (dout.double().norm(dim=0).max() * (v.double().norm(dim=0).max() + out.double().norm(dim=0).max())).item()
    coarse = 2.0 ** -25 * max(0.0, 2 ** 1.5 * N / 2 ** 15 - 1) if dtype is torch.float16 else 0.0
    bound['dq'] = bound['dq'] + coarse * how['scale'] * k.double().abs().sum(3, keepdim=True).repeat_interleave(H // G, 1)
    bound['dk'] = bound['dk'] + coarse * how['scale'] * q.double().abs().sum(3, keepdim=True).unflatten(1, (G, H // G)).sum(2)
    for name in got:
        held = want[name].abs() + bound[name] < torch.finfo(dtype).max
        assert ((got[name].double() - want[name]).abs() <= bound[name])[held].all(), name


# ---- what float16's range costs ----------------------------------------------------------------------------------------
@pytest.mark.parametrize('J,K', [(64, 65536), (16384, 128)])
def test_the_range_of_float16_costs_little_whatever_the_shape(J, K):
    """What is looked at to find an item's powers of two grows as the item does: a backward call of few queries against many keys takes as
    long in float16 as in bfloat16, which has no such thing (twice as long where every item looked at all values)."""
    ops = _ops()
    took = []
    for dtype in BOTH:
        gen = torch.Generator(device=DEV).manual_seed(1)
        q, k, v, dout = (_make((64, 1, 1, n), 'BJHP', dtype, gen) for n in (J, K, K, J))
        table = torch.randn(32, 1, generator=gen, device=DEV).to(dtype)
        how = dict(buckets=ops.relative_buckets(), scale=0.125)
        out, lse = torch.empty_like(q), torch.empty(1, 1, J, device=DEV)
        got = [torch.empty_like(x) for x in (q, k, v, table)]
        ops.relative_attention(q, k, v, table, out, lse, **how)
        call = lambda: ops.backward_relative_attention(dout, q, k, v, table, out, lse, *got, **how)
        graph = torch.cuda.CUDAGraph()
        call()
        with torch.cuda.graph(graph):
            for _ in range(4):
                call()
        times = []
        for _ in range(9):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            graph.replay()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        took.append(min(times))
    assert took[0] <= 1.3 * took[1], took
