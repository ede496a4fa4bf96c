"""Position operators on the GPU at the ends of their ranges, against float64 and against themselves: NaN and infinity inside a
sequence."""

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
