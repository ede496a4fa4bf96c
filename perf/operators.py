"""Performance cases of the operators that give attention its positions.

Two pairs of operators and the attention that reads what they prepare (``substation_b200.ops``):

norm               ``query_key_norm_rotation``: root-mean-square norm of every query and key head with a learned gain,
                   then the rotation of feature pairs by position, queries and keys in one call
norm_backward      ``backward_query_key_norm_rotation``: gradients of queries, keys and both gains
attention          ``relative_attention``: attention with a learned bias per head and bucket of relative positions, with
                   the length of each sample's keys, and with few queries against a long cache
attention_training the same and ``backward_relative_attention``: output, gradients of queries, keys, values and of the
                   table of biases

A case is a dict of plain values: ``kind`` (above), ``batch``, ``queries``, ``keys`` (attention only), ``heads``,
``kv_heads``, ``head`` (features of a head), ``dtype``, and

layout      'feature': [batch, token, head, feature] in memory, 'head_first': [feature, head, batch, token], the order of
            the layer's stacked projections
rotary, pairing, far     rotated features of a head, 'halves' or 'adjacent' pairs, the largest position
buckets, distance        entries of the table and the distance from which on all keys share one
causal      queries see no later keys; the buckets then know one direction only
ragged      keys per sample: 'full', 'ragged' (from all down to about half of them), 'empty' (the same, and the last
            sample has none), or 'cache' (ragged, and the queries are the last tokens of what the cache holds)
"""

import math

import torch

own = False

BASE = 10000.0
EPS = 1e-6
DTYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16}


def _norm(name, kind, batch, queries, heads, kv_heads, head, dtype, layout='feature', rotary=None, pairing='halves', far=4096):
    c = {'kind': kind, 'batch': batch, 'queries': queries, 'heads': heads, 'kv_heads': kv_heads, 'head': head, 'dtype': dtype,
         'layout': layout, 'rotary': head if rotary is None else rotary, 'pairing': pairing, 'far': far}
    if name:
        c['name'] = name
    return c


def _attention(name, kind, batch, queries, keys, heads, kv_heads, head, dtype, layout='feature', buckets=32, distance=128,
               causal=False, ragged='full'):
    c = {'kind': kind, 'batch': batch, 'queries': queries, 'keys': keys, 'heads': heads, 'kv_heads': kv_heads, 'head': head,
         'dtype': dtype, 'layout': layout, 'buckets': buckets, 'distance': distance, 'causal': causal, 'ragged': ragged}
    if name:
        c['name'] = name
    return c


def listed():
    return [
        # one new token of each of a few sequences: nothing but latency
        _norm('norm_single_tokens', 'norm', 8, 1, 16, 16, 64, 'bf16'),
        # the projections of one BERT-large layer at the headline batch
        _norm('norm_b8_l512', 'norm', 8, 512, 16, 16, 64, 'fp16'),
        # projections in the layer's head-first order, a length that no tile divides, half of the features rotated
        _norm('norm_b12_l200_head_first', 'norm', 12, 200, 12, 12, 64, 'fp16', 'head_first', 32, 'adjacent'),
        # the backward pass of the headline batch
        _norm('norm_backward_b8_l512', 'norm_backward', 8, 512, 16, 16, 64, 'bf16'),
        # long documents, wide heads, four query heads to a key head, positions far out
        _norm('norm_backward_b4_l4096_p128', 'norm_backward', 4, 4096, 32, 8, 128, 'bf16', far=1 << 20),
        # inference over a padded batch, one place of which is not taken
        _attention('attention_b16_l384_padded', 'attention', 16, 384, 384, 16, 16, 64, 'bf16', ragged='empty'),
        # a step of the headline layer's attention
        _attention('training_b8_l512', 'attention_training', 8, 512, 512, 16, 16, 64, 'bf16'),
        # large batch, short sequences (the first pre-training phase)
        _attention('training_b96_l128', 'attention_training', 96, 128, 128, 16, 16, 64, 'fp16'),
        # a decoder's attention: causal, shared key heads, a length that no tile divides
        _attention('training_b2_l2000_causal_p128', 'attention_training', 2, 2000, 2000, 16, 4, 128, 'bf16', causal=True),
        # long documents
        _attention('training_b2_l4096', 'attention_training', 2, 4096, 4096, 16, 16, 64, 'bf16', buckets=64, distance=512),
        # one new token against a short cache: latency
        _attention('token_b1_k77', 'attention', 1, 1, 77, 16, 16, 64, 'fp16', causal=True, ragged='cache'),
        # one new token of each of many sequences against long caches: reading the caches
        _attention('token_b16_k8192_p128', 'attention', 16, 1, 8192, 32, 8, 128, 'bf16', causal=True, ragged='cache'),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['norm', 'norm_backward', 'attention', 'attention_training', 'attention_training', 'token'])
    head = rng.choice([32, 64, 64, 80, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 4] if kv_heads <= 8 else [1])
    dtype = rng.choice(['fp16', 'bf16'])
    layout = rng.choice(['feature', 'feature', 'head_first'])
    if kind in ('norm', 'norm_backward'):
        tokens = _log(rng, 1, 16384)
        batch = min(tokens, _log(rng, 1, 64))
        return _norm(None, kind, batch, max(1, tokens // batch), heads, kv_heads, head, dtype, layout,
                     rng.choice([head, head, head // 2]), rng.choice(['halves', 'adjacent']), rng.choice([512, 4096, 1 << 20]))
    buckets = rng.choice([16, 32, 32, 64, 320])
    distance = rng.choice([64, 128, 128, 512, 800]) if buckets <= 64 else 800
    if kind == 'token':
        keys = _log(rng, 1, 16384)
        batch = max(1, min(_log(rng, 1, 64), 10 ** 8 // (keys * kv_heads * head)))
        return _attention(None, 'attention', batch, min(keys, rng.choice([1, 1, 1, 2, 5])), keys, heads, kv_heads, head, dtype,
                          'feature', buckets, distance, True, 'cache')
    # (a single key has a probability of one and no gradient but rounding, so training starts at a few)
    keys = _log(rng, 4 if kind == 'attention_training' else 1, 4096)
    queries = keys if rng.random() < 0.8 else _log(rng, 1, 4096)
    causal = queries == keys and rng.random() < 0.4
    batch = max(1, min(_log(rng, 1, 96), 2 ** 28 // (queries * keys * heads)))
    return _attention(None, kind, batch, queries, keys, heads, kv_heads, head, dtype, layout, buckets, distance, causal,
                      rng.choice(['full', 'ragged', 'empty']))


# ---- sizes that follow from a case ----------------------------------------------------------------------------------
def _lengths(case):
    """Keys of each sample."""
    B, K = case['batch'], case['keys']
    if case['ragged'] == 'full':
        return [K] * B
    n = [max(1, K - b * K // (2 * B)) for b in range(B)]
    if case['ragged'] == 'cache':
        n = [max(x, min(K, case['queries'])) for x in n]
    if case['ragged'] == 'empty' and B > 1:
        n[-1] = 0
    return n


def _first(case):
    """Position of each sample's first query among its keys."""
    return [n - case['queries'] if case['ragged'] == 'cache' else 0 for n in _lengths(case)]


def _pairs(case):
    """Pairs of a query and a key that it sees, over the batch and for one head."""
    J, total = case['queries'], 0
    for n, s in zip(_lengths(case), _first(case)):
        if not case['causal']:
            total += J * n
        else:
            # row j sees min(n, s + j + 1) keys, at least none
            full = max(0, min(J, J - (n - s) + 1))       # rows that see all n
            rest = J - full
            lo = max(0, -s)                              # rows before the first key
            total += full * n + sum(s + j + 1 for j in range(lo, rest))
    return total


def work(case):
    B, J, H, G, P = case['batch'], case['queries'], case['heads'], case['kv_heads'], case['head']
    if case['kind'] in ('norm', 'norm_backward'):
        elements = B * J * (H + G) * P
        back = case['kind'] == 'norm_backward'
        return {'bytes': elements * (6 if back else 4) + 4 * B * J + 2 * P * (4 if back else 2), 'flops': elements * (14 if back else 7)}
    keys = sum(_lengths(case))
    q, kv = 2 * B * J * H * P, 2 * keys * G * P
    table = 2 * case['buckets'] * H
    if case['kind'] == 'attention':
        return {'bytes': 2 * q + 2 * kv + table + 8 * B, 'flops': 4 * P * H * _pairs(case)}
    return {'bytes': 4 * q + 2 * kv + 2 * 2 * B * case['keys'] * G * P + 2 * table, 'flops': 12 * P * H * _pairs(case)}


# ---- buckets --------------------------------------------------------------------------------------------------------
def _bucket_starts(buckets, distance):
    """First distance of each bucket of one direction: one distance a bucket in the first half, then a constant ratio up
    to ``distance``.  Whole numbers throughout, because some borders are distances themselves."""
    exact = buckets // 2
    steps = buckets - exact
    starts = list(range(exact))
    d = exact
    for i in range(steps):
        # smallest d with log(d / exact) / log(distance / exact) >= i / steps
        while d ** steps * exact ** i < distance ** i * exact ** steps:
            d += 1
        starts.append(d)
    return starts


_starts_of = {}


def _starts(case):
    n = case['buckets'] if case['causal'] else case['buckets'] // 2
    key = (n, case['distance'])
    if key not in _starts_of:
        _starts_of[key] = _bucket_starts(*key)
    return _starts_of[key]


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _random(gen, case, tokens, heads, scale=1.0):
    """[feature, head, batch, token] view of normal numbers in the case's memory order."""
    B, P = case['batch'], case['head']
    shape = (B, tokens, heads, P) if case['layout'] == 'feature' else (P, heads, B, tokens)
    t = (torch.randn(shape, generator=gen, device='cuda') * scale).to(DTYPES[case['dtype']])
    return t.permute(3, 2, 0, 1) if case['layout'] == 'feature' else t


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    dtype = DTYPES[case['dtype']]
    B, J, H, G, P = case['batch'], case['queries'], case['heads'], case['kv_heads'], case['head']
    s = {'case': case}
    if case['kind'] in ('norm', 'norm_backward'):
        s['q'], s['k'] = _random(gen, case, J, H, 2.0), _random(gen, case, J, G, 2.0)
        s['q_gain'] = (1 + 0.2 * torch.randn(P, generator=gen, device='cuda')).to(dtype)
        s['k_gain'] = (1 + 0.2 * torch.randn(P, generator=gen, device='cuda')).to(dtype)
        first = torch.randint(0, case['far'], (B, 1), generator=gen, device='cuda')
        s['positions'] = (first + torch.arange(J, device='cuda')).to(torch.int32)
        if case['kind'] == 'norm_backward':
            s['dq_out'], s['dk_out'] = _random(gen, case, J, H), _random(gen, case, J, G)
        return s
    K = case['keys']
    s['q'], s['k'], s['v'] = _random(gen, case, J, H), _random(gen, case, K, G), _random(gen, case, K, G)
    s['table'] = torch.randn(case['buckets'], H, generator=gen, device='cuda').to(dtype)
    s['scale'] = P ** -0.5
    ragged = case['ragged'] != 'full'
    s['lengths'] = torch.tensor(_lengths(case), dtype=torch.int32, device='cuda') if ragged else None
    s['first'] = torch.tensor(_first(case), dtype=torch.int32, device='cuda') if case['ragged'] == 'cache' else None
    if case['kind'] == 'attention_training':
        s['dout'] = _random(gen, case, J, H)
    return s


# ---- the framework's calls ------------------------------------------------------------------------------------------
def _run_own(s):
    from substation_b200 import ops
    case = s['case']
    if case['kind'] in ('norm', 'norm_backward'):
        how = dict(base=BASE, rotary=case['rotary'], pairing=case['pairing'], eps=EPS)
        q, k = s['q'], s['k']
        a, b = torch.empty_like(q), torch.empty_like(k)
        if case['kind'] == 'norm':
            ops.query_key_norm_rotation(q, k, s['q_gain'], s['k_gain'], s['positions'], a, b, **how)
            return {'q': a, 'k': b}
        dqg, dkg = torch.empty_like(s['q_gain']), torch.empty_like(s['k_gain'])
        ops.backward_query_key_norm_rotation(s['dq_out'], s['dk_out'], q, k, s['q_gain'], s['k_gain'], s['positions'], a, b, dqg,
                                             dkg, **how)
        return {'dq': a, 'dk': b, 'dq_gain': dqg, 'dk_gain': dkg}
    q, k, v, table = s['q'], s['k'], s['v'], s['table']
    how = dict(buckets=ops.relative_buckets(case['buckets'], case['distance'], bidirectional=not case['causal']), scale=s['scale'],
               causal=case['causal'], lengths=s['lengths'], first=s['first'])
    out = torch.empty_like(q)
    if case['kind'] == 'attention':
        ops.relative_attention(q, k, v, table, out, **how)
        return {'out': out}
    lse = torch.empty(q.shape[1:], dtype=torch.float32, device=q.device)
    ops.relative_attention(q, k, v, table, out, lse, **how)
    dq, dk, dv, dtable = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.empty_like(table)
    ops.backward_relative_attention(s['dout'], q, k, v, table, out, lse, dq, dk, dv, dtable, **how)
    return {'out': out, 'dq': dq, 'dk': dk, 'dv': dv, 'dtable': dtable}


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _angles(case, positions):
    """cos and sin of [batch, token, pair]: the angle in 64 bits, far positions turn many times."""
    R = case['rotary']
    f = BASE ** (-torch.arange(0, R, 2, device=positions.device, dtype=torch.float64) / R)
    a = positions.double()[..., None] * f
    return a.cos().float(), a.sin().float()


def _rotate(case, y, cos, sin):
    """y [head, batch, token, feature]; the rotation's transpose for a negated ``sin``."""
    R = case['rotary']
    if case['pairing'] == 'halves':
        a, b = y[..., :R // 2], y[..., R // 2:R]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = y[..., 0:R:2], y[..., 1:R:2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([r, y[..., R:]], -1)


def _plain_norm(s):
    case = s['case']
    cos, sin = _angles(case, s['positions'])
    out = {}
    for name in ('q', 'k'):
        x = s[name].permute(1, 2, 3, 0).float()
        gain = s[name + '_gain'].float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        n = x * r
        if case['kind'] == 'norm':
            out[name] = _rotate(case, n * gain, cos, sin).to(s[name].dtype).permute(3, 0, 1, 2)
            continue
        g = _rotate(case, s['d%s_out' % name].permute(1, 2, 3, 0).float(), cos, -sin)
        w = g * gain
        out['d' + name] = (r * (w - n * (w * n).mean(-1, keepdim=True))).to(s[name].dtype).permute(3, 0, 1, 2)
        out['d%s_gain' % name] = (g * n).sum((0, 1, 2)).to(s[name].dtype)
    return out


def _plain_attention(s):
    case = s['case']
    dev, dtype = s['q'].device, s['q'].dtype
    B, J, K, H, G = case['batch'], case['queries'], case['keys'], case['heads'], case['kv_heads']
    shared = H // G
    q = s['q'].permute(1, 2, 3, 0).float()                                       # [head, batch, token, feature]
    keys = torch.arange(K, device=dev)
    seen = torch.ones(B, 1, K, dtype=torch.bool, device=dev)
    if s['lengths'] is not None:
        seen = (keys < s['lengths'][:, None])[:, None]                           # [batch, 1, key]
    k, v = (torch.where(seen.transpose(1, 2), s[n].permute(1, 2, 3, 0).float(), 0.0).repeat_interleave(shared, 0) for n in 'kv')
    first = torch.zeros(B, dtype=torch.int32, device=dev) if s['first'] is None else s['first']
    place = first[:, None] + torch.arange(J, device=dev)                         # [batch, query]
    rel = keys - place[..., None]                                                # [batch, query, key]
    starts = torch.tensor(_starts(case), device=dev)
    if case['causal']:
        seen = seen & (rel <= 0)
        bucket = torch.searchsorted(starts, (-rel).clamp(min=0), right=True) - 1
    else:
        bucket = torch.searchsorted(starts, rel.abs(), right=True) - 1 + (rel > 0) * (case['buckets'] // 2)
    p = q @ k.transpose(-1, -2) * s['scale']
    p += s['table'].float()[bucket].permute(3, 0, 1, 2)
    p.masked_fill_(~seen, -math.inf)
    m = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = p @ v
    out = {'out': o.to(dtype).permute(3, 0, 1, 2)}
    if case['kind'] == 'attention':
        return out
    do = s['dout'].permute(1, 2, 3, 0).float()
    dv = p.transpose(-1, -2) @ do
    ds = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True))
    dq = ds @ k * s['scale']
    dk = ds.transpose(-1, -2) @ q * s['scale']
    out['dq'] = dq.to(dtype).permute(3, 0, 1, 2)
    for name, d in (('dk', dk), ('dv', dv)):
        out[name] = d.unflatten(0, (G, shared)).sum(1).to(dtype).permute(3, 0, 1, 2)
    flat = bucket.flatten()
    dtable = [torch.bincount(flat, ds[h].flatten().double(), case['buckets']) for h in range(H)]
    out['dtable'] = torch.stack(dtable, 1).to(dtype)
    return out


def run(state):
    if own:
        return _run_own(state)
    if state['case']['kind'] in ('norm', 'norm_backward'):
        return _plain_norm(state)
    return _plain_attention(state)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _exact_norm(s):
    case = s['case']
    P, R = case['head'], case['rotary']
    dev = s['q'].device
    half = R // 2
    pairs = [(i, i + half) if case['pairing'] == 'halves' else (2 * i, 2 * i + 1) for i in range(half)]
    ia = torch.tensor([a for a, _ in pairs], device=dev)
    ib = torch.tensor([b for _, b in pairs], device=dev)
    freq = torch.tensor([math.pow(BASE, -2.0 * i / R) for i in range(half)], dtype=torch.float64, device=dev)
    angle = s['positions'].double().unsqueeze(-1) * freq                         # [batch, token, pair]
    z = torch.polar(torch.ones_like(angle), angle)

    def spin(x, w):                                                              # [batch, token, head, feature]
        c = torch.complex(x[..., ia], x[..., ib]) * w.unsqueeze(2)
        y = x.clone()
        y[..., ia], y[..., ib] = c.real, c.imag
        return y
    out = {}
    for name in ('q', 'k'):
        x = s[name].double().permute(2, 3, 1, 0)
        gain = s[name + '_gain'].double()
        rms = (x.square().sum(-1, keepdim=True) / P + EPS).sqrt()
        if case['kind'] == 'norm':
            out[name] = spin(x / rms * gain, z).permute(3, 2, 0, 1)
            continue
        g = spin(s['d%s_out' % name].double().permute(2, 3, 1, 0), z.conj())
        along = (g * gain * x).sum(-1, keepdim=True) / (P * rms ** 3)
        out['d' + name] = (g * gain / rms - x * along).permute(3, 2, 0, 1)
        out['d%s_gain' % name] = (g * x / rms).flatten(0, 2).sum(0)
    return out


def _exact_attention(s):
    case = s['case']
    dev = s['q'].device
    B, J, K, H, G, P = (case[n] for n in ('batch', 'queries', 'keys', 'heads', 'kv_heads', 'head'))
    train = case['kind'] == 'attention_training'
    f8 = dict(dtype=torch.float64, device=dev)
    out = {'out': torch.zeros(P, H, B, J, **f8)}
    if train:
        out.update(dq=torch.zeros(P, H, B, J, **f8), dk=torch.zeros(P, G, B, K, **f8), dv=torch.zeros(P, G, B, K, **f8),
                   dtable=torch.zeros(case['buckets'], H, **f8))
    # the bucket of every distance, counted off one by one
    starts = _starts(case)
    reach = max(J, K) + max([0] + _first(case)) + 1
    of, i = [], 0
    for d in range(reach):
        while i + 1 < len(starts) and starts[i + 1] <= d:
            i += 1
        of.append(i)
    of = torch.tensor(of, device=dev)
    for b, (n, s0) in enumerate(zip(_lengths(case), _first(case))):
        if n == 0:
            continue
        gap = torch.arange(n, device=dev)[None, :] - (s0 + torch.arange(J, device=dev))[:, None]
        if case['causal']:
            hidden, index = gap > 0, of[(-gap).clamp(min=0)]
        else:
            hidden, index = None, of[gap.abs()] + torch.where(gap > 0, case['buckets'] // 2, 0)
        for h in range(H):
            q, k, v = s['q'][:, h, b].double(), s['k'][:, h // (H // G), b, :n].double(), s['v'][:, h // (H // G), b, :n].double()
            w = torch.einsum('pj,pk->jk', q, k) * s['scale'] + s['table'][:, h].double()[index]
            if hidden is not None:
                w = w.masked_fill(hidden, -math.inf)
            w = torch.softmax(w, -1).nan_to_num(0.0)                             # a row that sees nothing gives zeros
            o = torch.einsum('jk,pk->pj', w, v)
            out['out'][:, h, b] = o
            if not train:
                continue
            g = s['dout'][:, h, b].double()
            d = w * (torch.einsum('pj,pk->jk', g, v) - (g * o).sum(0)[:, None])
            out['dq'][:, h, b] = torch.einsum('jk,pk->pj', d, k) * s['scale']
            out['dk'][:, h // (H // G), b, :n] += torch.einsum('jk,pj->pk', d, q) * s['scale']
            out['dv'][:, h // (H // G), b, :n] += torch.einsum('jk,pj->pk', w, g)
            out['dtable'][:, h] += torch.bincount(index.flatten(), d.flatten(), case['buckets'])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case['kind'] in ('norm', 'norm_backward'):
        return _exact_norm(s)
    if case['batch'] * case['heads'] > 8192:       # one matrix after the other: more would take too long
        return None
    return _exact_attention(s)
