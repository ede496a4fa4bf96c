"""Float64 restatements of the position operators, with what 16-bit storage may add to each result.

``norm_forward`` / ``norm_backward``: root-mean-square norm and rotation.  ``attention`` returns outputs, gradients and, for
each of them, a bound on the distance of a kernel that rounds exponentials and score gradients to 16 bits once each, keeps
sums in 32 bits and rounds results once.  ``h`` is half a step of the storage type, ``torch.finfo(t).eps / 2``.
"""

import math

import torch

SMALL = 2.0 ** -25        # half the smallest fp16 step: what rounding to a subnormal number may be off by
F32 = 1e-5                # 32-bit sums of a few hundred products, exponents up to about 60: 2^-24 * 60 * some


def angles(positions, rotary, base):
    i = torch.arange(0, rotary, 2, dtype=torch.float64, device=positions.device)
    return positions.double()[..., None] * base ** (-i / max(rotary, 1))


def turn(x, ang, rotary, pairing, back=False):
    """x [P,H,B,J], ang [B,J,R/2]"""
    x = x.clone()
    c, s = ang.cos().permute(2, 0, 1)[:, None], ang.sin().permute(2, 0, 1)[:, None]
    if back:
        s = -s
    half = rotary // 2
    ia = torch.arange(half, device=x.device) * (1 if pairing == 'halves' else 2)
    ib = ia + (half if pairing == 'halves' else 1)
    a, b = x[ia], x[ib]
    x[ia], x[ib] = a * c - b * s, b * c + a * s
    return x


def norm_forward(x, gain, positions, base, rotary, pairing, eps):
    x, gain = x.double(), gain.double()
    n = x / (x.square().mean(0, keepdim=True) + eps).sqrt()
    return turn(n * gain[:, None, None, None], angles(positions, rotary, base), rotary, pairing)


def norm_backward(dout, x, gain, positions, base, rotary, pairing, eps):
    x, gain = x.double(), gain.double()
    r = 1 / (x.square().mean(0, keepdim=True) + eps).sqrt()
    n = x * r
    g = turn(dout.double(), angles(positions, rotary, base), rotary, pairing, back=True)
    w = g * gain[:, None, None, None]
    return r * (w - n * (w * n).mean(0, keepdim=True)), (g * n).sum((1, 2, 3)), (g * n).abs().sum((1, 2, 3))


def attention(q, k, v, table, buckets, scale, causal=False, lengths=None, first=None, dout=None, out_used=None, half=0.0):
    """Everything about one call.  ``out_used``: the rounded output that the kernel's backward pass was given."""
    dev = q.device
    P, H, B, J = q.shape
    G, K = k.shape[1], k.shape[3]
    rep = H // G
    q, k, v, table = q.double(), k.double(), v.double(), table.double()
    pos = torch.arange(J, device=dev) + (torch.zeros(B, 1, device=dev, dtype=torch.long) if first is None else first.long()[:, None])
    rel = torch.arange(K, device=dev) - pos[..., None]                             # [B,J,K]
    seen = torch.ones_like(rel, dtype=torch.bool)
    if lengths is not None:
        seen &= torch.arange(K, device=dev) < lengths.long().clamp(0, K)[:, None, None]
        pad = (torch.arange(K, device=dev) >= lengths.long().clamp(0, K)[:, None])
        k = k.masked_fill(pad[None, None], 0.0)
        v = v.masked_fill(pad[None, None], 0.0)
    if causal:
        seen &= rel <= 0
    lo, hi = int(rel.min()), int(rel.max())
    lookup = torch.tensor([buckets.bucket(r) for r in range(lo, hi + 1)], device=dev)
    bucket = lookup[rel - lo]
    bias = table[bucket].permute(3, 0, 1, 2)                                       # [H,B,J,K]
    kk, vv = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    s = scale * torch.einsum('phbj,phbk->hbjk', q, kk) + bias
    s = s.masked_fill(~seen | (bias <= -2.0 ** 126), -math.inf)
    m = s.amax(-1, keepdim=True)
    e = (s - torch.where(m.isinf(), torch.zeros_like(m), m)).exp()
    total = e.sum(-1, keepdim=True)
    p = e / total.masked_fill(total == 0, 1.0)
    r = {'out': torch.einsum('hbjk,phbk->phbj', p, vv), 'lse': (m + total.log())[..., 0]}
    mass = torch.einsum('hbjk,phbk->phbj', p, vv.abs())
    tiny = SMALL * K * float(v.detach().abs().max()) if v.numel() else 0.0
    bound = {'out': half * (mass + r['out'].abs()) * 1.01 + F32 * mass + tiny}
    if dout is None:
        return r, bound
    g = dout.double()
    dp = torch.einsum('phbj,phbk->hbjk', g, vv)
    d = (g * r['out']).sum(0)
    ds = p * (dp - d[..., None])
    r['dv'] = torch.einsum('hbjk,phbj->phbk', p, g).unflatten(1, (G, rep)).sum(2)
    r['dk'] = scale * torch.einsum('hbjk,phbj->phbk', ds, q).unflatten(1, (G, rep)).sum(2)
    r['dq'] = scale * torch.einsum('hbjk,phbk->phbj', ds, kk)
    r['dtable'] = torch.zeros(len(buckets), H, dtype=torch.float64, device=dev)
    r['dtable'].index_add_(0, bucket.flatten(), ds.permute(1, 2, 3, 0).reshape(-1, H))
    # distances: the score gradient is off by what D is off by (the output that it reads is rounded) and by 32-bit sums, and is
    # rounded itself on its way into dq and dk, but not into the table's sums
    used = r['out'] if out_used is None else out_used.double()
    dd = (g.abs() * (used - r['out']).abs()).sum(0)[..., None]
    size = (g.abs() * r['out'].abs()).sum(0)[..., None] + torch.einsum('phbj,phbk->hbjk', g.abs(), vv.abs())
    off = p * (dd + 2 * F32 * size)
    rounded = off + half * 1.01 * ds.abs() + SMALL
    pg = torch.einsum('hbjk,phbj->phbk', p * (half * 1.01 + F32) + SMALL, g.abs()).unflatten(1, (G, rep)).sum(2)
    end = lambda x: half * 1.01 * x.abs() + SMALL
    bound['dv'] = pg + end(r['dv'])
    bound['dk'] = scale * torch.einsum('hbjk,phbj->phbk', rounded, q.abs()).unflatten(1, (G, rep)).sum(2) + end(r['dk'])
    bound['dq'] = scale * torch.einsum('hbjk,phbk->phbj', rounded, kk.abs()) + end(r['dq'])
    bound['dtable'] = end(r['dtable'])
    bound['dtable'].index_add_(0, bucket.flatten(), off.permute(1, 2, 3, 0).reshape(-1, H))
    # How far the table's gradient may stray although its sums are 32 bits: D comes from the output, whose P numbers are rounded
    # once themselves and are sums of rounded exponentials.  A rounding is uniform in +-half |x| at most, of variance
    # (half x)^2 / 3, and they are independent: var D = sum_p dout^2 half^2 / 3 (out^2 + sum_k p^2 v^2), and D's error enters bucket
    # n with the probability of its keys.  Rows whose keys share a bucket do not take part.
    var = half ** 2 / 3 * torch.einsum('phbj,phbj->hbj', g * g, r['out'] ** 2 + torch.einsum('hbjk,phbk->phbj', p * p, vv * vv))
    stray = torch.zeros(H, dtype=torch.float64, device=dev)
    for n in range(len(buckets)):
        mass = (p * (bucket == n)).sum(-1)
        mass[(bucket == n).masked_fill(~seen, True).all(-1).expand_as(mass)] = 0.0
        stray += (mass ** 2 * var).sum((1, 2))
    r['dtable_stray'] = float(stray.sum()) ** 0.5
    return r, bound
