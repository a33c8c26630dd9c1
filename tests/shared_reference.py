"""Positions, head norms and shared prefixes in 64 bits and plain Python: what the tests of their kernels compare with."""
import math

import torch


def share(of, seq, cu, max_tokens):
    """Lists in, dict of lists out."""
    n = len(of)
    of = [p if 0 <= p < n and p != b and seq[p] > 0 and seq[b] > 0 else -1 for b, p in enumerate(of)]
    readers, positions = [[] for _ in of], [-1] * max_tokens
    for b, p in enumerate(of):
        for t in range(cu[b], min(cu[b + 1], max_tokens)):
            pos = seq[b] - cu[b + 1] + t
            if pos >= 0:
                positions[t] = pos + (seq[p] if p >= 0 else 0)
                if p >= 0:
                    readers[p].append(t)
    starts, rows = [0], []
    for r in readers:
        rows += r
        starts.append(len(rows))
    return dict(prefix_of=of, starts=starts, rows=rows + [-1] * (max_tokens - len(rows)), positions=positions)


def turned(x, weight, angles, eps, interleaved):
    """Norm of each head and rotation in 64 bits, and what the rotation's two products come to."""
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    out, size = y.clone(), y.abs()
    if angles is not None:
        n = angles.shape[1]
        c, s = angles[:x.shape[0], None, :, 0].double(), angles[:x.shape[0], None, :, 1].double()
        first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
        a, b = y[..., first], y[..., second]
        out[..., first], out[..., second] = a * c - b * s, b * c + a * s
        size[..., first], size[..., second] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return out, size


def turned_bound(out, size, dtype):
    """The rounding of the output: half a step (2^-11 or 2^-8 of it, 2^-25 below fp16's normal range).  fp32 before that: a mean of squares of up to 13
    additions, whose root halves their error, a reciprocal root of 2 units, two products (together below 2^-20 of a value), and two
    products and a sum of those: below 2^-19 of the products' sizes."""
    return out.abs() * (2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8) + 2.0 ** -25 + size * 2.0 ** -19


def attention(q, k, v, table, seq_lens, cu_lens, prefix_of, scale, window=0):
    """q (tokens, q_heads, dim); k, v (pages, heads, page, dim) in 64 bits; prefix_of: a list, -1: none.  The four results of
    cache_reference.attention: each request's keys and values are its prefix's and then its own."""
    page, heads = k.shape[2], k.shape[1]
    group, capacity = q.shape[1] // heads, table.shape[1] * k.shape[2]
    seq, cu, ids = seq_lens.tolist(), cu_lens.tolist(), table.long()
    out, size = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    reach, tail = (torch.zeros(q.shape[:2] + (1,), dtype=torch.float64, device=q.device) for _ in range(2))

    def held(b, n):
        i = ids[b, :-(-n // page)]
        ok = (i >= 0) & (i < k.shape[0])
        pick = lambda c: c[i.clamp(0, k.shape[0] - 1)].transpose(0, 1).flatten(1, 2)[:, :n].repeat_interleave(group, 0)  # noqa: E731
        return pick(k), pick(v), ok.repeat_interleave(page)[:n]

    for b, total in enumerate(seq):
        lo, hi = cu[b], min(cu[b + 1], q.shape[0])
        own = min(total, capacity)
        if hi <= lo or own <= 0:
            continue
        kk, vv, ok = held(b, own)
        key, before, p = torch.arange(own, device=q.device), 0, prefix_of[b]
        if p >= 0:
            before, there = seq[p], min(seq[p], capacity)
            pk, pv, pok = held(p, there)
            kk, vv, ok = torch.cat([pk, kk], 1), torch.cat([pv, vv], 1), torch.cat([pok, ok])
            key = torch.cat([torch.arange(there, device=q.device), before + key])
        pos = torch.arange(lo, hi, device=q.device) + (total - cu[b + 1])
        sees = (key[None] <= before + pos[:, None]) & ok[None] & (pos >= 0)[:, None]
        if window:
            sees &= key[None] > before + pos[:, None] - window
        qq = q[lo:hi].double().transpose(0, 1)
        s = (qq @ kk.transpose(1, 2) * scale).masked_fill(~sees, -math.inf)
        m = s.amax(-1, keepdim=True)
        w = torch.exp(s - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
        hidden = torch.where(sees.any(0)[:, None], vv, torch.zeros_like(vv))     # (what nobody sees may hold anything)
        out[lo:hi] = (w @ hidden).transpose(0, 1)
        size[lo:hi] = (w @ hidden.abs()).transpose(0, 1)
        reach[lo:hi] = ((qq.abs() @ kk.abs().transpose(1, 2)) * abs(scale) * sees).amax(-1, keepdim=True).transpose(0, 1)
        tail[lo:hi] = (w.amax(-1, keepdim=True) * hidden.abs().amax() * sees.sum(-1)[None, :, None]).transpose(0, 1)
    return out, size, reach, tail
