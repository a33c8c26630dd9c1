"""The paged 8-bit cache in 64 bits and plain Python: what the tests of its kernels compare with."""
import math

import torch

MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def plan(seq, new, table, stack, page, width, max_tokens):
    """Lists in, dict of lists out; `table` (lists) and `stack` are changed as the operator changes its arrays."""
    seq, table, stack = list(seq), [list(r) for r in table], list(stack)
    for b, n in enumerate(new):
        if n < 0:
            stack += table[b][:min(-(-seq[b] // page), width)]
    pushed = list(stack)
    out = dict(lens=[], cu=[0], slots=[], positions=[], requests=[], missing=0)
    for b, n in enumerate(new):
        total = 0 if n < 0 else seq[b] + n
        for j in range(-(-seq[b] // page), -(-total // page)):
            got = stack.pop() if j < width and stack else -1
            out["missing"] += got < 0
            if j < width:
                table[b][j] = got
        for pos in range(seq[b], total):
            id = table[b][pos // page] if pos // page < width else -1
            out["slots"].append(id * page + pos % page if id >= 0 else -1)
            out["positions"].append(pos)
            out["requests"].append(b)
        out["lens"].append(total)
        out["cu"].append(len(out["slots"]))
    for n in ("slots", "positions", "requests"):
        out[n] = (out[n] + [-1] * max_tokens)[:max_tokens]
    return dict(out, table=table, free=len(stack), pushed=pushed)


def round_to(x, dtype):
    """The nearest value of an 8-bit type, ties to even; x in its range."""
    if dtype == torch.int8:
        return torch.round(x)
    grid = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / grid) * grid


def scale_for(a, dtype):
    """The least power of two s (at least 2^-100) with a <= most * s; 0 for a = 0."""
    if a == 0:
        return 0.0
    e = math.frexp(a)[1] - 12
    while MOST[dtype] * 2.0 ** e < a:
        e += 1
    return 2.0 ** max(e, -100)


def write_one(held, scales, x, slots, page, dtype):
    """held (pages, heads, page, dim) and scales (pages, heads) in 64 bits, changed in place; x (tokens, heads, dim) in 64 bits."""
    runs, slots = {}, [int(s) for s in slots]
    for t, s in enumerate(slots[:x.shape[0]]):
        if 0 <= s < held.shape[0] * page:
            runs.setdefault(s // page, []).append((s % page, t))
    for id, places in runs.items():
        first = places[0][0]
        for h in range(held.shape[1]):
            rows = x[[t for _, t in places], h]
            finite = rows[torch.isfinite(rows)].abs()
            old = float(scales[id, h]) if first else 0.0
            s = max(old, scale_for(float(finite.max()) if finite.numel() else 0.0, dtype))
            if s > old and old > 0:
                held[id, h, :first] = round_to(held[id, h, :first] * (old / s), dtype)
            q = torch.nan_to_num(rows, nan=0.0, posinf=math.inf, neginf=-math.inf) / (s if s > 0 else 1.0)
            held[id, h, [p for p, _ in places]] = round_to(q.clamp(-MOST[dtype], MOST[dtype]), dtype)
            scales[id, h] = s


def values(cache, scales):
    """(pages, heads, page, dim) in 64 bits"""
    return cache.view(torch.int8).clone().view(cache.dtype).double() * scales.double()[:, :, None, None]


def attention(q, k, v, table, seq_lens, cu_lens, scale, window=0):
    """q (tokens, q_heads, dim); k, v (pages, heads, page, dim) in 64 bits.  Returns the output and, for the bound on a kernel's error, the same sum with
    |v| in the place of v, the largest sum of |q_d k_d| * scale over the tokens that a row sees, and max w * max |v| * (their number)."""
    page, heads = k.shape[2], k.shape[1]
    group = q.shape[1] // heads
    seq, table = seq_lens.tolist(), table.long()
    cu = list(range(len(seq) + 1)) if cu_lens is None else cu_lens.tolist()
    out, size = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    reach, tail = (torch.zeros(q.shape[:2] + (1,), dtype=torch.float64, device=q.device) for _ in range(2))
    for b, total in enumerate(seq):
        lo, hi = cu[b], min(cu[b + 1], q.shape[0])
        total_in = min(total, table.shape[1] * page)
        if hi <= lo or total_in <= 0:
            continue
        ids = table[b, :-(-total_in // page)]
        ok = (ids >= 0) & (ids < k.shape[0])
        pick = lambda c: c[ids.clamp(0, k.shape[0] - 1)].transpose(0, 1).flatten(1, 2)[:, :total_in].repeat_interleave(group, 0)  # noqa: E731
        kk, vv = pick(k), pick(v)
        pos = torch.arange(total - (cu[b + 1] - lo), total - (cu[b + 1] - lo) + (hi - lo), device=q.device)
        key = torch.arange(total_in, device=q.device)
        sees = (key[None] <= pos[:, None]) & ok.repeat_interleave(page)[None, :total_in]
        if window:
            sees &= key[None] > pos[:, None] - window
        qq = q[lo:hi].double().transpose(0, 1)
        s = (qq @ kk.transpose(1, 2) * scale).masked_fill(~sees, -math.inf)
        m = s.amax(-1, keepdim=True)
        w = torch.exp(s - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
        hidden = torch.where(sees.any(0)[:, None], vv, torch.zeros_like(vv))     # (what nobody sees may hold anything)
        out[lo:hi] = (w @ hidden).transpose(0, 1)
        size[lo:hi] = (w @ hidden.abs()).transpose(0, 1)
        reach[lo:hi] = ((qq.abs() @ kk.abs().transpose(1, 2)) * scale * sees).amax(-1, keepdim=True).transpose(0, 1)
        tail[lo:hi] = (w.amax(-1, keepdim=True) * hidden.abs().amax() * sees.sum(-1)[None, :, None]).transpose(0, 1)
    return out, size, reach, tail


def attention_bound(out, size, reach, tail, dtype):
    """What a kernel's output may be off by.  Rounding of the output: half a unit in the last place (2^-11 and 2^-8 of the value; 2^-25 below
    fp16's normal range).  Weights rounded to fp16 in the range of the largest one: 2^-11 of each, or 2^-25 of the largest where they are
    smaller than fp16's normal numbers.  Scores of fp32 sums over dim / 16 tensor-core steps whose additions may truncate, for the token and
    for the maximum: 2 * (8 + 1) * 2^-23 * reach, times log2(e) rounded once more, below 2^-17 * reach; fp32 exponentials and sums: 2^-17."""
    rounding = out.abs() * (2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8) + 2.0 ** -25
    return rounding + (2.0 ** -11 + 2.0 ** -17 * (1 + reach)) * size * 1.01 + 2.0 ** -25 * tail
