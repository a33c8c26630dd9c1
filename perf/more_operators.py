"""Performance cases of positions, head norms and shared prefixes in the paged 8-bit key-value cache.

What a server's decoder does around `cache.attention` once its tokens have positions and its requests begin alike:

    angles      cosines and sines of the step's positions, once a step for all layers
    share       which of the step's rows read which shared prefix, once a step for all layers
    append      norms of queries and keys for each head, their rotation, and keys and values quantised into their pages
    attention   of rows that see a shared prefix, held once in the cache, and then their own tokens

A prefix (a system prompt, a document) is a place of the batch like any request; requests that begin with it name that place and hold only
what comes after it.  Head layouts are 40 heads of 128 (the 13B-class stack: 5120 wide) and grouped heads of 64 and 128.  Lengths that vary
within a batch are spread evenly by index, so that a case has the same lengths whatever the seed.
"""
from __future__ import annotations

import math

import torch

own = False

_INPUT = {"fp16": torch.float16, "bf16": torch.bfloat16}
_HELD = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_TOP = {"int8": 127.0, "e4m3": 448.0}
_EPS = 1e-6


def _angles(tokens, farthest, rot, theta, salt=0, name=None):
    return _named(name, dict(op="angles", tokens=tokens, farthest=farthest, rot=rot, theta=theta, salt=salt))


def _share(b, prefixes, c_lo, c_hi, n_lo, n_hi, lone, salt=0, name=None):
    return _named(name, dict(op="share", b=b, prefixes=prefixes, c_lo=c_lo, c_hi=c_hi, n_lo=n_lo, n_hi=n_hi, lone=lone, salt=salt))


def _append(b, c_lo, c_hi, n_lo, n_hi, hq, hkv, d, page, held, dtype, rot, norm, interleaved, salt=0, name=None):
    return _named(name, dict(op="append", b=b, c_lo=c_lo, c_hi=c_hi, n_lo=n_lo, n_hi=n_hi, hq=hq, hkv=hkv, d=d, page=page, held=held,
                             dtype=dtype, rot=rot, norm=norm, interleaved=interleaved, salt=salt))


def _attend(prefixes, p_lo, p_hi, b, c_lo, c_hi, n_lo, n_hi, hq, hkv, d, page, held, dtype, lone=0, chunk=0, window=0, salt=0, name=None):
    return _named(name, dict(op="attention", prefixes=prefixes, p_lo=p_lo, p_hi=p_hi, b=b, c_lo=c_lo, c_hi=c_hi, n_lo=n_lo, n_hi=n_hi,
                             hq=hq, hkv=hkv, d=d, page=page, held=held, dtype=dtype, lone=lone, chunk=chunk, window=window, salt=salt))


def _named(name, case):
    return dict(case, name=name) if name else case


def listed():
    return [
        # positions of a decoding step of a few dozen requests: latency
        _angles(64, 30000, 128, 10000.0, name="angles_decode_64"),
        # positions of a server's step with prompts, far into long contexts
        _angles(36000, 1000000, 128, 500000.0, name="angles_prompts_36000"),
        # a few requests that share one prefix, a token each: latency
        _share(4, 1, 100, 2000, 1, 1, 0, name="share_decode_b4"),
        # a server's step: hundreds of requests under a dozen prefixes, some of them chunks of prompts, every ninth without a prefix
        _share(500, 12, 0, 4000, 0, 160, 9, name="share_mixed_b500"),
        # one token of one request: latency
        _append(1, 1000, 1000, 1, 1, 40, 40, 128, 16, "int8", "fp16", 128, True, False, name="append_b1_h40"),
        # a decoding step of a large batch, grouped heads of which half is rotated, pair by pair
        _append(150, 30, 6000, 1, 1, 32, 8, 128, 64, "e4m3", "bf16", 64, True, True, name="append_b150_gqa"),
        # prompts of odd lengths
        _append(3, 0, 90, 900, 2100, 40, 40, 128, 16, "int8", "fp16", 128, True, False, name="append_prompts_h40"),
        # a few requests decoding after a short prefix: latency
        _attend(1, 500, 500, 4, 5, 60, 1, 1, 40, 40, 128, 16, "int8", "fp16", name="shared_b4_h40"),
        # a batch that decodes after one system prompt
        _attend(1, 4011, 4011, 64, 1, 600, 1, 1, 40, 40, 128, 16, "int8", "fp16", name="shared_b64_h40"),
        # questions about one long document, grouped heads
        _attend(1, 31500, 31500, 96, 10, 900, 1, 1, 64, 8, 128, 64, "e4m3", "bf16", name="shared_b96_long_gqa"),
        # drafts of one to four tokens under several prefixes, every sixth request without one
        _attend(5, 700, 9000, 60, 20, 700, 1, 4, 32, 8, 64, 32, "int8", "bf16", lone=6, name="shared_drafts_p5"),
        # a request's first chunk beside others that decode
        _attend(1, 3000, 3000, 31, 10, 500, 1, 1, 32, 8, 128, 16, "int8", "fp16", chunk=512, name="shared_b31_chunk"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MOST_KEYS = 96 * 8 * 128 * 33000              # values of all requests' keys, the prefix counted for each
_MOST_SCORES = 31 * 32 * 512 * 4100            # of the batch padded to its longest request
_MOST = dict(bytes=377000000, flops=100000000000)


def _no_more(case):
    """Whether it costs no more than the largest listed ones."""
    w = work(case)
    return all(w[k] <= most for k, most in _MOST.items())


def draw(rng):
    op = rng.choice(["angles", "share", "append", "append", "append", "attention", "attention", "attention", "attention", "attention"])
    page, salt = rng.choice([16, 16, 32, 64, 128]), rng.randrange(1, 1000)
    held, dtype = rng.choice(["int8", "int8", "e4m3"]), rng.choice(["fp16", "fp16", "bf16"])
    if op == "angles":
        return _angles(_log_int(rng, 1, 36000), _log_int(rng, 10, 2000000), rng.choice([16, 32, 64, 96, 128]),
                       rng.choice([10000.0, 500000.0, 1000000.0]), salt)
    if op == "share":
        n_hi = rng.choice([1, 1, 4, _log_int(rng, 5, 160)])
        return _share(_log_int(rng, 1, 600), _log_int(rng, 1, 40), rng.choice([0, 1]), _log_int(rng, 10, 8000), rng.choice([0, 1]), n_hi,
                      rng.choice([0, 0, 3, 9]), salt)
    if op == "append":
        hkv, g, d, b = rng.choice([1, 4, 5, 8, 10, 40]), rng.choice([1, 1, 2, 4, 8]), rng.choice([64, 128, 128]), _log_int(rng, 1, 200)
        if hkv == 40:
            g = 1
        n_hi = 1 if rng.random() < 0.5 else _log_int(rng, 2, 4000)
        c_lo, c_hi, rot = rng.choice([0, 1]), _log_int(rng, 10, 6000), rng.choice([d, d, d // 2, 48])
        norm, interleaved = rng.random() < 0.7, rng.random() < 0.4
        while True:
            case = _append(b, c_lo, c_hi, max(1, n_hi // 3), n_hi, hkv * g, hkv, d, page, held, dtype, rot, norm, interleaved, salt)
            if _no_more(case):
                return case
            b, n_hi = max(1, b * 3 // 4), max(1, n_hi * 3 // 4)
    hkv, g, d = rng.choice([1, 2, 4, 5, 8, 10, 40]), rng.choice([1, 1, 2, 4, 5, 8]), rng.choice([64, 128, 128, 128])
    if hkv == 40:
        g = 1
    kind = rng.choice(["decode", "decode", "decode", "draft", "chunk"])
    prefixes = rng.choice([1, 1, 1, 2, 7])
    b = max(prefixes, _log_int(rng, 2, 120) if kind != "chunk" else _log_int(rng, 2, 31))
    p_hi, c_hi = _log_int(rng, 50, 31500), _log_int(rng, 5, 900)
    n_hi = 1 if kind != "draft" else rng.choice([2, 3, 4, 5, 8])
    chunk = _log_int(rng, 17, 512) if kind == "chunk" else 0
    window = _log_int(rng, 16, 5000) if rng.random() < 0.12 else 0
    p_part, c_part, lone = rng.choice([1, 1, 3]), rng.choice([2, 50]), rng.choice([0, 0, 3, 6])
    while True:
        case = _attend(prefixes, p_hi // p_part, p_hi, b, c_hi // c_part, c_hi, 1, n_hi, hkv * g, hkv, d, page, held, dtype, lone, chunk, window, salt)
        if (b * hkv * d * (p_hi + c_hi + chunk) <= _MOST_KEYS and b * hkv * g * max(chunk, n_hi) * (p_hi + c_hi + chunk) <= _MOST_SCORES and
                _no_more(case)):
            return case
        p_hi, c_hi, chunk = max(20, p_hi * 3 // 4), max(5, c_hi * 7 // 8), chunk * 7 // 8


# ---- lengths --------------------------------------------------------------------------------------------------------
def _spread(n, lo, hi, salt):
    """n whole numbers spread evenly over lo .. hi, in no order."""
    return [lo + int(math.fmod((i + 1) * 0.6180339887498949 + salt * 0.7548776662466927, 1.0) * (hi - lo + 1)) for i in range(n)]


def _lengths(case):
    """(tokens held before the step, new tokens) of every request."""
    b, salt = case["b"], case["salt"]
    held, new = _spread(b, case["c_lo"], case["c_hi"], salt), _spread(b, case["n_lo"], case["n_hi"], salt + 7)
    if case.get("chunk"):
        new[b // 2] = case["chunk"]
    return held, new


def _places(case):
    """The batch: prefixes first, without new tokens, then the requests: (tokens after the step, new tokens, place of the prefix or -1)."""
    held, new = _lengths(case)
    np, lone = case["prefixes"], case["lone"]
    before = _spread(np, case.get("p_lo", case["c_lo"]), case.get("p_hi", case["c_hi"]), case["salt"] + 3)
    of = [-1 if lone and i % lone == lone - 1 else i % np for i in range(len(held))]
    return before + [c + n for c, n in zip(held, new)], [0] * np + new, [-1] * np + of


def _pages(n, page):
    return -(-n // page)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _generator(seed, salt):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + salt)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _sums(v):
    out = [0]
    for n in v:
        out.append(out[-1] + n)
    return out


def _table(gen, counts, pages, width):
    """Each place's pages, drawn without repetition; -1 where it has none."""
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    counts = _ints(counts)
    at = torch.arange(width, device="cuda", dtype=torch.int32)[None, :]
    start = (counts.cumsum(0, dtype=torch.int32) - counts)[:, None]
    return torch.where(at < counts[:, None], order[(start + at).clamp(max=pages - 1).long()], -1).to(torch.int32)


def _projected(gen, shape, dtype, spread=None):
    """Normal values with a few channels larger than the rest, as projections give them; `spread`: a factor for each of the leading sizes."""
    x = torch.randn(shape, device="cuda", generator=gen)
    channel = torch.exp(0.4 * torch.randn(shape[-1], device="cuda", generator=gen))
    x = x * channel / channel.square().mean().sqrt()
    return (x if spread is None else x * spread).to(dtype)


def _filled(gen, pages, heads, page, d, held):
    """One of the cache's two arrays and its scales (pages, heads): values of about 1, pages of different sizes."""
    dtype = _HELD[held]
    out = torch.empty((pages, heads, page, d), dtype=dtype, device="cuda")
    scales = torch.empty((pages, heads), dtype=torch.float32, device="cuda")
    step = max(1, (1 << 27) // (heads * page * d))
    for i in range(0, pages, step):
        n = min(step, pages - i)
        x = _projected(gen, (n, heads, page, d), torch.float32, torch.exp(0.3 * torch.randn((n, heads, 1, 1), device="cuda", generator=gen)))
        scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax(dim=(2, 3), keepdim=True) / _TOP[held])))
        q = (x / scale).clamp(-_TOP[held], _TOP[held])
        out[i:i + n] = (q.round() if held == "int8" else q).to(dtype)
        scales[i:i + n] = scale[:, :, 0, 0]
    return out, scales


def _freqs(rot, theta):
    return (theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().cuda()


def _table_of_angles(positions, freqs):
    a = positions.double()[:, None] * freqs.double()
    return torch.stack([a.cos(), a.sin()], dim=-1).float()


def _shared_rows(after, new, of):
    """What a program holds of a step's sharing, from its lengths: (prefix_of, starts, rows, positions)."""
    cu = _sums(new)
    lists, positions = [[] for _ in after], []
    for b, (total, n, p) in enumerate(zip(after, new, of)):
        for i in range(n):
            positions.append(total - n + i + (after[p] if p >= 0 else 0))
            if p >= 0:
                lists[p].append(cu[b] + i)
    rows = [t for rows in lists for t in rows]
    return [_ints(of), _ints(_sums(len(r) for r in lists)), _ints(rows + [-1] * (cu[-1] - len(rows))), _ints(positions)]


def prepare(case, seed):
    gen = _generator(seed, 1 + case["salt"])
    if case["op"] == "angles":
        positions = torch.randint(0, case["farthest"] + 1, (case["tokens"],), device="cuda", generator=gen, dtype=torch.int32)
        if case["tokens"] > 8:
            positions[-3:] = -1                                 # padding
        return dict(case=case, positions=positions, freqs=_freqs(case["rot"], case["theta"]))
    if case["op"] == "share":
        after, new, of = _places(case)
        # the batch's order is another for each seed: prefixes may stand anywhere in it
        order = torch.randperm(len(after), device="cuda", generator=gen).tolist()
        at = {old: i for i, old in enumerate(order)}
        after, new, of = [after[i] for i in order], [new[i] for i in order], [at[of[i]] if of[i] >= 0 else -1 for i in order]
        tokens = sum(new)
        return dict(case=case, prefix_of=_ints(of), seq_lens=_ints(after), cu_lens=_ints(_sums(new)), max_tokens=max(8, -(-tokens // 8) * 8))
    page, d, hkv, hq = case["page"], case["d"], case["hkv"], case["hq"]
    if case["op"] == "append":
        held, new = _lengths(case)
        after = [c + n for c, n in zip(held, new)]
        begin = [c // page for c in held]                       # the first page that the step touches
        touched = [_pages(a, page) - f for a, f in zip(after, begin)]
        pages = sum(touched) + 5
        order = torch.randperm(pages, device="cuda", generator=gen)[:sum(touched)]
        first = _sums(touched)
        rel = [(c % page, c % page + n) for c, n in zip(held, new)]
        place = torch.cat([f * page + torch.arange(lo, hi) for f, (lo, hi) in zip(first, rel)]).cuda()
        live = torch.cat([f * page + torch.arange(0, hi) for f, (_, hi) in zip(first, rel)]).cuda()
        positions = torch.cat([torch.arange(c, a) for c, a in zip(held, after)]).cuda()
        k_cache, ks = _filled(gen, pages, hkv, page, d, case["held"])
        v_cache, vs = _filled(gen, pages, hkv, page, d, case["held"])
        spread = torch.exp(0.3 * torch.randn((place.numel(), 1, 1), device="cuda", generator=gen))
        dtype = _INPUT[case["dtype"]]
        wide = _projected(gen, (place.numel(), hq + 2 * hkv, d), dtype, spread)
        weights = [(1 + 0.2 * torch.randn(d, device="cuda", generator=gen)).to(dtype) if case["norm"] else None for _ in range(2)]
        return dict(case=case, k_cache=k_cache, v_cache=v_cache, scales=torch.stack([ks, vs], dim=-1).contiguous(),
                    q=wide[:, :hq], k=wide[:, hq:hq + hkv], v=wide[:, hq + hkv:],       # columns of one projection's output
                    slots=(order[place // page] * page + place % page).to(torch.int32),
                    live=(order[live // page] * page + live % page).to(torch.int32), pages=order,
                    angles=_table_of_angles(positions, _freqs(case["rot"], 10000.0)), q_weight=weights[0], k_weight=weights[1])
    after, new, of = _places(case)
    counts = [_pages(n, page) for n in after]
    pages = sum(counts) + 3
    k_cache, ks = _filled(gen, pages, hkv, page, d, case["held"])
    v_cache, vs = _filled(gen, pages, hkv, page, d, case["held"])
    return dict(case=case, k_cache=k_cache, v_cache=v_cache, scales=torch.stack([ks, vs], dim=-1).contiguous(),
                table=_table(gen, counts, pages, max(counts)), seq_lens=_ints(after), cu_lens=_ints(_sums(new)), max_len=max(new),
                shared=_shared_rows(after, new, of), q=1.3 * _projected(gen, (sum(new), hq, d), _INPUT[case["dtype"]]))


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _plain_share(s):
    seq, cu, of = s["seq_lens"].long(), s["cu_lens"].long(), s["prefix_of"].long()
    b, dev = seq.numel(), seq.device
    place = torch.arange(b, device=dev)
    there = (of >= 0) & (of < b) & (of != place) & (seq > 0)
    there &= seq[of.clamp(0, b - 1)] > 0
    of = torch.where(there, of, -1)
    t = torch.arange(s["max_tokens"], device=dev)
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    real = r < b
    r = r.clamp(max=b - 1)
    pos = seq[r] - (cu[r + 1] - cu[r]) + t - cu[r]
    real &= pos >= 0
    p = torch.where(real, of[r], -1)
    positions = torch.where(real, pos + torch.where(p >= 0, seq[p.clamp(min=0)], 0), -1)
    order = torch.sort(torch.where(p >= 0, p, b), stable=True).indices
    starts = torch.searchsorted(torch.where(p >= 0, p, b)[order], torch.arange(b + 1, device=dev))
    rows = torch.where(t < starts[b], order, -1)
    return dict(prefix_of=of.int(), starts=starts.int(), rows=rows.int(), positions=positions.int())


def _raw(cache):
    """Indexable bytes of a cache."""
    return cache.view(torch.int8)


def _scale_for(amax, held):
    """The least power of two s with amax <= most * s; 0 where there is nothing to hold."""
    _, e = torch.frexp(amax)
    s = torch.ldexp(torch.ones_like(amax), e - (7 if held == "int8" else 9))
    s = torch.where(amax > _TOP[held] * s, 2 * s, s)
    return torch.where(amax > 0, s, 0)


def _to_held(x, held):
    x = x.clamp(-_TOP[held], _TOP[held])
    return (x.round() if held == "int8" else x).to(_HELD[held]).view(torch.int8)


def _plain_write_one(cache, scales, x, slots, page, held, pages):
    heads, size = cache.shape[1], cache.shape[0]
    slots = slots.long()
    at, off = slots // page, slots % page
    x = x.float()
    amax = x.abs().amax(dim=-1)
    most = torch.zeros((size, heads), device=x.device).scatter_reduce_(0, at[:, None].expand(-1, heads), amax, "amax")[pages]
    first = torch.full((size,), page, device=x.device).scatter_reduce_(0, at, off, "amin")[pages]
    old = torch.where((first == 0)[:, None], 0, scales[pages])
    s = torch.maximum(old, _scale_for(most, held))
    scales[pages] = s
    ratio = torch.where(s > 0, old / s.clamp(min=1e-38), 1)
    rows = _raw(cache)[pages].view(cache.dtype).float() * ratio[:, :, None, None]
    kept = torch.arange(page, device=x.device)[None, :] < first[:, None]
    keep = kept[:, None, :, None] & (ratio < 1)[:, :, None, None]
    _raw(cache)[pages] = torch.where(keep, _to_held(rows, held), _raw(cache)[pages])
    st = scales[at][:, :, None]
    _raw(cache)[at, :, off] = _to_held(x / torch.where(st > 0, st, 1), held)


def _plain_read_one(cache, scales, slots, page, dtype):
    slots = slots.long()
    at, off = slots // page, slots % page
    return (_raw(cache)[at, :, off].view(cache.dtype).float() * scales[at][:, :, None]).to(dtype)


def _plain_turned(x, weight, angles, interleaved):
    """Norm of each head, rotation of its first 2 * angles.shape[1] values, one rounding."""
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(dim=-1, keepdim=True) + _EPS) * weight.float()
    n = angles.shape[1]
    c, s = angles[:, None, :, 0], angles[:, None, :, 1]
    a, b = (y[..., 0:2 * n:2], y[..., 1:2 * n:2]) if interleaved else (y[..., :n], y[..., n:2 * n])
    turned = torch.stack([a * c - b * s, b * c + a * s], dim=-1 if interleaved else -2).flatten(-2)
    return torch.cat([turned, y[..., 2 * n:]], dim=-1).to(x.dtype)


def _plain_append(s):
    case = s["case"]
    q = _plain_turned(s["q"], s["q_weight"], s["angles"], case["interleaved"])
    k = _plain_turned(s["k"], s["k_weight"], s["angles"], case["interleaved"])
    _plain_write_one(s["k_cache"], s["scales"][..., 0], k, s["slots"], case["page"], case["held"], s["pages"])
    _plain_write_one(s["v_cache"], s["scales"][..., 1], s["v"], s["slots"], case["page"], case["held"], s["pages"])
    k, v = (_plain_read_one(c, s["scales"][..., i], s["live"], case["page"], q.dtype) for i, c in enumerate((s["k_cache"], s["v_cache"])))
    return dict(q=q, k=k, v=v)


def _plain_attention(s):
    """Each request's keys and values are its prefix's and then its own."""
    case, q = s["case"], s["q"]
    page, d, hkv, g, np = case["page"], case["d"], case["hkv"], case["hq"] // case["hkv"], case["prefixes"]
    dev, n = q.device, s["max_len"]
    cu, seq, of = s["cu_lens"].long()[np:], s["seq_lens"].long(), s["shared"][0].long()[np:]
    total = torch.where(of >= 0, seq[of.clamp(min=0)], 0)                         # of the prefix
    seq, b = seq[np:], of.numel()
    before, mine = _pages(case["p_hi"], page), _pages(case["c_hi"] + n, page)
    width = s["table"].shape[1]
    table = torch.cat([s["table"][of.clamp(min=0)][:, :before], s["table"][np:, :min(mine, width)]], dim=1).long()
    at, before = table.clamp(min=0), min(before, width) * page
    keys = at.shape[1] * page

    def tokens(cache, scales):                                # (b, hkv, keys, d)
        x = _raw(cache)[at].view(cache.dtype).float() * scales[at][:, :, :, None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(b, hkv, keys, d)

    k, v = tokens(s["k_cache"], s["scales"][..., 0]), tokens(s["v_cache"], s["scales"][..., 1])
    row = torch.arange(n, device=dev)[None, :]
    lens = cu[1:] - cu[:-1]
    rows = (cu[:-1, None] + row).clamp(max=q.shape[0] - 1)
    pad = q[rows].float().view(b, n, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, n * g, d)
    scores = torch.matmul(pad, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    pos = (total + seq - lens)[:, None] + row                                     # (b, n), the prefix counted
    j = torch.arange(keys, device=dev)[None, :]
    key = torch.where(j < before, j, total[:, None] + j - before)                 # (b, keys)
    real = torch.where(j < before, j < total[:, None], j - before < seq[:, None])
    sees = (key[:, None, :] <= pos[:, :, None]) & real[:, None, :] & (row < lens[:, None])[:, :, None]
    if case["window"]:
        sees &= key[:, None, :] > pos[:, :, None] - case["window"]
    sees = sees[:, None, :, None, :].expand(b, 1, n, g, keys).reshape(b, 1, n * g, keys)
    scores = torch.where(sees, scores, -math.inf)
    most = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(most), most, 0))
    sums = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(sums > 0, sums, 1)
    o = o.view(b, hkv, n, g, d).permute(0, 2, 1, 3, 4).reshape(b, n, hkv * g, d)
    t = torch.arange(q.shape[0], device=dev)
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return o[r, t - cu[r]].to(q.dtype)


def run(state):
    s, case = state, state["case"]
    if own:
        from int4matmul_kernels_b200 import cache
    if case["op"] == "angles":
        return dict(angles=cache.angles(s["positions"], s["freqs"]) if own else _table_of_angles(s["positions"].clamp(min=0), s["freqs"]))
    if case["op"] == "share":
        if not own:
            return _plain_share(s)
        return cache.share(s["prefix_of"], s["seq_lens"], s["cu_lens"], s["max_tokens"])._asdict()
    if case["op"] == "append":
        if not own:
            return _plain_append(s)
        q = cache.append(s["k_cache"], s["v_cache"], s["scales"], s["q"], s["k"], s["v"], s["slots"], s["angles"],
                         q_weight=s["q_weight"], k_weight=s["k_weight"], eps=_EPS, interleaved=case["interleaved"])
        k, v = cache.read(s["k_cache"], s["v_cache"], s["scales"], s["live"], q.dtype)
        return dict(q=q, k=k, v=v)
    if not own:
        return dict(out=_plain_attention(s))
    return dict(out=cache.attention(s["q"], s["k_cache"], s["v_cache"], s["scales"], s["table"], s["seq_lens"], s["cu_lens"], s["max_len"],
                                    window=case["window"], shared=cache.Shared(*s["shared"])))


def work(case):
    if case["op"] == "angles":
        return dict(bytes=4.0 * case["tokens"] * (1 + case["rot"]) + 2 * case["rot"], flops=0.0)
    if case["op"] == "share":
        places = case["b"] + case["prefixes"]
        return dict(bytes=4.0 * (5 * places + 2 * sum(_places(case)[1])), flops=0.0)
    page, d, hkv, hq = case["page"], case["d"], case["hkv"], case["hq"]
    if case["op"] == "append":
        held, new = _lengths(case)
        live = sum(c % page + n for c, n in zip(held, new))
        touched = sum(_pages(c % page + n, page) for c, n in zip(held, new))
        tokens = sum(new)
        return dict(bytes=float(tokens * (hq * d * 4 + hkv * d * 6 + 4 * case["rot"] + 4) + live * (hkv * d * 6 + 4) + touched * hkv * 16), flops=0.0)
    after, new, of = _places(case)
    window, size, pairs = case["window"], 0, 0
    reach = {}                                               # of a place's tokens: the first that any row sees
    for b, (total, n, p) in enumerate(zip(after, new, of)):
        if n == 0:
            continue
        shared = after[p] if p >= 0 else 0
        low = max(0, shared + total - n + 1 - window) if window else 0
        if p >= 0:
            reach[p] = min(reach.get(p, shared), low)
        reach[b] = max(0, low - shared)
        seen = [shared + total - n + 1 + i for i in range(n)]
        pairs += sum(min(r, window) if window else r for r in seen)
    for b, first in reach.items():
        if first < after[b]:
            size += (after[b] - first) * hkv * 2 * d + (_pages(after[b], page) - first // page) * (8 * hkv + 4)
    return dict(bytes=float(size + 2 * 2 * sum(new) * hq * d), flops=4.0 * d * hq * pairs)


# ---- 64 bits ----------------------------------------------------------------------------------------------------------
def _exact_share(case, s):
    of, seq, cu = s["prefix_of"].tolist(), s["seq_lens"].tolist(), s["cu_lens"].tolist()
    n = len(of)
    of = [p if 0 <= p < n and p != b and seq[p] > 0 and seq[b] > 0 else -1 for b, p in enumerate(of)]
    readers, positions = {}, [-1] * s["max_tokens"]
    for b, p in enumerate(of):
        for t in range(cu[b], cu[b + 1]):
            pos = seq[b] - cu[b + 1] + t
            if pos < 0:
                continue
            positions[t] = pos + (seq[p] if p >= 0 else 0)
            if p >= 0:
                readers.setdefault(p, []).append(t)
    starts, rows = [], []
    for p in range(n):
        starts.append(len(rows))
        rows += readers.get(p, [])
    starts.append(len(rows))
    return dict(prefix_of=_ints(of), starts=_ints(starts), rows=_ints(rows + [-1] * (s["max_tokens"] - len(rows))), positions=_ints(positions))


def _exact_round(x, held):
    """The nearest value of the type to x, ties to even; x within its range."""
    if held == "int8":
        return torch.round(x)
    grid = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / grid) * grid


def _exact_write_one(cache, scales, x, s, case):
    page, most, pages = case["page"], _TOP[case["held"]], s["pages"]
    where = torch.full((cache.shape[0],), -1, dtype=torch.int64, device="cuda")
    where[pages] = torch.arange(pages.numel(), device="cuda")
    slots = s["slots"].long()
    at, off = where[slots // page], slots % page
    heads, d = cache.shape[1], cache.shape[3]
    fresh = torch.zeros((pages.numel(), page), dtype=torch.bool, device="cuda")
    fresh[at, off] = True
    dense = torch.zeros((pages.numel(), page, heads, d), dtype=torch.float64, device="cuda")
    dense[at, off] = x
    amax = dense.abs().amax(dim=(1, 3))
    e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / most))
    e = torch.where(torch.exp2(e) * most < amax, e + 1, e)
    e = torch.where(torch.exp2(e - 1) * most >= amax, e - 1, e)
    need = torch.where(amax > 0, torch.exp2(e), 0)
    began = fresh[:, 0][:, None]
    old = torch.where(began, 0, scales[pages].double())
    scale = torch.maximum(need, old)[:, None, :, None]
    stored = cache.view(torch.int8)[pages].view(cache.dtype).double().transpose(1, 2)
    stored = stored * torch.where(scale > 0, old[:, None, :, None] / scale, 1)
    before = torch.where(scale > old[:, None, :, None], _exact_round(stored, case["held"]), stored)
    codes = torch.where(fresh[:, :, None, None], _exact_round(dense / torch.where(scale > 0, scale, 1), case["held"]), before)
    values = codes.clamp(-most, most) * scale
    live = s["live"].long()
    return values[where[live // page], live % page]


def _exact_turned(x, weight, angles, interleaved):
    """The rotation as a product of complex numbers."""
    y = x.double()
    if weight is not None:
        y = y / (y.pow(2).sum(dim=-1, keepdim=True) / y.shape[-1] + _EPS).sqrt() * weight.double()
    n = angles.shape[1]
    turn = torch.view_as_complex(angles.double())[:, None, :]
    head = y[..., :2 * n]
    pairs = head.unflatten(-1, (n, 2)) if interleaved else head.unflatten(-1, (2, n)).transpose(-1, -2)
    pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    out = y.clone()
    out[..., :2 * n] = pairs.flatten(-2) if interleaved else pairs.transpose(-1, -2).flatten(-2)
    return out


def _exact_append(case, s):
    q = _exact_turned(s["q"], s["q_weight"], s["angles"], case["interleaved"])
    k = _exact_turned(s["k"], s["k_weight"], s["angles"], case["interleaved"])
    k = k.to(s["k"].dtype).double()                           # keys are rounded to the activations' type, then held
    return dict(q=q, k=_exact_write_one(s["k_cache"], s["scales"][..., 0], k, s, case),
                v=_exact_write_one(s["v_cache"], s["scales"][..., 1], s["v"].double(), s, case))


def _exact_attention(case, s):
    hkv, g, page, d = case["hkv"], case["hq"] // case["hkv"], case["page"], case["d"]
    after, new, of = _places(case)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")

    def held(b, cache, which):                                # (hkv, tokens, d)
        pages = s["table"][b, :_pages(after[b], page)].long()
        x = cache.view(torch.int8)[pages].view(cache.dtype).double() * s["scales"][pages, :, which].double()[:, :, None, None]
        return x.transpose(0, 1).flatten(1, 2)[:, :after[b]]

    both = ((s["k_cache"], 0), (s["v_cache"], 1))
    prefixes = {p: [held(p, *c) for c in both] for p in sorted(set(of)) if p >= 0}
    lo = 0
    for b, (total, n, p) in enumerate(zip(after, new, of)):
        if n == 0:
            continue
        k, v = (held(b, *c) for c in both)
        shared = 0
        if p >= 0:
            shared = after[p]
            k, v = torch.cat([prefixes[p][0], k], dim=1), torch.cat([prefixes[p][1], v], dim=1)
        q = s["q"][lo:lo + n].double().view(n, hkv, g, d).permute(1, 2, 0, 3).reshape(hkv, g * n, d)
        pos = torch.arange(shared + total - n, shared + total, device="cuda").repeat(g)
        key = torch.arange(shared + total, device="cuda")
        hidden = key[None, :] > pos[:, None]
        if case["window"]:
            hidden |= key[None, :] <= pos[:, None] - case["window"]
        w = torch.softmax((q @ k.transpose(1, 2) / d ** 0.5).masked_fill(hidden, -math.inf), dim=-1)
        out[lo:lo + n] = (w @ v).view(hkv, g, n, d).permute(2, 0, 1, 3).reshape(n, hkv * g, d)
        lo += n
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "angles":
        a = s["positions"].clamp(min=0).double()[:, None] * s["freqs"].double()
        turn = torch.polar(torch.ones_like(a), a)
        return dict(angles=torch.view_as_real(turn))
    if case["op"] == "share":
        return _exact_share(case, s)
    if case["op"] == "append":
        return _exact_append(case, s)
    return dict(out=_exact_attention(case, s))
