"""Performance cases of the paged 8-bit key-value cache: its tables, its writer and the attention that reads it.

What a program that serves a decoder has the GPU do between its quantized linears: build the step's block tables and slot
maps from the requests' lengths (`plan`), quantise the step's keys and values into the cache's pages (`write`, and `read`, which
gives tokens back as the values that they stand for), and attend over the pages (`attention`) with one query per request while
decoding, a few when a draft is checked, hundreds or thousands for prompts, and mixtures of those.

Head layouts are 40 heads of 128 (the 13B-class stack: 5120 wide) and grouped heads of 64 and 128.  Lengths that vary within a
batch are spread evenly by index, so that a case has the same lengths whatever the seed.
"""
from __future__ import annotations

import math

import torch

own = False

_INPUT = {"fp16": torch.float16, "bf16": torch.bfloat16}
_HELD = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_MOST = {"int8": 127.0, "e4m3": 448.0}


def _plan(b, c_lo, c_hi, n_lo, n_hi, page, ending=0, salt=0, name=None):
    return _named(name, dict(op="plan", b=b, c_lo=c_lo, c_hi=c_hi, n_lo=n_lo, n_hi=n_hi, page=page, ending=ending, salt=salt))


def _write(b, c_lo, c_hi, n_lo, n_hi, heads, d, page, held, dtype, salt=0, name=None):
    return _named(name, dict(op="write", b=b, c_lo=c_lo, c_hi=c_hi, n_lo=n_lo, n_hi=n_hi, heads=heads, d=d, page=page, held=held,
                             dtype=dtype, salt=salt))


def _attend(b, c_lo, c_hi, n_lo, n_hi, hq, hkv, d, page, held, dtype, chunk=0, idle=0, window=0, salt=0, name=None):
    return _named(name, dict(op="attention", b=b, c_lo=c_lo, c_hi=c_hi, n_lo=n_lo, n_hi=n_hi, hq=hq, hkv=hkv, d=d, page=page,
                             held=held, dtype=dtype, chunk=chunk, idle=idle, window=window, salt=salt))


def _named(name, case):
    return dict(case, name=name) if name else case


def listed():
    return [
        # tables of a decoding step of a few requests: latency
        _plan(4, 100, 2000, 1, 1, 16, name="plan_decode_b4"),
        # a server's step: hundreds of requests, some of them prompts, every ninth one ending
        _plan(500, 0, 4000, 0, 160, 64, ending=9, name="plan_mixed_b500"),
        # one token of one request into the cache: latency
        _write(1, 1000, 1000, 1, 1, 40, 128, 16, "int8", "fp16", name="write_b1_h40"),
        # a decoding step of a large batch, grouped heads
        _write(150, 30, 6000, 1, 1, 8, 128, 64, "e4m3", "bf16", name="write_b150_h8"),
        # prompts of odd lengths
        _write(3, 0, 90, 900, 2100, 40, 128, 16, "int8", "fp16", name="write_prompts_h40"),
        # one request decoding: latency
        _attend(1, 1011, 1011, 1, 1, 40, 40, 128, 16, "int8", "fp16", name="decode_b1_h40"),
        # a batch of requests of all lengths decoding, some of its places idle: the cache is what is read
        _attend(64, 1, 4000, 1, 1, 40, 40, 128, 16, "int8", "fp16", idle=13, name="decode_b64_h40"),
        # long contexts, grouped heads
        _attend(12, 20000, 34000, 1, 1, 64, 8, 128, 64, "e4m3", "bf16", name="decode_b12_long_gqa"),
        # drafts of one to four tokens checked at once, a sliding window
        _attend(33, 300, 9000, 1, 4, 32, 8, 64, 32, "int8", "bf16", window=4000, name="draft_b33_window"),
        # a prompt of the 13B-class stack
        _attend(1, 0, 0, 2048, 2048, 40, 40, 128, 16, "int8", "fp16", name="prompt_2048_h40"),
        # chunks of long prompts, grouped heads
        _attend(2, 7000, 8300, 1000, 1024, 64, 8, 128, 64, "e4m3", "bf16", name="chunks_8k_gqa"),
        # requests decoding beside a chunk of a prompt
        _attend(17, 500, 4000, 1, 1, 32, 8, 128, 16, "int8", "fp16", chunk=256, name="mixed_b17_chunk"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "write", "write", "attention", "attention", "attention", "attention"])
    page, salt = rng.choice([16, 16, 32, 64, 128]), rng.randrange(1, 1000)
    held, dtype = rng.choice(["int8", "int8", "e4m3"]), rng.choice(["fp16", "fp16", "bf16"])
    if op == "plan":
        b, n_hi = _log_int(rng, 1, 600), rng.choice([1, 1, 4, _log_int(rng, 5, 160)])
        return _plan(b, 0, _log_int(rng, 10, 8000), rng.choice([0, 1]), n_hi, page, rng.choice([0, 0, 5, 11]), salt)
    if op == "write":
        heads, d, b = rng.choice([1, 4, 5, 8, 10, 40]), rng.choice([64, 128, 128]), _log_int(rng, 1, 200)
        n_hi = 1 if rng.random() < 0.5 else _log_int(rng, 2, 4000)
        n_hi = max(1, min(n_hi, 4000 * 40 * 128 // (b * heads * d)))
        return _write(b, rng.choice([0, 1]), _log_int(rng, 10, 6000), max(1, n_hi // 3), n_hi, heads, d, page, held, dtype, salt)
    hkv, g, d = rng.choice([1, 2, 4, 5, 8, 10, 40]), rng.choice([1, 1, 2, 4, 5, 8]), rng.choice([64, 128, 128, 128])
    if hkv == 40:
        g = 1
    kind = rng.choice(["decode", "decode", "draft", "prompt", "mixed"])
    window = _log_int(rng, 16, 5000) if rng.random() < 0.2 else 0
    if kind in ("decode", "draft"):
        b = _log_int(rng, 1, 100)
        c_hi = min(_log_int(rng, 20, 34000), 64 * 2000 * 40 * 128 // (b * hkv * d))
        n_hi = 1 if kind == "decode" else rng.choice([2, 3, 4, 5, 8])
        return _attend(b, c_hi // rng.choice([1, 2, 50]), c_hi, 1, n_hi, hkv * g, hkv, d, page, held, dtype, 0,
                       rng.choice([0, 0, 7]) if kind == "decode" else 0, window, salt)
    if kind == "prompt":
        b = rng.choice([1, 1, 2, 3])
        n_hi, c_hi = _log_int(rng, 17, 2048), rng.choice([0, 0, _log_int(rng, 16, 8000)])
        while b * hkv * g * n_hi * (n_hi + c_hi) > 2 * 64 * 1000 * 9000:
            n_hi, c_hi = max(1, n_hi * 3 // 4), c_hi * 3 // 4
        return _attend(b, c_hi // 2, c_hi, max(1, n_hi // 2), n_hi, hkv * g, hkv, d, page, held, dtype, 0, 0, window, salt)
    b, chunk, c_hi = _log_int(rng, 2, 24), _log_int(rng, 17, 300), _log_int(rng, 50, 4000)
    while b * hkv * g * chunk * (c_hi + chunk) > 2 * 64 * 1000 * 9000:
        chunk, c_hi = max(2, chunk * 3 // 4), max(2, c_hi * 3 // 4)
    return _attend(b, c_hi // 8, c_hi, 1, 1, hkv * g, hkv, d, page, held, dtype, chunk, 0, window, salt)


# ---- lengths --------------------------------------------------------------------------------------------------------
def _spread(n, lo, hi, salt):
    """n whole numbers spread evenly over lo .. hi, in no order."""
    return [lo + int(math.fmod((i + 1) * 0.6180339887498949 + salt * 0.7548776662466927, 1.0) * (hi - lo + 1)) for i in range(n)]


def _lengths(case):
    """(tokens held before the step, new tokens) of every request; -1 new tokens: the request ends, 0 held and 1 new: an idle place."""
    b, salt = case["b"], case["salt"]
    held, new = _spread(b, case["c_lo"], case["c_hi"], salt), _spread(b, case["n_lo"], case["n_hi"], salt + 7)
    if case.get("chunk"):
        new[b // 2] = case["chunk"]
    if case.get("ending"):
        new = [-1 if i % case["ending"] == case["ending"] - 1 else n for i, n in enumerate(new)]
    return held, new


def _seen(case):
    """Lengths after the step; an idle place has none."""
    held, new = _lengths(case)
    idle = case.get("idle", 0)
    return [0 if idle and i % idle == idle - 1 else c + max(n, 0) for i, (c, n) in enumerate(zip(held, new))]


def _pages(n, page):
    return -(-n // page)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _generator(seed, salt):
    return torch.Generator(device="cuda").manual_seed(seed * 1000003 + salt)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _table(gen, counts, pages, width):
    """Each request's pages, drawn without repetition; -1 where it has none."""
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
        scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax(dim=(2, 3), keepdim=True) / _MOST[held])))
        q = (x / scale).clamp(-_MOST[held], _MOST[held])
        out[i:i + n] = (q.round() if held == "int8" else q).to(dtype)
        scales[i:i + n] = scale[:, :, 0, 0]
    return out, scales


def prepare(case, seed):
    gen = _generator(seed, 1 + case["salt"])
    held, new = _lengths(case)
    page = case["page"]
    if case["op"] == "plan":
        after = [0 if n < 0 else c + n for c, n in zip(held, new)]
        width = max(1, _pages(max(c + max(n, 0) for c, n in zip(held, new)), page))
        used = [_pages(c, page) for c in held]
        pages = sum(used) + sum(_pages(a, page) for a in after) + 8
        order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
        counts, at = _ints(used), torch.arange(width, device="cuda", dtype=torch.int32)[None, :]
        start = (counts.cumsum(0, dtype=torch.int32) - counts)[:, None]
        table = torch.where(at < counts[:, None], order[(start + at).clamp(max=pages - 1).long()], -1).to(torch.int32)
        free = torch.zeros(pages, dtype=torch.int32, device="cuda")
        free[:pages - sum(used)] = order[sum(used):]
        tokens = sum(max(n, 0) for n in new)
        return dict(case=case, seq_lens=_ints(held), new_lens=_ints(new), table=table, free_pages=free,
                    free_count=_ints([pages - sum(used)]), max_tokens=max(8, -(-tokens // 8) * 8))
    if case["op"] == "write":
        heads, d = case["heads"], case["d"]
        after = [c + n for c, n in zip(held, new)]
        begin = [c // page for c in held]                       # the first page that the step touches
        touched = [_pages(a, page) - f for a, f in zip(after, begin)]
        pages = sum(touched) + 5
        order = torch.randperm(pages, device="cuda", generator=gen)[:sum(touched)]
        first = [sum(touched[:i]) for i in range(len(touched))]
        rel = [(c % page, c % page + n) for c, n in zip(held, new)]
        place = torch.cat([f * page + torch.arange(lo, hi) for f, (lo, hi) in zip(first, rel)]).cuda()
        live = torch.cat([f * page + torch.arange(0, hi) for f, (_, hi) in zip(first, rel)]).cuda()
        k_cache, ks = _filled(gen, pages, heads, page, d, case["held"])
        v_cache, vs = _filled(gen, pages, heads, page, d, case["held"])
        spread = torch.exp(0.3 * torch.randn((place.numel(), heads, 1), device="cuda", generator=gen))
        wide = _projected(gen, (place.numel(), 2 * heads, d), _INPUT[case["dtype"]], spread.repeat(1, 2, 1))
        return dict(case=case, k_cache=k_cache, v_cache=v_cache, scales=torch.stack([ks, vs], dim=-1).contiguous(),
                    k=wide[:, :heads], v=wide[:, heads:],       # columns of one projection's output
                    slots=(order[place // page] * page + place % page).to(torch.int32),
                    live=(order[live // page] * page + live % page).to(torch.int32), pages=order)
    seen = _seen(case)
    counts = [_pages(n, page) for n in seen]
    pages = sum(counts) + 3
    k_cache, ks = _filled(gen, pages, case["hkv"], page, case["d"], case["held"])
    v_cache, vs = _filled(gen, pages, case["hkv"], page, case["d"], case["held"])
    tokens = sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    single = max(new) == 1 and min(new) == 1
    return dict(case=case, k_cache=k_cache, v_cache=v_cache, scales=torch.stack([ks, vs], dim=-1).contiguous(),
                table=_table(gen, counts, pages, max(1, max(counts))), seq_lens=_ints(seen), cu_lens=None if single else _ints(cu),
                max_len=max(new), q=1.3 * _projected(gen, (tokens, case["hq"], case["d"]), _INPUT[case["dtype"]]))


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _plain_plan(s):
    seq, new, table, page = s["seq_lens"].long(), s["new_lens"].long(), s["table"], s["case"]["page"]
    b, width = table.shape
    ends = new < 0
    add = torch.where(ends, 0, new)
    after = torch.where(ends, 0, seq + add)
    held = (seq + page - 1) // page
    given_up = torch.where(ends, held.clamp(max=width), 0)
    need = torch.where(ends, 0, ((after + page - 1) // page).clamp(max=width) - held.clamp(max=width))
    wanted = torch.where(ends, 0, (after + page - 1) // page - held)
    # the pages of the requests that end go on top of the free ones, in request order
    free, count = s["free_pages"], s["free_count"].long()
    column = torch.arange(width, device=table.device)[None, :]
    place = count + (given_up.cumsum(0) - given_up)[:, None] + column
    of_ended = column < given_up[:, None]
    spare = torch.cat([free, free.new_zeros(1)])
    spare[torch.where(of_ended, place, free.numel()).reshape(-1)] = table.reshape(-1)
    free.copy_(spare[:-1])
    # new pages come off the top, in request order
    top = count + given_up.sum()
    j = column - held[:, None]
    taken = top - 1 - ((need.cumsum(0) - need)[:, None] + j)
    is_new = (j >= 0) & (j < need[:, None])
    got = torch.where(taken >= 0, free[taken.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where(is_new, got, table))
    cu = torch.cat([add.new_zeros(1), add.cumsum(0)])
    t = torch.arange(s["max_tokens"], device=table.device)
    r = torch.searchsorted(cu[1:], t, right=True)
    real = r < b
    r = r.clamp(max=b - 1)
    pos = seq[r] + t - cu[r]
    at = table[r, (pos // page).clamp(0, width - 1)].long()
    slot = torch.where(real & (pos // page < width) & (at >= 0), at * page + pos % page, -1)
    left = (top - need.sum()).clamp(min=0)
    missing = wanted.sum() - (top - left)
    return dict(seq_lens=after.int(), cu_lens=cu.int(), slots=slot.int(), positions=torch.where(real, pos, -1).int(),
                requests=torch.where(real, r, -1).int(), free_count=left.int(), missing=missing.reshape(1).int(), table=table, free_pages=free)


def _raw(cache):
    """Indexable bytes of a cache."""
    return cache.view(torch.int8)


def _scale_for(amax, held):
    """The least power of two s with amax <= most * s; 0 where there is nothing to hold."""
    _, e = torch.frexp(amax)
    s = torch.ldexp(torch.ones_like(amax), e - (7 if held == "int8" else 9))
    s = torch.where(amax > _MOST[held] * s, 2 * s, s)
    return torch.where(amax > 0, s, 0)


def _to_held(x, held):
    x = x.clamp(-_MOST[held], _MOST[held])
    return (x.round() if held == "int8" else x).to(_HELD[held]).view(torch.int8)


def _plain_write_one(cache, scales, x, slots, page, held, pages):
    heads, size = cache.shape[1], cache.shape[0]
    slots = slots.long()
    at, off = slots // page, slots % page
    x = x.float()
    finite = torch.isfinite(x)
    amax = torch.where(finite, x.abs(), 0).amax(dim=-1)
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
    value = torch.where(torch.isnan(x), 0, x / torch.where(st > 0, st, 1))
    _raw(cache)[at, :, off] = _to_held(value, held)


def _plain_read_one(cache, scales, slots, page, dtype):
    slots = slots.long()
    at, off = slots // page, slots % page
    return (_raw(cache)[at, :, off].view(cache.dtype).float() * scales[at][:, :, None]).to(dtype)


def _plain_attention(s):
    case, q, table = s["case"], s["q"], s["table"].long()
    b, width = table.shape
    page, d, hkv, g = case["page"], case["d"], case["hkv"], case["hq"] // case["hkv"]
    dev, n = q.device, s["max_len"]
    cu = torch.arange(b + 1, device=dev) if s["cu_lens"] is None else s["cu_lens"].long()
    lens, seq = cu[1:] - cu[:-1], s["seq_lens"].long()
    valid = table >= 0
    at = table.clamp(min=0)

    def tokens(cache, scales):                                # (b, hkv, width * page, d)
        x = _raw(cache)[at].view(cache.dtype).float() * scales[at][:, :, :, None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(b, hkv, width * page, d)

    k, v = tokens(s["k_cache"], s["scales"][..., 0]), tokens(s["v_cache"], s["scales"][..., 1])
    row = torch.arange(n, device=dev)[None, :]
    rows = (cu[:-1, None] + row).clamp(max=q.shape[0] - 1)
    pad = q[rows].float().view(b, n, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, n * g, d)
    scores = torch.matmul(pad, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    pos = (seq - lens)[:, None] + row                                             # (b, n)
    key = torch.arange(width * page, device=dev)
    sees = (key <= pos[:, :, None]) & (key < seq[:, None, None]) & (row < lens[:, None])[:, :, None]
    if case["window"]:
        sees &= key > pos[:, :, None] - case["window"]
    sees &= valid.repeat_interleave(page, dim=1)[:, None, :]
    sees = sees[:, None, :, None, :].expand(b, 1, n, g, width * page).reshape(b, 1, n * g, width * page)
    scores = torch.where(sees, scores, -math.inf)
    most = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(most), most, 0))
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1)
    o = o.view(b, hkv, n, g, d).permute(0, 2, 1, 3, 4).reshape(b, n, hkv * g, d)
    t = torch.arange(q.shape[0], device=dev)
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return o[r, t - cu[r]].to(q.dtype)


def run(state):
    s, case = state, state["case"]
    if own:
        from int4matmul_kernels_b200 import cache
    if case["op"] == "plan":
        if not own:
            return _plain_plan(s)
        p = cache.plan(s["seq_lens"], s["new_lens"], s["table"], s["free_pages"], s["free_count"], case["page"], s["max_tokens"])
        return dict(seq_lens=p.seq_lens, cu_lens=p.cu_lens, slots=p.slots, positions=p.positions, requests=p.requests,
                    free_count=p.free_count, missing=p.missing, table=s["table"], free_pages=s["free_pages"])
    if case["op"] == "write":
        dtype = _INPUT[case["dtype"]]
        if own:
            cache.write(s["k_cache"], s["v_cache"], s["scales"], s["k"], s["v"], s["slots"])
            k, v = cache.read(s["k_cache"], s["v_cache"], s["scales"], s["live"], dtype)
        else:
            for i, (c, x) in enumerate(((s["k_cache"], s["k"]), (s["v_cache"], s["v"]))):
                _plain_write_one(c, s["scales"][..., i], x, s["slots"], case["page"], case["held"], s["pages"])
            k, v = (_plain_read_one(c, s["scales"][..., i], s["live"], case["page"], dtype) for i, c in enumerate((s["k_cache"], s["v_cache"])))
        return dict(k=k, v=v, scales=s["scales"])
    if not own:
        return dict(out=_plain_attention(s))
    return dict(out=cache.attention(s["q"], s["k_cache"], s["v_cache"], s["scales"], s["table"], s["seq_lens"], s["cu_lens"], s["max_len"],
                                    window=case["window"]))


def work(case):
    held, new = _lengths(case)
    page = case["page"]
    if case["op"] == "plan":
        tokens = sum(max(n, 0) for n in new)
        pages = sum(_pages(c + n, page) - _pages(c, page) if n >= 0 else _pages(c, page) for c, n in zip(held, new))
        return dict(bytes=4.0 * (4 * case["b"] + 2 * pages + 3 * tokens), flops=0.0)
    if case["op"] == "write":
        size = case["heads"] * case["d"] * 2
        live = sum(c % page + n for c, n in zip(held, new))
        touched = sum(_pages(c % page + n, page) for c, n in zip(held, new))
        return dict(bytes=float(sum(new) * size * 3 + live * size * 3 + touched * case["heads"] * 16 + 4 * (sum(new) + live)), flops=0.0)
    size, pairs, window = 0, 0, case["window"]
    for n, total in zip(new, _seen(case)):
        first = max(0, total - n + 1 - window) if window else 0            # of the keys that any row sees
        size += (total - first) * case["hkv"] * 2 * case["d"] + (_pages(total, page) - first // page) * (8 * case["hkv"] + 4)
        reach = [max(0, total - n + 1 + i) for i in range(n)]
        pairs += sum(min(r, window) if window else r for r in reach)
    return dict(bytes=float(size + 2 * 2 * sum(new) * case["hq"] * case["d"]), flops=4.0 * case["d"] * case["hq"] * pairs)


# ---- 64 bits ----------------------------------------------------------------------------------------------------------
def _exact_plan(case, s):
    seq, new, page = s["seq_lens"].tolist(), s["new_lens"].tolist(), case["page"]
    table, count = s["table"].tolist(), s["free_count"].item()
    stack = s["free_pages"].tolist()
    size = len(stack)
    stack = stack[:count]
    below = s["free_pages"].tolist()
    for c, n, row in zip(seq, new, table):
        if n < 0:
            stack += row[:_pages(c, page)]
    below[:len(stack)] = stack
    missing, cu, after, slots, positions, requests = 0, [0], [], [], [], []
    for b, (c, n, row) in enumerate(zip(seq, new, table)):
        total = 0 if n < 0 else c + n
        for j in range(_pages(c, page), _pages(total, page)):
            row[j] = stack.pop() if stack else -1
            missing += row[j] < 0
        for p in range(c, total):
            slots.append(row[p // page] * page + p % page if row[p // page] >= 0 else -1)
            positions.append(p)
            requests.append(b)
        after.append(total)
        cu.append(len(slots))
    pad = [-1] * (s["max_tokens"] - len(slots))
    return dict(seq_lens=_ints(after), cu_lens=_ints(cu), slots=_ints(slots + pad), positions=_ints(positions + pad), requests=_ints(requests + pad),
                free_count=_ints([len(stack)]), missing=_ints([missing]), table=_ints(table), free_pages=_ints(below[:size]))


def _exact_round(x, held):
    """The nearest value of the type to x, ties to even; x within its range."""
    if held == "int8":
        return torch.round(x)
    grid = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / grid) * grid


def _exact_write_one(cache, scales, x, s, case):
    page, most, pages = case["page"], _MOST[case["held"]], s["pages"]
    where = torch.full((cache.shape[0],), -1, dtype=torch.int64, device="cuda")
    where[pages] = torch.arange(pages.numel(), device="cuda")
    slots = s["slots"].long()
    at, off = where[slots // page], slots % page
    heads, d = cache.shape[1], cache.shape[3]
    fresh = torch.zeros((pages.numel(), page), dtype=torch.bool, device="cuda")
    fresh[at, off] = True
    dense = torch.zeros((pages.numel(), page, heads, d), dtype=torch.float64, device="cuda")
    dense[at, off] = x.double()
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
    everywhere = scales.double().clone()
    everywhere[pages] = scale[:, 0, :, 0]
    return values[where[live // page], live % page], everywhere


def _exact_attention(case, s):
    g, page, d = case["hq"] // case["hkv"], case["page"], case["d"]
    seq = s["seq_lens"].tolist()
    cu = list(range(len(seq) + 1)) if s["cu_lens"] is None else s["cu_lens"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, total in enumerate(seq):
        lo, hi = cu[b], cu[b + 1]
        if total == 0 or lo == hi:
            continue
        pages = s["table"][b, :_pages(total, page)].long()
        scale = s["scales"][pages].double()
        k = (s["k_cache"].view(torch.int8)[pages].view(s["k_cache"].dtype).double() * scale[:, :, 0, None, None]).transpose(0, 1).flatten(1, 2)[:, :total]
        v = (s["v_cache"].view(torch.int8)[pages].view(s["v_cache"].dtype).double() * scale[:, :, 1, None, None]).transpose(0, 1).flatten(1, 2)[:, :total]
        pos = torch.arange(total - (hi - lo), total, device="cuda")
        key = torch.arange(total, device="cuda")
        hidden = key[None, :] > pos[:, None]
        if case["window"]:
            hidden |= key[None, :] <= pos[:, None] - case["window"]
        for h in range(case["hkv"]):
            for i in range(h * g, (h + 1) * g):
                w = (s["q"][lo:hi, i].double() @ k[h].T / d ** 0.5).masked_fill(hidden, -math.inf)
                out[lo:hi, i] = torch.softmax(w, dim=-1) @ v[h]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return _exact_plan(case, s)
    if case["op"] == "write":
        k, ks = _exact_write_one(s["k_cache"], s["scales"][..., 0], s["k"], s, case)
        v, vs = _exact_write_one(s["v_cache"], s["scales"][..., 1], s["v"], s, case)
        return dict(k=k, v=v, scales=torch.stack([ks, vs], dim=-1))
    return dict(out=_exact_attention(case, s))
