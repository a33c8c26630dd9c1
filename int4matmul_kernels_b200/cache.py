"""The paged key-value cache in 8 bits, and attention over it: what a decoder needs between its quantized linears.

    plan       the step's block tables and slot maps, on the GPU, from the requests' lengths
    share      which of the step's rows read which shared prefix, and their positions
    angles     cosines and sines of positions
    write      quantise the step's keys and values into their pages
    append     norm the step's queries and keys, rotate them, and write keys and values, in one launch
    read       tokens of the cache as the values that they stand for
    attention  softmax attention of the step's queries over the cached tokens, those of a shared prefix among them
    PagedCache one layer's arrays;  PageTable  the requests' lengths, block table and free pages

The cache is (pages, heads, page_size, head_dim) int8 or float8_e4m3fn for keys and values, with fp32 scales (pages, heads, 2): a
byte q stands for q * scale.  page_size is 16, 32, 64 or 128 and head_dim 64 or 128.  Activations are fp16 or bf16.  Everything runs on
torch's current stream and nothing waits for the GPU, but for the first `attention` of a stream if it is made inside a graph capture: that
waits until its scratch has been cleared.  There are no backward passes: what these calls return carries no gradient.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional

import torch

from . import capi, ops

_HELD = {torch.int8: capi.CACHE_INT8, torch.float8_e4m3fn: capi.CACHE_E4M3}
_INPUT = {torch.float16: capi.TYPE_FP16, torch.bfloat16: capi.TYPE_BF16}


class Plan(NamedTuple):
    """One step's tables; int32 on the GPU."""
    seq_lens: torch.Tensor      # (requests) tokens after the step
    cu_lens: torch.Tensor       # (requests + 1) packed place of each request's first new token
    slots: torch.Tensor         # (max_tokens) where each packed token goes; -1: padding, or no page could be had
    positions: torch.Tensor     # (max_tokens) its position in its request; -1: padding
    requests: torch.Tensor      # (max_tokens) its request; -1: padding
    free_count: torch.Tensor    # (1) pages left on the stack
    missing: torch.Tensor       # (1) pages that the step asked for and did not get


class Shared(NamedTuple):
    """A step's shared prefixes; int32 on the GPU."""
    prefix_of: torch.Tensor     # (requests) the place of the batch whose tokens come before the request's own; -1: none
    starts: torch.Tensor        # (requests + 1) where the list of each place's readers begins in `rows`
    rows: torch.Tensor          # (max_tokens) packed tokens that read a prefix, by place and then in order; -1 behind the last
    positions: torch.Tensor     # (max_tokens) position of each packed token, its prefix counted; -1: padding


def _workspace(device: torch.device, stream: torch.cuda.Stream) -> torch.Tensor:
    key = (device.index if device.index is not None else torch.cuda.current_device(), stream.cuda_stream)
    ws = ops._cache_workspaces.get(key)
    if ws is None:
        ws = ops.zeroed_scratch(capi.load().i4mm_cache_attention_workspace_bytes(), device)
        ops._cache_workspaces[key] = ws
    return ws


def _check(status: int, what: str) -> None:
    if status != capi.OK:
        raise ops.Int4MatmulError(status, what)


def _int32(t: torch.Tensor, name: str, device: torch.device, shape: Optional[tuple] = None) -> None:
    if not t.is_cuda or t.device != device:
        raise ValueError(f"{name} must be a CUDA tensor on {device}")
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}")
    if not (t.is_contiguous() or (t.dim() == 2 and t.stride(1) == 1)):
        raise ValueError(f"{name} must be contiguous")


def _table(t: torch.Tensor, device: torch.device, requests: Optional[int] = None) -> tuple[int, int]:
    """(width, row stride) of a block table"""
    _int32(t, "block_table", device)
    if t.dim() != 2 or (requests is not None and t.shape[0] != requests):
        raise ValueError("block_table must be (requests, width)")
    return t.shape[1], t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _rows(t: torch.Tensor, name: str, device: torch.device, heads: Optional[int], dim: int) -> int:
    if not t.is_cuda or t.device != device:
        raise ValueError(f"{name} must be a CUDA tensor on {device}")
    if t.dtype not in _INPUT:
        raise TypeError(f"{name} must be float16 or bfloat16")
    if t.dim() != 3 or t.shape[2] != dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be (tokens, {'heads' if heads is None else heads}, {dim})")
    if t.stride(2) != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    return _INPUT[t.dtype]


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor, scales: torch.Tensor) -> capi.Cache:
    if not k_cache.is_cuda:
        raise ValueError("k_cache must be a CUDA tensor")
    dev = k_cache.device
    for t, name in ((v_cache, "v_cache"), (scales, "scales")):
        if not t.is_cuda or t.device != dev:
            raise ValueError(f"{name} must be a CUDA tensor on {dev}")
    if k_cache.dtype not in _HELD or v_cache.dtype != k_cache.dtype:
        raise TypeError("k_cache and v_cache must both be int8 or float8_e4m3fn")
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError("k_cache and v_cache must both be (pages, heads, page_size, head_dim)")
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise ValueError("k_cache and v_cache must be contiguous in their last dimension")
    pages, heads, page_size, dim = k_cache.shape
    if scales.dtype != torch.float32:
        raise TypeError("scales must be float32")
    if tuple(scales.shape) != (pages, heads, 2) or not scales.is_contiguous():
        raise ValueError("scales must be contiguous (pages, heads, 2)")
    return capi.Cache(k_cache.data_ptr(), v_cache.data_ptr(), scales.data_ptr(), pages, heads, page_size, dim,
                      k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
                      v_cache.stride(0), v_cache.stride(1), v_cache.stride(2), _HELD[k_cache.dtype])


def plan(seq_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
         free_count: torch.Tensor, page_size: int, max_tokens: int) -> Plan:
    """The tables of a step in which request b, holding seq_lens[b] tokens, adds new_lens[b] (negative: it ends and gives its pages back).

    `block_table` (requests, width) gets the pages that the step begins, in place; `free_pages` is a stack with its first free_count[0]
    entries free: the pages of requests that end are pushed, then new ones popped, in request order.  seq_lens, new_lens and
    free_count are left alone: the next step takes the Plan's.  Where no page is left the table's entry and the slots become -1, so that
    nothing is written or seen there, and Plan.missing counts it: drop such a Plan and make a smaller step from the same lengths and count
    (a request that goes on without its pages must not end: it would give -1 back as pages)."""
    mod = ops.native()
    if mod:
        out = mod._try_cache_plan(seq_lens, new_lens, block_table, free_pages, free_count, page_size, max_tokens)
        if not isinstance(out, int):
            return Plan._make(out)
        _check(max(out, 0), "cache plan")
    if not seq_lens.is_cuda:
        raise ValueError("seq_lens must be a CUDA tensor")
    dev, n = seq_lens.device, seq_lens.shape[0] if seq_lens.dim() == 1 else -1
    _int32(seq_lens, "seq_lens", dev, (n,))
    _int32(new_lens, "new_lens", dev, (n,))
    width, row_stride = _table(block_table, dev, n)
    _int32(free_pages, "free_pages", dev)
    _int32(free_count, "free_count", dev, (1,))
    if free_pages.dim() != 1:
        raise ValueError("free_pages must be (capacity)")
    max_tokens = int(max_tokens)
    if max_tokens < 0:
        raise ValueError("max_tokens must not be negative")
    sizes = (n, n + 1, max_tokens, max_tokens, max_tokens, 1, 1)
    with torch.cuda.device(dev):
        flat = torch.empty(sum(sizes), dtype=torch.int32, device=dev)
        out = Plan(*flat.split(sizes))
        status = capi.load().i4mm_cache_plan(
            n, seq_lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(), width, row_stride,
            free_pages.data_ptr(), free_pages.shape[0], free_count.data_ptr(), int(page_size), max_tokens,
            out.seq_lens.data_ptr(), out.cu_lens.data_ptr(), out.slots.data_ptr(), out.positions.data_ptr(), out.requests.data_ptr(),
            out.free_count.data_ptr(), torch.cuda.current_stream(dev).cuda_stream)
    _check(status, "cache plan")
    return out


def share(prefix_of: torch.Tensor, seq_lens: torch.Tensor, cu_lens: torch.Tensor, max_tokens: int) -> Shared:
    """Which rows of a step read which shared prefix, for `attention`, and the rows' positions, for `angles`; once a step, for all layers.

    A prefix (a system prompt, a document) is a place of the batch like any request: its tokens are written and its pages given back as theirs
    are.  prefix_of[b] is the place whose tokens come before those of request b, which holds only what comes after; a negative number, no place
    of the batch, the request itself or a place without tokens: none.  One level: a prefix's own prefix is not looked at.  `seq_lens`
    and `cu_lens` are the Plan's, after the step; `max_tokens` as for `plan`.  A place must go on holding its tokens while requests name it, and where
    keys are rotated it must not grow any more: positions behind it count its tokens, and keys that were rotated for fewer of them stay as they are."""
    mod = ops.native()
    if mod:
        out = mod._try_cache_share(prefix_of, seq_lens, cu_lens, max_tokens)
        if not isinstance(out, int):
            return Shared._make(out)
        _check(max(out, 0), "cache share")
    if not seq_lens.is_cuda:
        raise ValueError("seq_lens must be a CUDA tensor")
    dev, n = seq_lens.device, seq_lens.shape[0] if seq_lens.dim() == 1 else -1
    _int32(seq_lens, "seq_lens", dev, (n,))
    _int32(prefix_of, "prefix_of", dev, (n,))
    _int32(cu_lens, "cu_lens", dev, (n + 1,))
    max_tokens = int(max_tokens)
    if max_tokens < 0:
        raise ValueError("max_tokens must not be negative")
    sizes = (n, n + 1, max_tokens, max_tokens)
    with torch.cuda.device(dev):
        out = Shared(*torch.empty(sum(sizes), dtype=torch.int32, device=dev).split(sizes))
        status = capi.load().i4mm_cache_share(n, prefix_of.data_ptr(), seq_lens.data_ptr(), cu_lens.data_ptr(), max_tokens, *(t.data_ptr() for t in out),
                                              torch.cuda.current_stream(dev).cuda_stream)
    _check(status, "cache share")
    return out


def angles(positions: torch.Tensor, freqs: torch.Tensor) -> torch.Tensor:
    """(tokens, pairs, 2) fp32: cos and sin of positions[t] * freqs[i]; (1, 0) for negative positions.  The angle is off by at most 9.4e-8 (its
    rounding to fp32 once whole turns are taken off) and 2^-51 of itself (fp64): 1.5e-7 for 2^27 radians, 1.1e-6 for 2^31.

    positions (tokens) int32, freqs (pairs) fp32, their number a multiple of 8 up to 128.  Once a step, for all layers."""
    mod = ops.native()
    if mod:
        out = mod._try_cache_angles(positions, freqs)
        if not isinstance(out, int):
            return out
        _check(max(out, 0), "cache angles")
    if not positions.is_cuda:
        raise ValueError("positions must be a CUDA tensor")
    dev = positions.device
    _int32(positions, "positions", dev)
    if positions.dim() != 1:
        raise ValueError("positions must be (tokens)")
    if freqs.device != dev:
        raise ValueError(f"freqs must be a CUDA tensor on {dev}")
    if freqs.dtype != torch.float32:
        raise TypeError("freqs must be float32")
    if freqs.dim() != 1 or not freqs.is_contiguous():
        raise ValueError("freqs must be contiguous (pairs)")
    with torch.cuda.device(dev):
        out = torch.empty((positions.shape[0], freqs.shape[0], 2), dtype=torch.float32, device=dev)
        status = capi.load().i4mm_cache_angles(out.data_ptr(), positions.data_ptr(), freqs.data_ptr(), positions.shape[0], freqs.shape[0],
                                               torch.cuda.current_stream(dev).cuda_stream)
    _check(status, "cache angles")
    return out


def write(k_cache: torch.Tensor, v_cache: torch.Tensor, scales: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantises k and v (tokens, heads, head_dim) into the cache, in place, at `slots` (tokens or more; those below 0 are skipped).

    The tokens of a page that one call writes are neighbours with ascending slots, as `plan` lays them out.  A page's scale is
    the least power of two that holds its values; where new tokens raise it, the bytes that the page holds already are requantised.  A page
    whose first place is written begins anew."""
    mod = ops.native()
    if mod:
        status = mod._try_cache_write(k_cache, v_cache, scales, k, v, slots)
        if status == capi.OK:
            return
        _check(max(status, 0), "cache write")
    c = _cache(k_cache, v_cache, scales)
    dev = k_cache.device
    kind = _rows(k, "k", dev, c.heads, c.head_dim)
    if _rows(v, "v", dev, c.heads, c.head_dim) != kind or v.shape != k.shape:
        raise ValueError("k and v must have one type and shape")
    _int32(slots, "slots", dev)
    if slots.dim() != 1 or slots.shape[0] < k.shape[0]:
        raise ValueError("slots must be (tokens)")
    with torch.cuda.device(dev):
        status = capi.load().i4mm_cache_write(
            ctypes.byref(c), k.data_ptr(), v.data_ptr(), kind, k.shape[0], k.stride(0), k.stride(1), v.stride(0), v.stride(1),
            slots.data_ptr(), torch.cuda.current_stream(dev).cuda_stream)
    _check(status, "cache write")


def append(k_cache: torch.Tensor, v_cache: torch.Tensor, scales: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
           slots: torch.Tensor, angles: Optional[torch.Tensor] = None, *, q_weight: Optional[torch.Tensor] = None,
           k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False) -> torch.Tensor:
    """`write` of a model whose queries and keys are normed and rotated: returns the queries (tokens, q_heads, head_dim), and quantises the keys so
    treated, and the values as they are, into the cache.

    Each head of q (k) is divided by the root of its mean square (+ eps) and multiplied by q_weight (k_weight), (head_dim) in q's type; None: no
    norm.  Then its first 2 * pairs values are rotated by `angles` (tokens or more, pairs, 2), as `angles` makes them: value i with value i + pairs,
    or, `interleaved`, value 2 i with value 2 i + 1; None: no rotation.  All in fp32, rounded once to q's type, so that the cache
    holds what a `write` of such keys would put there.  q, k and v may be columns of one projection's output; padding (slots below 0) is not written.
    There is no backward pass: the queries returned carry no gradient."""
    mod = ops.native()
    if mod:
        out = mod._try_cache_append(k_cache, v_cache, scales, q, k, v, slots, angles, q_weight, k_weight, eps, interleaved)
        if not isinstance(out, int):
            return out
        _check(max(out, 0), "cache append")
    c = _cache(k_cache, v_cache, scales)
    dev = k_cache.device
    kind = _rows(k, "k", dev, c.heads, c.head_dim)
    if _rows(v, "v", dev, c.heads, c.head_dim) != kind or v.shape != k.shape:
        raise ValueError("k and v must have one type and shape")
    if _rows(q, "q", dev, None, c.head_dim) != kind or q.shape[0] != k.shape[0]:
        raise ValueError("q must have the type and tokens of k")
    _int32(slots, "slots", dev)
    if slots.dim() != 1 or slots.shape[0] < k.shape[0]:
        raise ValueError("slots must be (tokens)")
    if angles is None and q_weight is None and k_weight is None:
        raise ValueError("without angles and weights there is nothing to append that write does not")
    pairs = 0
    if angles is not None:
        if angles.device != dev or angles.dtype != torch.float32:
            raise TypeError(f"angles must be float32 on {dev}")
        if angles.dim() != 3 or angles.shape[0] < k.shape[0] or angles.shape[2] != 2 or not angles.is_contiguous():
            raise ValueError("angles must be contiguous (tokens, pairs, 2)")
        pairs = angles.shape[1]
    for t, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if t is not None and (t.device != dev or t.dtype != k.dtype or tuple(t.shape) != (c.head_dim,) or not t.is_contiguous()):
            raise ValueError(f"{name} must be ({c.head_dim}) in the type of k on {dev}")
    with torch.cuda.device(dev):
        out = torch.empty((q.shape[0], q.shape[1], c.head_dim), dtype=q.dtype, device=dev)
        status = capi.load().i4mm_cache_append(
            ctypes.byref(c), out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), kind, k.shape[0], q.shape[1], q.stride(0), q.stride(1),
            k.stride(0), k.stride(1), v.stride(0), v.stride(1), slots.data_ptr(), angles.data_ptr() if angles is not None else None, pairs,
            int(interleaved), q_weight.data_ptr() if q_weight is not None else None, k_weight.data_ptr() if k_weight is not None else None,
            float(eps), torch.cuda.current_stream(dev).cuda_stream)
    _check(status, "cache append")
    return out


def read(k_cache: torch.Tensor, v_cache: torch.Tensor, scales: torch.Tensor, slots: torch.Tensor,
         dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
    """k, v (len(slots), heads, head_dim): the values that the cache holds at `slots` (zeros for slots outside of it)."""
    mod = ops.native() if dtype in _INPUT else False
    if mod:
        out = mod._try_cache_read(k_cache, v_cache, scales, slots, dtype == torch.bfloat16)
        if not isinstance(out, int):
            return out
        _check(max(out, 0), "cache read")
    c = _cache(k_cache, v_cache, scales)
    dev = k_cache.device
    if dtype not in _INPUT:
        raise TypeError("dtype must be float16 or bfloat16")
    _int32(slots, "slots", dev)
    if slots.dim() != 1:
        raise ValueError("slots must be (tokens)")
    with torch.cuda.device(dev):
        k, v = (torch.empty((slots.shape[0], c.heads, c.head_dim), dtype=dtype, device=dev) for _ in range(2))
        status = capi.load().i4mm_cache_read(ctypes.byref(c), k.data_ptr(), v.data_ptr(), _INPUT[dtype], slots.shape[0], slots.data_ptr(),
                                             torch.cuda.current_stream(dev).cuda_stream)
    _check(status, "cache read")
    return k, v


def attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor,
              seq_lens: torch.Tensor, cu_lens: Optional[torch.Tensor] = None, max_len: int = 1, *, scale: Optional[float] = None,
              window: int = 0, shared: Optional[Shared] = None) -> torch.Tensor:
    """softmax(scale * q k^T) v over the cached tokens that each row sees; (tokens, q_heads, head_dim) in q's type.

    q (tokens, q_heads, head_dim), q_heads a multiple of the cache's heads (query head h reads head h * heads // q_heads).  Rows
    cu_lens[b] .. cu_lens[b + 1] (without cu_lens: row b) are the last tokens of request b, which has seq_lens[b] tokens in the cache, their
    own included; each sees the tokens up to its own, with window > 0 the last `window` of them.  A row that sees none is 0.
    `max_len`: the most rows of a request; a wrong one costs time, nothing else.  `scale`: 1 / sqrt(head_dim) unless given.

    `shared`, of the same step: rows of a request that has a prefix see all of the prefix's tokens and then their own, as if the request held both
    (a window counts over both).  Its pages are fetched once for every 64 rows of a key head (a row: a token times a query head of it), once for every
    256 where there are more than 256, not once for each request.  That saves memory always and time from some readers on: 40 heads of 128, 8 readers of 2000
    tokens, 32 of 512; 32 query heads on 8, 32 readers of 2000, 8 of 16000.  Below that a block table whose rows name the pages of a prefix
    that fills them is faster, without `shared`.
    The call takes scratch of 4 bytes a value of q, whichever rows have a prefix.

    Two kernels serve it, chosen by sizes, and one for few readers and one for many work on shared prefixes.  All keep sums in fp32; but for the one of few rows
    they round weights to fp16 before they multiply the values.
    There is no backward pass: the output carries no gradient."""
    mod = ops.native()
    if mod:
        out = mod._try_cache_attention(q, k_cache, v_cache, scales, block_table, seq_lens, cu_lens, max_len, scale, window, shared, ops._cache_workspaces)
        if not isinstance(out, int):
            return out
        _check(max(out, 0), "cache attention")
    c = _cache(k_cache, v_cache, scales)
    dev = k_cache.device
    kind = _rows(q, "q", dev, None, c.head_dim)
    if q.shape[1] % c.heads:
        raise ValueError("q's heads must be a multiple of the cache's")
    width, row_stride = _table(block_table, dev)
    n = block_table.shape[0]
    _int32(seq_lens, "seq_lens", dev, (n,))
    if cu_lens is not None:
        _int32(cu_lens, "cu_lens", dev, (n + 1,))
    elif q.shape[0] < n:
        raise ValueError("without cu_lens, q must have a row for each request")
    if int(window) < 0 or int(max_len) < 0:
        raise ValueError("window and max_len must not be negative")
    if shared is not None:
        _int32(shared.prefix_of, "shared.prefix_of", dev, (n,))
        _int32(shared.starts, "shared.starts", dev, (n + 1,))
        _int32(shared.rows, "shared.rows", dev)
        if shared.rows.dim() != 1 or shared.rows.shape[0] < q.shape[0]:
            raise ValueError("shared.rows must have an entry for each row of q")
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev)
        ws = _workspace(dev, stream)
        out = torch.empty((q.shape[0], q.shape[1], c.head_dim), dtype=q.dtype, device=dev)
        lib = capi.load()
        args = (ctypes.byref(c), out.data_ptr(), q.data_ptr(), kind, q.shape[0], q.shape[1], q.stride(0), q.stride(1), block_table.data_ptr(),
                width, row_stride, seq_lens.data_ptr(), cu_lens.data_ptr() if cu_lens is not None else None, n,
                int(max_len), 1.0 / math.sqrt(c.head_dim) if scale is None else float(scale), int(window))
        if shared is None:
            status = lib.i4mm_cache_attention(*args, ws.data_ptr(), ws.numel(), stream.cuda_stream)
        else:
            room = torch.empty(lib.i4mm_cache_shared_scratch_bytes(q.shape[0], q.shape[1], c.head_dim), dtype=torch.uint8, device=dev)
            status = lib.i4mm_cache_attention_shared(*args, shared.prefix_of.data_ptr(), shared.starts.data_ptr(), shared.rows.data_ptr(),
                                                     shared.rows.shape[0], room.data_ptr(), room.numel(), ws.data_ptr(), ws.numel(), stream.cuda_stream)
    _check(status, "cache attention")
    return out


class PageTable:
    """The requests' lengths, their block table and the free pages, all on the GPU; `step` moves them on.

    A place of the batch (a row of the table) that holds no request has length 0; a request begins there with its first step and ends
    with a step of -1 tokens.  A step that cannot have all of its pages is not made: see `step`.  The arrays stay where they are, so that a step captured in a CUDA graph is the next step whenever the graph
    is replayed."""

    def __init__(self, requests: int, pages: int, page_size: int, max_seq: int, device="cuda"):
        dev = torch.device(device)
        self.page_size = int(page_size)
        with torch.inference_mode(False):             # (`step` writes to them, in that mode or not)
            # lengths and the count of free pages lie together: what `undo` keeps of them is one copy
            self._state = torch.zeros(requests + 1, dtype=torch.int32, device=dev)
            self._saved = torch.empty_like(self._state)
            self.seq_lens, self.free_count = self._state[:requests], self._state[requests:]
            self.free_count.fill_(pages)
            self.block_table = torch.full((requests, -(-max_seq // self.page_size)), -1, dtype=torch.int32, device=dev)
            self.free_pages = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=dev)
        self._can_undo = False

    def step(self, new_lens: torch.Tensor, max_tokens: int) -> Plan:
        """Request b adds new_lens[b] tokens (int32 on the GPU; -1: it ends).  max_tokens: their sum, or more.

        Where Plan.missing is not 0 there were too few pages, and the step is not made: all of Plan.slots are -1, so that its tokens
        are written nowhere, no request ends, and lengths and free pages stay.  (They are kept on the GPU: nothing waits.  What is
        computed with such a Plan is void; Plan.seq_lens and free_count are what would have come.)  The next step may be any other one."""
        p = plan(self.seq_lens, new_lens, self.block_table, self.free_pages, self.free_count, self.page_size, max_tokens)
        short = p.missing != 0
        p.slots.masked_fill_(short, -1)
        self._saved.copy_(self._state)
        torch.where(short, self.seq_lens, p.seq_lens, out=self.seq_lens)
        torch.where(short, self.free_count, p.free_count, out=self.free_count)
        self._can_undo = self._can_undo or not torch.cuda.is_current_stream_capturing()
        return p

    def share(self, prefix_of: torch.Tensor, plan: Plan) -> Shared:
        """`share` of the step that this table has just made, which was `plan`: prefix_of (requests) int32 on the GPU, places of this table."""
        return share(prefix_of, self.seq_lens, plan.cu_lens, plan.slots.shape[0])

    def undo(self) -> None:
        """Takes the last step back, before any of its tokens has been written into a cache: what a write does to a page (pages of requests
        that end are given out again in the same step; a scale that grows rounds the bytes beside the new ones again) is not undone."""
        if not self._can_undo:
            raise ValueError("there is no step to take back")
        self._state.copy_(self._saved)
        self._can_undo = False


class PagedCache:
    """One layer's keys and values: `pages` pages of `page_size` tokens, `heads` heads of `head_dim`, in int8 or float8_e4m3fn."""

    def __init__(self, pages: int, heads: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.int8, device="cuda"):
        if dtype not in _HELD:
            raise TypeError("dtype must be int8 or float8_e4m3fn")
        # (bytes of places that nothing was written to are read by no result, but they should be numbers)
        self.k, self.v = (torch.zeros((pages, heads, page_size, head_dim), dtype=torch.int8, device=device).view(dtype) for _ in range(2))
        self.scales = torch.zeros((pages, heads, 2), dtype=torch.float32, device=device)

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        write(self.k, self.v, self.scales, k, v, slots)

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, angles: Optional[torch.Tensor] = None, *,
               q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
               interleaved: bool = False) -> torch.Tensor:
        return append(self.k, self.v, self.scales, q, k, v, slots, angles, q_weight=q_weight, k_weight=k_weight, eps=eps, interleaved=interleaved)

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
        return read(self.k, self.v, self.scales, slots, dtype)

    def attention(self, q: torch.Tensor, table: PageTable, cu_lens: Optional[torch.Tensor] = None, max_len: int = 1, *,
                  scale: Optional[float] = None, window: int = 0, shared: Optional[Shared] = None) -> torch.Tensor:
        """Of the step that `table` has just made: its lengths include the step's tokens."""
        more = {} if shared is None else {"shared": shared}
        return attention(q, self.k, self.v, self.scales, table.block_table, table.seq_lens, cu_lens, max_len, scale=scale, window=window, **more)
