"""The paged key-value cache in 8 bits, and attention over it: what a decoder needs between its quantized linears.

    plan       the step's block tables and slot maps, on the GPU, from the requests' lengths
    write      quantise the step's keys and values into their pages
    read       tokens of the cache as the values that they stand for
    attention  softmax attention of the step's queries over the cached tokens
    PagedCache one layer's arrays;  PageTable  the requests' lengths, block table and free pages

The cache is (pages, heads, page_size, head_dim) int8 or float8_e4m3fn for keys and values, with fp32 scales (pages, heads, 2): a
byte q stands for q * scale.  page_size is 16, 32, 64 or 128 and head_dim 64 or 128.  Activations are fp16 or bf16.  Everything runs on
torch's current stream and nothing waits for the GPU, but for the first `attention` of a stream if it is made inside a graph capture: that
waits until its scratch has been cleared.
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
              window: int = 0) -> torch.Tensor:
    """softmax(scale * q k^T) v over the cached tokens that each row sees; (tokens, q_heads, head_dim) in q's type.

    q (tokens, q_heads, head_dim), q_heads a multiple of the cache's heads (query head h reads head h * heads // q_heads).  Rows
    cu_lens[b] .. cu_lens[b + 1] (without cu_lens: row b) are the last tokens of request b, which has seq_lens[b] tokens in the cache, their
    own included; each sees the tokens up to its own, with window > 0 the last `window` of them.  A row that sees none is 0.
    `max_len`: the most rows of a request; a wrong one costs time, nothing else.  `scale`: 1 / sqrt(head_dim) unless given.

    Two kernels serve it, chosen by sizes.  Both keep sums in fp32; the one for prompts rounds weights to fp16 before they multiply the values.
    There is no backward pass: the output carries no gradient."""
    mod = ops.native()
    if mod:
        out = mod._try_cache_attention(q, k_cache, v_cache, scales, block_table, seq_lens, cu_lens, max_len, scale, window, ops._cache_workspaces)
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
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev)
        ws = _workspace(dev, stream)
        out = torch.empty((q.shape[0], q.shape[1], c.head_dim), dtype=q.dtype, device=dev)
        status = capi.load().i4mm_cache_attention(
            ctypes.byref(c), out.data_ptr(), q.data_ptr(), kind, q.shape[0], q.shape[1], q.stride(0), q.stride(1), block_table.data_ptr(),
            width, row_stride, seq_lens.data_ptr(), cu_lens.data_ptr() if cu_lens is not None else None, n,
            int(max_len), 1.0 / math.sqrt(c.head_dim) if scale is None else float(scale), int(window), ws.data_ptr(), ws.numel(),
            stream.cuda_stream)
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

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
        return read(self.k, self.v, self.scales, slots, dtype)

    def attention(self, q: torch.Tensor, table: PageTable, cu_lens: Optional[torch.Tensor] = None, max_len: int = 1, *,
                  scale: Optional[float] = None, window: int = 0) -> torch.Tensor:
        """Of the step that `table` has just made: its lengths include the step's tokens."""
        return attention(q, self.k, self.v, self.scales, table.block_table, table.seq_lens, cu_lens, max_len, scale=scale, window=window)
