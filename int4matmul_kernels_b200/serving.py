"""The 13B-class layer stack as a server runs it: requests that come and go, prompts and single tokens in one batch, attention over a
paged 8-bit cache between the quantized linears.

    stack = sharding.DecoderStack(sharding.STACK_13B, 0, 1, "cuda")
    server = CachedStack(stack, heads=40, pages=4096, page_size=16, requests=64, max_seq=4096)
    h = server.step(prompts, new_lens, max_len)         # packed rows of the step's new tokens, request by request
    h = server.step(tokens, ones, 1)                    # one token of every request
    server.plan.missing                                 # of the last step, on the GPU: not 0 where there were too few pages

With positions, and requests that share a prefix which place 0 of the batch holds:

    server = CachedStack(stack, heads=40, ..., freqs=10000.0 ** (-torch.arange(64, device="cuda") / 64), norm=True)
    h = server.step(system_prompt, first_place_only, max_len)
    h = server.step(tokens, new_lens, max_len, prefix_of=prefix_of)
"""
from __future__ import annotations

from typing import Optional

import torch

from . import cache
from .sharding import DecoderStack


class CachedStack:
    """`DecoderStack` with attention in the place of its stand-in for it:

        q, k, v = qkv(norm(h));  k and v are written into the layer's cache;  t = norm(attention(q))
        h       = norm(h + norm(o(t)));   g, u = gate_up(h);   h = norm(h + norm(down(norm(g * u))))

    One set of tables (built on the GPU, once a step) serves all layers.  There are no learned parameters in it, as in the stack it wraps, and
    no positions unless `freqs` are given: it exists to run the operators together as a model does.  One GPU.

    freqs (pairs) fp32 on the GPU: queries and keys are rotated by position * freqs (`cache.append`: halves, or `interleaved` pairs).  norm: their
    heads are divided by the root of their mean square (weights of 1) before that."""

    def __init__(self, stack: DecoderStack, heads: int, pages: int, page_size: int, requests: int, max_seq: int,
                 dtype: torch.dtype = torch.int8, window: int = 0, freqs: Optional[torch.Tensor] = None, norm: bool = False,
                 interleaved: bool = False):
        if stack.world != 1:
            raise ValueError("CachedStack runs on one GPU")
        hidden = stack.cfg.hidden
        if hidden % heads:
            raise ValueError("heads must divide the stack's width")
        self.stack, self.heads, self.head_dim, self.window = stack, heads, hidden // heads, window
        device = stack.layers[0]["qkv"].matrix.device
        self.table = cache.PageTable(requests, pages, page_size, max_seq, device)
        self.plan = None                               # the last step's
        if freqs is not None and (freqs.device != device or freqs.dtype != torch.float32 or freqs.dim() != 1 or freqs.shape[0] % 8 or
                                  not 0 < 2 * freqs.shape[0] <= self.head_dim):
            raise ValueError(f"freqs must be float32 (pairs) on {device}, a multiple of 8 pairs within a head")
        self.freqs, self.interleaved = None if freqs is None else freqs.contiguous(), interleaved
        self.weight = torch.ones(self.head_dim, dtype=torch.float16, device=device) if norm else None
        self.caches = [cache.PagedCache(pages, heads, page_size, self.head_dim, dtype, device) for _ in stack.layers]

    def step(self, h: torch.Tensor, new_lens: torch.Tensor, max_len: int, prefix_of: Optional[torch.Tensor] = None) -> torch.Tensor:
        """h (tokens, hidden) fp16: the new tokens' rows, request by request; new_lens (requests) int32 on the GPU, -1 where a request
        ends; max_len: the most new tokens of a request; prefix_of (requests) int32 on the GPU: the place whose tokens come before each request's own,
        -1 for none (`cache.share`).  Returns the last layer's rows.  Nothing here waits for the GPU.

        Where self.plan.missing (on the GPU) is not 0, there were too few pages: the rows are void, tables and caches are as before the
        step, and a smaller one, or one in which requests end, can be made instead."""
        hidden = self.stack.cfg.hidden
        # (refused before the table moves)
        if h.device != self.table.seq_lens.device or h.dim() != 2 or h.shape[1] != hidden or h.stride(1) != 1:
            raise ValueError(f"h must be (tokens, {hidden}) on {self.table.seq_lens.device}, contiguous in its last dimension")
        if h.dtype != torch.float16:
            raise TypeError("h must be float16")
        if int(max_len) < 0:
            raise ValueError("max_len must not be negative")
        lens = self.table.seq_lens
        if prefix_of is not None and (prefix_of.device != lens.device or prefix_of.dtype != torch.int32 or prefix_of.shape != lens.shape or
                                      not prefix_of.is_contiguous()):
            raise ValueError(f"prefix_of must be contiguous int32 ({lens.shape[0]}) on {lens.device}")
        plan = self.plan = self.table.step(new_lens, h.shape[0])
        shared = None if prefix_of is None else self.table.share(prefix_of, plan)
        angles = None if self.freqs is None else cache.angles(plan.positions if shared is None else shared.positions, self.freqs)
        shape = (h.shape[0], self.heads, self.head_dim)
        comb = self.stack.combine
        x = comb(0, h)
        for i, (mats, held) in enumerate(zip(self.stack.layers, self.caches)):
            p = self.stack.multiply(mats["qkv"], x)
            q, k, v = (p[:, j * hidden:(j + 1) * hidden].unflatten(1, shape[1:]) for j in range(3))
            if angles is None and self.weight is None:
                held.write(k, v, plan.slots)
            else:
                q = held.append(q, k, v, plan.slots, angles, q_weight=self.weight, k_weight=self.weight, interleaved=self.interleaved)
            t = held.attention(q, self.table, plan.cu_lens, max_len, window=self.window, shared=shared)
            h = comb(2, h, self.stack.multiply(mats["o"], comb(0, t.flatten(1))))
            gate, up = self.stack._linear(mats["gate_up"], h, 2, "gate_up")
            d = self.stack.multiply(mats["down"], comb(3, gate, up))
            if i + 1 == len(self.caches):
                h = comb(2, h, d)
            else:
                h, x = self.stack.combine_and_normalise(h, d)
        return h
