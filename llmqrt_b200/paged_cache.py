"""A paged key/value cache in 8 bits for ragged batches: pages and slots of a step's tokens, the cache's writes, and the
attention that reads it.

Codes are [pages, Hkv, page, d] in float8_e4m3fn or int8, with an fp32 scale for each page and head ([pages, Hkv]); a value is
code * scale.  A request's tokens lie in the pages that its row of the block table names, token i in row i % page of
the (i // page)-th; slot = page number * page + row.  Nothing here waits for the GPU, and all of it can be captured into a CUDA graph
(the calls return or update tensors of fixed sizes).

    cache = PagedKVCache8(layers, pages, page, Hkv, d, max_requests, max_seqlen, device)
    step = cache.plan(new_lens, max_tokens)             # once a step, for all layers
    cache.append(layer, k, v, step, cos, sin)           # k, v [max_tokens, Hkv, d], the new tokens of all requests back to back
    out = cache.attend(layer, q, cos=cos, sin=sin)      # q [B, Hq, d]: each request's newest token
    cache.release(done)                                 # requests that have ended

The reference has contiguous 16-bit caches only (runtime/nn_models/modules/nonlinear/cache.py:12-27).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib as L

CACHE_DTYPES = (torch.float8_e4m3fn, torch.int8)


def plan_step(context_lens, new_lens, block_table, free_pages, free_count, page_size: int, max_tokens: int, free_left=None,
              seq_lens=None):
    """Pages and slots of a step's new tokens, built on the GPU from the requests' lengths.

    context_lens, new_lens [B] int32 (B <= 8192): tokens that a request holds and those it is to get.  The pages that this takes
    come from the top of the stack free_pages[:free_count[0]] (int32; free_count [1] int32, on the device), in the order of the
    requests, and are written into block_table [B, width] (int32) behind those in use.  A request gets nothing where its tokens
    end beyond `max_tokens`, its pages beyond the table, or where the stack does not hold its pages and those of the requests
    before it; its seq_lens is then its context.
    The stack's new count goes to free_left (default: free_count itself), the lengths to seq_lens if given (it may be context_lens).
    Returns (seq_lens [B], cu_new [B + 1] running sums of
    new_lens, slots [max_tokens] int64, positions [max_tokens] int32): of the new tokens of all requests back to back, -1
    and 0 where there is none."""
    return L.fast.plan_step(context_lens, new_lens, block_table, free_pages, free_count, page_size, max_tokens, free_left,
                            seq_lens)


def release_pages(done, seq_lens, block_table, free_pages, free_count, page_size: int) -> None:
    """The pages of the requests that `done` [B] bool marks go back onto the stack, in place; their seq_lens become 0."""
    L.fast.release_pages(done, seq_lens, block_table, free_pages, free_count, page_size)


def kv8_append(k_cache, v_cache, k_scale, v_scale, k, v, slots, cos=None, sin=None, positions=None) -> None:
    """k, v [T, Hkv, d] (fp16 / bf16; slices of a fused projection's rows are read in place) into slots [T] int64; tokens whose
    slot lies outside the cache are skipped.

    With cos / sin (fp32 [rows, d/2], see glue.rope_tables) and positions [T] int32 the keys are rotated first (half-split pairing).
    The tokens of one page must stand next to one another in the order of their slots, as plan_step gives them: rows written before
    them in the page are requantized where the new tokens make its scale grow, and a call that writes one page in two
    places, or one slot twice, leaves that page undefined.  int8: scale = absmax / 127; e4m3: the least power of two that brings the
    absmax within 448.  Infinities are stored as the greatest code, NaN as NaN (int8: 0)."""
    L.fast.kv8_append(k_cache, v_cache, k_scale, v_scale, k, v, slots, cos, sin, positions)


def attn_decode_kv8(q, k_cache, v_cache, k_scale, v_scale, block_table, seqlens, max_seqlen: int, softcap: float = 0.0, cos=None,
                    sin=None):
    """Attention of the newest token of each sequence (q [B, Hq, d]), or of its newest Sq <= 16 (q [B, Sq, Hq, d], causal among
    themselves), over the cache; returns a tensor like q.  seqlens [B] int32 count the newest tokens, which are in the cache
    already; `max_seqlen` bounds them (the splits of the keys are sized by it: of a longer sequence only so many tokens are seen).

    At most 16 query heads per KV head, d = 64 or 128.  cos / sin: q is rotated at its token's position first.  q may be a slice of
    a fused projection's rows.  Table entries outside the cache are not read and their tokens get no weight; a query without a
    key gives zeros."""
    return L.fast.attn_decode_kv8(q, k_cache, v_cache, k_scale, v_scale, block_table, seqlens, max_seqlen, softcap, cos, sin)


class StepPlan(NamedTuple):
    """A step's new tokens, those of all requests back to back (PagedKVCache8.plan)."""
    cu_new: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor


class PagedKVCache8:
    """The caches of all layers, the pages' stack, the block table and the lengths of up to `max_requests` requests, on one device.
    All layers share one numbering of pages."""

    def __init__(self, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, max_requests: int,
                 max_seqlen: int, device, dtype: torch.dtype = torch.float8_e4m3fn):
        if dtype not in CACHE_DTYPES:
            raise TypeError(f"PagedKVCache8: the cache holds float8_e4m3fn or int8, not {dtype}")
        if page_size not in (16, 32, 64, 128) or head_dim not in (64, 128):
            raise ValueError("PagedKVCache8: pages hold 16, 32, 64 or 128 tokens, heads 64 or 128 features")
        if num_pages < 1 or not 0 < max_requests <= 8192:
            raise ValueError("PagedKVCache8: need a page, and 1 to 8192 requests")
        self.page_size, self.num_pages, self.max_requests = page_size, num_pages, max_requests
        self.width = -(-max_seqlen // page_size)
        self.max_seqlen = self.width * page_size
        shape = (num_layers, num_pages, num_kv_heads, page_size, head_dim)
        self.k, self.v = (torch.zeros(shape, dtype=torch.int8, device=device).view(dtype) for _ in range(2))
        self.k_scale, self.v_scale = (torch.ones(shape[:3], dtype=torch.float32, device=device) for _ in range(2))
        self.block_table = torch.full((max_requests, self.width), -1, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(max_requests, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device)      # (page 0 on top)
        self.free_count = torch.full((1,), num_pages, dtype=torch.int32, device=device)

    def plan(self, new_lens, max_tokens: int) -> StepPlan:
        """Pages and slots for new_lens[b] more tokens of every request (int32 [max_requests]); seq_lens count them from here on.
        A request that gets nothing (see plan_step) keeps its length: its slots are -1."""
        _, cu, slots, positions = plan_step(self.seq_lens, new_lens, self.block_table, self.free_pages, self.free_count,
                                            self.page_size, max_tokens, seq_lens=self.seq_lens)
        return StepPlan(cu, slots, positions)

    def append(self, layer: int, k, v, step: StepPlan, cos=None, sin=None) -> None:
        """Keys and values [max_tokens, Hkv, d] of the step's new tokens into a layer's cache (see kv8_append)."""
        kv8_append(self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], k, v, step.slots, cos, sin, step.positions)

    def attend(self, layer: int, q, max_seqlen: int | None = None, softcap: float = 0.0, cos=None, sin=None):
        """Attention of the newest token(s) of every request (q [max_requests, Hq, d] or [max_requests, Sq, Hq, d]) over a layer's
        cache (see attn_decode_kv8); `max_seqlen` bounds the lengths (default: what the table holds)."""
        bound = self.max_seqlen if max_seqlen is None else min(max_seqlen, self.max_seqlen)
        return attn_decode_kv8(q, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], self.block_table,
                               self.seq_lens, bound, softcap, cos, sin)

    def release(self, done) -> None:
        """Pages of the requests marked in `done` [max_requests] bool go back to the stack; their lengths become 0."""
        release_pages(done, self.seq_lens, self.block_table, self.free_pages, self.free_count, self.page_size)
