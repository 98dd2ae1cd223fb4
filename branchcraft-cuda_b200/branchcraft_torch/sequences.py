"""Sequences over a paged copy-on-write cache whose bookkeeping lives on the GPU.

`PagedSequences` holds what a serving loop keeps between steps - the K/V cache,
page tables, lengths, reference counts and the free stack - and runs its steps
on the device, with no host round trip: `append` gives new tokens their pages
and writes their rows (prompts, chunks of prompts and single tokens alike),
`attend` lets them attend, `reorder` follows a beam search's parents. Every step
can be captured in a CUDA graph. `PagedTreeCache` (transaction.py) is the host's
form of the same pool: its rules, page order included, are these.
"""
from __future__ import annotations

import torch

from . import append_kv_, append_plan_, beam_reorder_, chunk_attention

__all__ = ["PagedSequences"]


class PagedSequences:
    """`requests` x `beams` rows (row request * beams + beam), all empty at first."""

    def __init__(self, requests: int, beams: int, max_pages: int, physical_pages: int,
                 kv_heads: int, head_dim: int, dtype: torch.dtype = torch.float16,
                 device: str = "cuda"):
        if min(requests, beams, max_pages, physical_pages, kv_heads) < 1:
            raise ValueError("all sizes must be positive")
        if head_dim not in (64, 128) or dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("head_dim must be 64/128, dtype float16 or bfloat16")
        i32 = dict(dtype=torch.int32, device=device)
        self.requests, self.beams = requests, beams
        self.k = torch.zeros((physical_pages, 16, kv_heads, head_dim), dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.pages = torch.full((requests * beams, max_pages), -1, **i32)
        self.lengths = torch.zeros(requests * beams, **i32)
        self.refcount = torch.zeros(physical_pages, **i32)
        # (the host pool's order: the last entry, page 0 at first, is popped first)
        self.free_stack = torch.arange(physical_pages - 1, -1, -1, **i32)
        self.free_count = torch.full((1,), physical_pages, **i32)
        self.counts = torch.zeros(3, **i32)  # of the last append: tokens, clones, status

    def append(self, k: torch.Tensor, v: torch.Tensor, new_tokens: torch.Tensor):
        """Append new_tokens [rows] (int32, on the device) tokens to the rows, row by row out
        of k, v [tokens, KV heads, head dim]; `tokens` may exceed their sum. Returns
        (query_start [rows + 1], positions [tokens]): which of the tokens are a row's, and
        where they stand in it (-1: in no row). When the plan fails (see check) nothing is
        appended and no token is in any row."""
        # (refused here: the plan below changes the tables before the rows are looked at)
        heads, dim = self.k.shape[2:]
        for t in (k, v):
            if (t.dim() != 3 or t.shape[0] != k.shape[0] or tuple(t.shape[1:]) != (heads, dim)
                    or t.dtype != self.k.dtype or t.device != self.k.device
                    or t.stride(2) != 1 or (heads > 1 and t.stride(1) != dim)
                    or (t.shape[0] > 1 and (t.stride(0) < 0 or t.stride(0) % 8))
                    or t.data_ptr() % 16):
                raise ValueError("k and v must be [tokens, KV heads, head dim] of the cache's type "
                                 "and device, each token's heads contiguous, 16-byte aligned")
        query_start, slot_map, positions, clones, counts = append_plan_(
            self.pages, self.lengths, new_tokens, self.refcount, self.free_stack,
            self.free_count, k.shape[0])
        append_kv_(self.k, self.v, k, v, slot_map, clones, counts)
        # (in place: a replayed step reports to the same tensor as the calls between)
        self.counts.copy_(counts)
        return query_start, positions

    def attend(self, q: torch.Tensor, query_start: torch.Tensor, **options) -> torch.Tensor:
        """Attention of the tokens just appended, q [tokens, query heads, head dim]; options as
        for chunk_attention."""
        return chunk_attention(q, self.k, self.v, self.pages, query_start, self.lengths, **options)

    def reorder(self, parents: torch.Tensor):
        """Row (r, j) becomes row (r, parents[r, j]) of before; -1 empties it."""
        if tuple(parents.shape) != (self.requests, self.beams):
            raise ValueError("parents must be [requests, beams]")
        shape = (self.requests, self.beams)
        pages, lengths = beam_reorder_(self.pages.view(*shape, -1), self.lengths.view(shape),
                                       parents, self.refcount, self.free_stack, self.free_count)
        # (in place, so that a captured step finds its tables again)
        self.pages.copy_(pages.view_as(self.pages))
        self.lengths.copy_(lengths.view_as(self.lengths))

    def check(self):
        """Raise what the host pool would have raised for the last append (synchronises)."""
        status = int(self.counts[2].item())
        if status == 1:
            raise ValueError("negative token count, or more tokens than rows were given")
        if status == 2:
            raise RuntimeError("KV page pool exhausted")
        if status:
            raise RuntimeError("malformed page table")
