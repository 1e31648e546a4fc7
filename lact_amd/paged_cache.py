"""A cache of keys and values in pages, as a server of many sequences keeps it: written token by token or prompt by prompt, in 8 bits where its memory counts, read back,
and attended to by single tokens.  Beside window_attention_step (attention.py), whose cache is one tensor for a batch.  No counterpart in the reference.  bf16 and fp32
tokens, heads of 64 and 128; the arithmetic runs in csrc/paged_cache.h and csrc/paged_attention.h, and there is no other path: what the kernels do not take raises."""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .attention import _autocast, _dims, _options, _plain_only


class PagedCache(NamedTuple):
    """k, v: [pages, hkv, page size, d], bf16, fp32 or float8_e4m3fn; the page size a multiple of 16.  With 8 bits k_scale, v_scale: [pages, hkv, page size],
    float8_e8m0fnu, the power of two that a row's numbers are multiplied by.  Pages may lie anywhere apart ([pages, 2, hkv, page size, d] holds keys and
    values of a page next to each other); what is inside one is contiguous, on 16-byte boundaries.

    Which page holds what is the caller's business.  In all three functions below

    page_table: [b, n] int32 (int64 is converted), on the device: entry i of a sequence is the page of its places i * page size up to the next.  What lies outside
    0 .. pages - 1 is no page: its places are not written, read as zeros, and not seen.  Nor are places behind the table.  Sequences may share pages."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    @classmethod
    def empty(cls, pages: int, heads: int, page_size: int, head_size: int, *, dtype: torch.dtype = torch.bfloat16, device="cuda") -> "PagedCache":
        """A cache that holds nothing yet (its memory is not cleared, and needs not to be)."""
        k, v = (torch.empty(pages, heads, page_size, head_size, dtype=dtype, device=device) for _ in range(2))
        if dtype != torch.float8_e4m3fn:
            return cls(k, v)
        return cls(k, v, *(torch.empty(pages, heads, page_size, dtype=torch.float8_e8m0fnu, device=device) for _ in range(2)))


def _tensors(name: str, cache: PagedCache, *more: Optional[torch.Tensor]) -> None:
    if not isinstance(cache, PagedCache):
        raise TypeError(f"{name} takes a PagedCache, got {type(cache).__name__}")
    if cache.k is None or cache.v is None:
        raise TypeError(f"{name} takes a PagedCache with keys and values")
    _plain_only(name, *cache, *more)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (*cache, *more)):
        raise RuntimeError(f"{name} is for inference: call it under torch.no_grad()")


def _as_pages(cache: PagedCache, *ts: torch.Tensor):
    """Under autocast, which cannot change the pages' type: tokens of theirs.  (8 bits take tokens of either type.)"""
    if cache.k.dtype == torch.float8_e4m3fn or not (ts[0].is_cuda and torch.is_autocast_enabled("cuda")):
        return ts
    return tuple(t.to(cache.k.dtype) if t.is_floating_point() else t for t in ts)


@torch.compiler.disable
def paged_cache_write(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, starts: Optional[torch.Tensor] = None,
                      counts: Optional[torch.Tensor] = None) -> None:
    """k, v: [b, l, hkv, d], or [b, hkv, d] for one token each, of the pages' type, or bf16 or fp32 for pages of 8 bits.  Token i of sequence s goes to its place
    starts[s] + i (starts None: i) if i < counts[s] (counts None: all do); what else lies in the pages stays.  Under autocast they are cast to the pages' type,
    and for pages of 8 bits taken as they are.

    In 8 bits a row (one head of one token) is multiplied by the power of two with which its largest magnitude just fits in e4m3 (448), and rounded to nearest; NaN and
    infinities become NaN, beside the others' own scale.

    starts, counts: [b] int32 (int64 is converted), on the device.  Places that two tokens of one call would go to hold something of either.  The pages are written in
    place, for autograd too."""
    name = "paged_cache_write"
    _tensors(name, cache, k, v, page_table, starts, counts)
    k, v = _as_pages(cache, k, v)
    _lib.host().paged_cache_write(*cache, k, v, page_table, starts, counts)


@torch.compiler.disable
def paged_cache_read(cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor, tokens: int, starts: Optional[torch.Tensor] = None, *,
                     dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v): [b, tokens, hkv, d], of the pages' type, or for pages of 8 bits bf16 (which holds their numbers exactly but for what is not a
    multiple of 2^-133 or reaches 2^128) or with `dtype` fp32: entry i of sequence s is
    its place starts[s] + i (starts None: i), zeros from place lengths[s] on and where there is no page.

    lengths, starts: [b] int32 (int64 is converted), on the device."""
    name = "paged_cache_read"
    _tensors(name, cache, page_table, lengths, starts)
    if int(tokens) != tokens or tokens < 0:
        raise ValueError(f"{name}: tokens must be a number of tokens, got {tokens}")
    if dtype is None:
        dtype = torch.bfloat16 if cache.k.dtype == torch.float8_e4m3fn else cache.k.dtype
    elif not isinstance(dtype, torch.dtype):
        raise TypeError(f"{name}: dtype must be a torch.dtype, got {dtype!r}")
    k, v = _lib.host().paged_cache_read(*cache, page_table, lengths, int(tokens), starts, dtype)
    return k, v


@torch.compiler.disable
def paged_attention_step(q: torch.Tensor, cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor, window: Optional[int] = None, *,
                         score_cap: Optional[float] = None, distance_slopes: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """window_attention_step over pages: q [b, hq, d], bf16 or fp32, of the pages' type unless they are of 8 bits -> [b, hq, d]; hkv divides hq.

    lengths: [b] int32 (int64 is converted), on the device: the first lengths[i] places of sequence i are its tokens, the last of them the one that q belongs to (its key
    and value are in the cache already).  Lengths are cut to what the table holds; a sequence that sees nothing (length 0, no page) has output 0.  Places past
    the length and further back than the window are not seen, whatever they hold, and need no page.  Values are weighed and summed in fp32, and divided
    by their weights' sum last: the places seen times the largest magnitude (in 8 bits 448 times the largest power of two) have to stay below 2^119.  Under autocast q is
    cast to the pages' type, for pages of 8 bits to autocast's.  For inference: under torch.no_grad(), or with operands that need no gradient."""
    name = "paged_attention_step"
    _tensors(name, cache, q, page_table, lengths, distance_slopes)
    _dims(name, 3, q=q)
    q, = _autocast(q) if cache.k.dtype == torch.float8_e4m3fn else _as_pages(cache, q)
    window, scale, cap = _options(name, q.shape[2], window, score_cap, scale, distance_slopes)
    return _lib.host().paged_attention_step(q, *cache, page_table, lengths, window, scale, cap, distance_slopes)
