"""The quantized KV cache in pages: roll-outs that branch, sessions of any length.

A contiguous cache (fp8_kv_cache) belongs to one roll-out; trying two actions from one
history, or holding many sessions of different lengths, would copy the history or
reserve the longest session's room for each. Here a layer's cache is a pool of pages of
64 to 1024 tokens, in the codes and scales of fp8_kv_cache, and a sequence is a row of
page numbers and a length:

  make_pages        a pool of one or of all layers
  write_pages       new K/V of every sequence, quantized into its pages
  copy_pages        pages copied, in all layers at once
  read_pages        keys or values of the sequences, decoded
  cache_attention.paged_attention
                    attention over each sequence's own pages
  PagedKVCache      the pages of all layers: sequences that share pages, forked without
                    a copy (the page that a branch writes next is copied then), cut,
                    freed, and moved to the pool's front

A page's scales lie head by head ([P, H, page], seen as [P, page, H, 1]): a head's scales
of consecutive tokens are one line of memory, where they are a line apart token by token.
Any strides are read.
"""
from __future__ import annotations

import heapq
from typing import Optional, Sequence

import torch

from . import ops
from .fp8_kv_cache import CODE_DTYPES, FP8, KV_KEYS, STORAGE_KEYS, _raise_if_flagged


def make_pages(pages: int, heads: int, dim: int = 128, *, page: int = 64, layers: Optional[int] = None,
               code_dtype: torch.dtype = FP8, device: torch.device | str) -> dict:
    """Uninitialised pages: "k"/"v" codes [P, page, H, D] and "k_scale"/"v_scale" fp32 [P,
    page, H, 1] (views of [P, H, page]); with ``layers`` each has that dim in front."""
    if page not in ops.BLOCK_SIZES:
        raise ValueError(f"page must be one of {ops.BLOCK_SIZES}")
    if code_dtype not in CODE_DTYPES:
        raise TypeError("pages hold float8_e4m3fn or int8 codes")
    lead = (pages,) if layers is None else (layers, pages)
    pool = {}
    for key in KV_KEYS:
        pool[key] = torch.empty((*lead, page, heads, dim), dtype=code_dtype, device=device)
        pool[f"{key}_scale"] = torch.empty((*lead, heads, page, 1), dtype=torch.float32, device=device).transpose(-3, -2)
    return pool


def write_pages(cache: dict, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor, *,
                counts: Optional[torch.Tensor] = None, assume_finite: bool = False,
                status: Optional[torch.Tensor] = None) -> None:
    """Quantize bf16 K/V [B, L, H, D] into a layer's pages: token j of sequence b becomes
    its token start[b] + j (start int32 [B]), for j < counts[b] (int32 [B]; None: all L).

    The codes are those of fp8_kv_cache.quantize_kv_pair_into, and so is the check: unless
    ``assume_finite``, nothing is written if a new token holds a NaN/Inf (ValueError, or
    status[0] = 1 when a status tensor is given). Tokens past the table, and those whose
    page number is not in the pool, are dropped. The sequences of one call must not share
    the pages that they write."""
    args = (*(cache[n] for n in STORAGE_KEYS), k, v, table, start, counts)
    if assume_finite:
        ops.kv_pages_write_(*args)
        return
    flag = status if status is not None else torch.empty(1, dtype=torch.int32, device=k.device)
    ops.kv_pages_write_(*args, flag)
    if status is None:
        _raise_if_flagged(flag)


def copy_pages(cache: dict, src: Sequence[int], dst: Sequence[int]) -> None:
    """Page dst[i] <- page src[i], codes and scales, of one layer's pool or of all layers
    ([layers, P, page, H, D]). The lists are the host's. One page may be copied to several;
    a page that is written occurs once, and is not read (ValueError)."""
    ops.kv_pages_copy_(*(cache[n] for n in STORAGE_KEYS), list(src), list(dst))


def read_pages(cache: dict, key: str, table: torch.Tensor, kv_len: torch.Tensor, max_len: int) -> torch.Tensor:
    """Keys or values (``key`` "k" or "v") of the sequences' tokens [0, max_len) as bf16
    [B, max_len, H, D]: bf16(code * scale) below kv_len[b] (int32 [B]), zeros behind."""
    if key not in KV_KEYS:
        raise ValueError(f"Invalid KV key: {key}")
    return ops.kv_pages_read(cache[key], cache[f"{key}_scale"], table, kv_len, max_len)
