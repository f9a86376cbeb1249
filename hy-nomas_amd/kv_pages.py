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

A page's codes and scales lie head by head ([P, H, page, D], seen as [P, page, H, D]): an
attention reads one head of many tokens, which is one run of memory then. (Single tokens of
eight sequences of 18000, 24 heads: 151 us, with codes that lie token by token 175; a scale
of every token would be a line of memory of its own.) Any strides are read.
"""
from __future__ import annotations

import heapq
from typing import Optional, Sequence

import torch

from . import _lib as L
from . import ops
from .fp8_kv_cache import CODE_DTYPES, FP8, KV_KEYS, STORAGE_KEYS, _raise_if_flagged


def make_pages(pages: int, heads: int, dim: int = 128, *, page: int = 64, layers: Optional[int] = None,
               code_dtype: torch.dtype = FP8, device: torch.device | str) -> dict:
    """Uninitialised pages: "k"/"v" codes [P, page, H, D] and "k_scale"/"v_scale" fp32 [P,
    page, H, 1] (views of [P, H, page, ..]); with ``layers`` each has that dim in front."""
    if page not in ops.BLOCK_SIZES:
        raise ValueError(f"page must be one of {ops.BLOCK_SIZES}")
    if code_dtype not in CODE_DTYPES:
        raise TypeError("pages hold float8_e4m3fn or int8 codes")
    lead = (pages,) if layers is None else (layers, pages)
    pool = {}
    for key in KV_KEYS:
        for name, last, dtype in ((key, dim, code_dtype), (f"{key}_scale", 1, torch.float32)):
            pool[name] = torch.empty((*lead, heads, page, last), dtype=dtype, device=device).transpose(-3, -2)
    return pool


def write_pages(cache: dict, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor, *,
                counts: Optional[torch.Tensor] = None, assume_finite: bool = False,
                status: Optional[torch.Tensor] = None, gpu_scales: bool = False) -> None:
    """Quantize bf16 K/V [B, L, H, D] into a layer's pages: token j of sequence b becomes
    its token start[b] + j (start int32 [B]), for j < counts[b] (int32 [B]; None: all L).

    The codes are those of fp8_kv_cache.quantize_kv_pair_into, and so is the check: unless
    ``assume_finite``, nothing is written if a new token holds a NaN/Inf (ValueError, or
    status[0] = 1 when a status tensor is given). Tokens past the table, and those whose
    page number is not in the pool, are dropped. The sequences of one call must not share
    the pages that they write.

    ``gpu_scales``: a row's scale is amax times the fp32 reciprocal of 448 (127), as torch
    on a GPU divides a tensor by a number, instead of the rounded quotient: pages that go
    on from codes a torch program made on the GPU hold what it would have, bit for bit."""
    args = (*(cache[n] for n in STORAGE_KEYS), k, v, table, start, counts)
    mode = L.HN_SCALE_RECIPROCAL if gpu_scales else L.HN_SCALE_ZERO_ONE
    if assume_finite:
        ops.kv_pages_write_(*args, None, mode)
        return
    flag = status if status is not None else torch.empty(1, dtype=torch.int32, device=k.device)
    ops.kv_pages_write_(*args, flag, mode)
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


class PagedKVCache:
    """The pages of all layers, and the sequences that hold them.

    A sequence is an id with a length and a list of pages; page p is the same place in
    every layer. Sequences share pages: ``fork`` gives a branch the pages of its origin,
    and a shared page is copied (all layers in one launch) when one of them is about to
    write it. A pass opens a ``PageBatch`` of its sequences, runs its layers with it and
    commits it; ``free``, ``truncate`` and ``compact`` run between passes.

    The pages are the host's: numbers and lengths live there, and a batch brings its
    tables to the GPU in one copy. All work is ordered on the current stream; ``open`` and
    ``compact`` cannot be captured into a graph (RuntimeError)."""

    def __init__(self, layers: int, pages: int, heads: int, dim: int = 128, *, page: int = 64,
                 code_dtype: torch.dtype = FP8, device: torch.device | str):
        if layers < 1 or pages < 1:
            raise ValueError("layers and pages must be positive")
        self.pool = make_pages(pages, heads, dim, page=page, layers=layers, code_dtype=code_dtype, device=device)
        self.layers, self.pages, self.page = layers, pages, page
        self.device = self.pool["k"].device  # (with its index)
        self._views = [{n: t[i] for n, t in self.pool.items()} for i in range(layers)]
        self._free = list(range(pages))             # a heap: the lowest number is taken first
        self._refs = [0] * pages
        self._table: dict[int, list[int]] = {}      # sequence -> its pages
        self._length: dict[int, int] = {}
        self._stamp: dict[int, int] = {}            # changes when a batch's view of the sequence is past
        self._turn: dict[int, int] = {}             # passes that were opened to add to the sequence
        self._next = 0

    def _not_captured(self) -> None:
        # (bookkeeping would run once, and the tables' copy replay from memory freed since)
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the pages of a PagedKVCache are the host's: open and compact cannot be captured")

    def layer(self, i: int) -> dict:
        """Layer i's pool, as write_pages and paged_attention take it."""
        return self._views[i]

    def length(self, seq: int) -> int:
        return self._length[self._known(seq)]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _known(self, seq: int) -> int:
        if seq not in self._table:
            raise ValueError(f"no sequence {seq}")
        return seq

    def new(self) -> int:
        """An empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._table[seq], self._length[seq], self._stamp[seq], self._turn[seq] = [], 0, 0, 0
        return seq

    def fork(self, seq: int) -> int:
        """A sequence with the tokens of ``seq``, on its pages: nothing is copied now."""
        self._known(seq)
        held = self._table[seq][:-(-self._length[seq] // self.page)]
        branch = self.new()
        self._table[branch], self._length[branch] = list(held), self._length[seq]
        for p in held:
            self._refs[p] += 1
        return branch

    def _drop(self, pages: list[int]) -> None:
        for p in pages:
            self._refs[p] -= 1
            if self._refs[p] == 0:
                heapq.heappush(self._free, p)

    def free(self, seq: int) -> None:
        """Forget a sequence; pages that no other one holds are free again."""
        self._drop(self._table.pop(self._known(seq)))
        del self._length[seq], self._stamp[seq], self._turn[seq]

    def truncate(self, seq: int, length: int) -> None:
        """Keep the first ``length`` tokens (drafted tokens that were refused go)."""
        if not 0 <= length <= self.length(seq):
            raise ValueError(f"cannot keep {length} of {self.length(seq)} tokens")
        held = self._table[seq]
        keep = -(-length // self.page)
        self._drop(held[keep:])
        del held[keep:]
        self._length[seq] = length
        self._stamp[seq] += 1

    def open(self, seqs: Sequence[int], tokens: int | Sequence[int] = 0) -> "PageBatch":
        """A pass of these sequences that adds ``tokens`` tokens to each (a number, or one
        for every sequence; 0: a pass that only reads). Room for them is taken now, and
        pages that they would write but share are copied; ValueError, with nothing
        changed, if the pool has not enough. A sequence grows in one pass at a time: an
        earlier batch that was to add to it is past."""
        self._not_captured()
        seqs = [self._known(s) for s in seqs]
        adds = [tokens] * len(seqs) if isinstance(tokens, int) else list(tokens)
        if len(adds) != len(seqs) or min(adds, default=0) < 0:
            raise ValueError("tokens: a number that is not negative, or one for every sequence")
        if any(adds) and len(set(seqs)) != len(seqs):
            raise ValueError("a sequence that grows occurs once in a pass")
        copies, grown, refs = [], [], {}  # (sequence, place), (sequence, pages), holders that leave a page
        for s, n in zip(seqs, adds):
            held, start = self._table[s], self._length[s]
            for i in range(start // self.page, min(len(held), -(-(start + n) // self.page))) if n else ():
                p = held[i]
                left = self._refs[p] - refs.get(p, 0)
                if left > 1:  # (the last holder writes it in place)
                    refs[p] = refs.get(p, 0) + 1
                    copies.append((s, i))
            grown.append((s, max(0, -(-(start + n) // self.page) - len(held))))
        if len(copies) + sum(n for _, n in grown) > len(self._free):
            raise ValueError(f"{len(copies) + sum(n for _, n in grown)} pages are needed, {len(self._free)} are free")
        src, dst = [], []
        for s, i in copies:
            held = self._table[s]
            src.append(held[i])
            dst.append(heapq.heappop(self._free))
            self._refs[held[i]] -= 1
            self._refs[dst[-1]] = 1
            held[i] = dst[-1]
            self._stamp[s] += 1
        for s, n in zip(seqs, adds):
            self._turn[s] += n > 0
        for s, n in grown:
            for _ in range(n):
                p = heapq.heappop(self._free)
                self._refs[p] = 1
                self._table[s].append(p)
        if src:
            copy_pages(self.pool, src, dst)
        return PageBatch(self, seqs, adds)

    def compact(self) -> int:
        """Move the pages in use to the lowest numbers (one copy over all layers); returns
        how many were moved. Batches opened before are of no use afterwards."""
        self._not_captured()
        used = [p for p in range(self.pages) if self._refs[p]]
        n = len(used)
        src = [p for p in used if p >= n]
        dst = [p for p in range(n) if not self._refs[p]]
        if src:
            copy_pages(self.pool, src, dst)
            to = dict(zip(src, dst))
            for s, held in self._table.items():
                held[:] = [to.get(p, p) for p in held]
                self._stamp[s] += 1
            for a, b in to.items():
                self._refs[b], self._refs[a] = self._refs[a], 0
            self._free = list(range(n, self.pages))
        return len(src)


class PageBatch:
    """One pass of some sequences of a PagedKVCache: their tables and lengths on the GPU.

    ``write`` puts a layer's new tokens into the pages, ``attend`` runs a layer's
    attention; ``commit`` makes the new tokens part of the sequences once every layer has
    written them. A batch that is not committed leaves the sequences as they were. Once
    it is committed or discarded, one of its sequences grows, is cut, freed or moved, or one
    that it adds to is opened to grow again, it is refused (ValueError)."""

    def __init__(self, cache: PagedKVCache, seqs: list[int], adds: list[int]):
        self.cache, self.seqs, self.adds = cache, seqs, adds
        self.lengths = [cache._length[s] for s in seqs]
        self._stamps = [cache._stamp[s] for s in seqs]
        self._turns = [(s, cache._turn[s]) for s, a in zip(seqs, adds) if a]
        B, tables = len(seqs), [cache._table[s] for s in seqs]
        width = max((len(t) for t in tables), default=0)
        flat = self.lengths + [n + a for n, a in zip(self.lengths, adds)] + adds
        for t in tables:
            flat += t + [-1] * (width - len(t))
        host = torch.tensor(flat, dtype=torch.int32)
        if cache.device.type == "cuda":
            host = host.pin_memory()
        flat = host.to(cache.device, non_blocking=True)
        self.start, self.end, counts = flat[:3 * B].view(3, B).unbind(0)    # tokens before and after the pass
        self.table = flat[3 * B:].view(B, width)
        self.counts = None if len(set(adds)) <= 1 else counts
        self._over = False

    def _check(self) -> None:
        if self._over:
            raise ValueError("the batch is past: it was committed or discarded")
        stamp, turn = self.cache._stamp, self.cache._turn
        if any(stamp.get(s) != n for s, n in zip(self.seqs, self._stamps)):
            raise ValueError("the batch is past: a sequence grew, was cut, freed or moved since it was opened")
        if any(turn[s] != n for s, n in self._turns):
            raise ValueError("the batch is past: a sequence that it adds to was opened to grow again")

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, *, assume_finite: bool = False,
              status: Optional[torch.Tensor] = None) -> None:
        """Layer ``layer``'s K/V [B, L, H, D] of the new tokens: the first of each
        sequence's L rows, as many as it adds (write_pages)."""
        self._check()
        if k.shape[0] != len(self.seqs) or k.shape[1] < max(self.adds, default=0) or (
                self.counts is None and k.shape[1] != max(self.adds, default=0)):
            raise ValueError("k and v must hold the tokens that the batch was opened for")
        write_pages(self.cache.layer(layer), k, v, self.table, self.start, counts=self.counts,
                    assume_finite=assume_finite, status=status)

    def attend(self, layer: int, q: torch.Tensor, *, causal: bool = False, k_cur: Optional[torch.Tensor] = None,
               v_cur: Optional[torch.Tensor] = None, cur_valid: Optional[torch.Tensor] = None,
               softmax_scale: Optional[float] = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Attention of q [B, Lq, Hq, D]: with k_cur/v_cur over the tokens before the pass
        and those, without over the tokens written by it too (paged_attention). Causal
        queries are every sequence's last Lq tokens. Where the sequences add different
        numbers of tokens, Lq queries, as many as the longest adds or more (padding), stand
        as write's rows do: query i is the sequence's i-th new token, and one past them
        sees what the last does."""
        from .cache_attention import paged_attention
        self._check()
        rows = causal and self.counts is not None and q.shape[1] >= max(self.adds)
        return paged_attention(q, self.cache.layer(layer), self.table, self.end if k_cur is None else self.start,
                               causal=causal, k_cur=k_cur, v_cur=v_cur, cur_valid=cur_valid,
                               softmax_scale=softmax_scale, q_start=self.start if rows else None)

    def commit(self) -> None:
        """The new tokens stand; the batch is of no use afterwards. Sequences to which it adds
        nothing, and other passes over those, go on."""
        self._check()
        self._over = True
        for s, n, a in zip(self.seqs, self.lengths, self.adds):
            if a:
                self.cache._length[s] = n + a
                self.cache._stamp[s] += 1

    def discard(self) -> None:
        """Give up the pass: the room that was taken for it is free again."""
        self._check()
        self._over = True
        for s, n, a in zip(self.seqs, self.lengths, self.adds):
            if a:
                self.cache.truncate(s, n)
