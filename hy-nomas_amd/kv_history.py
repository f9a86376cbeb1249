"""A history longer than what is read or kept: the quantized KV cache by blocks.

A roll-out outlives any fixed cache, and most of a long history draws little
attention. The reference answers with routed sparse attention and with history
policies (nomas_cache_sparse.py, swa_cache.py, uniform_history_cache.py); here
both work on the FP8/INT8 cache of fp8_kv_cache.py in place:

  make_block_bounds / update_block_bounds
      per block of tokens and head, the smallest and largest value of every key
      channel: kept beside the cache, brought up to date after each write
  select_blocks
      the blocks that each run of queries reads: those whose bounds allow the
      largest logits, with the first and the newest always among them;
      cache_attention.sparse_chunk_attention attends over them
  key_mass
      the attention weight that every cached key drew, added up over calls
  select_tokens / evict
      the tokens of largest mass, moved to the front of another cache; keys carry
      their rotation, so a moved token keeps its position

  LayerHistory
      one layer's bounds and mass, and the attention of its passes over them: what
      dit_block.FP8ARModel keeps per layer when it reads or cuts a long history

Scores are formed in 64 bits and rounded once to fp32, ties go to the lowest index:
the same call gives the same blocks and tokens.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import ops
from .fp8_kv_cache import _storage

STORAGE_KEYS = ("k", "v", "k_scale", "v_scale")


def make_block_bounds(cache: dict, *, block: int = 64) -> torch.Tensor:
    """Bounds of an empty cache: bf16 [B, ceil(cap / block), H, 2, D], +inf / -inf."""
    codes, _ = _storage(cache, "k")
    if block not in ops.BLOCK_SIZES:
        raise ValueError(f"block must be one of {ops.BLOCK_SIZES}")
    B, cap, H, D = codes.shape
    bounds = torch.empty((B, -(-cap // block), H, 2, D), dtype=torch.bfloat16, device=codes.device)
    bounds[:, :, :, 0].fill_(float("inf"))
    bounds[:, :, :, 1].fill_(float("-inf"))
    return bounds


def update_block_bounds(bounds: torch.Tensor, cache: dict, start: int, end: int, *, block: int = 64,
                        cache_valid: Optional[torch.Tensor] = None) -> None:
    """Bring the blocks that tokens [start, end) fall in up to date after a write of
    those tokens (``end`` is the cache's new length: later tokens do not count).
    cache_valid (bool [B or 1, >= end]) leaves invalid tokens out."""
    codes, scale = _storage(cache, "k")
    ops.kv_block_bounds_(bounds, codes, scale, start, end, block, cache_valid)


def select_blocks(q: torch.Tensor, bounds: torch.Tensor, kv_len: int, top_k: int, *, block: int = 64,
                  q_block: int = 128, keep_first: int = 0, keep_last: int = 0,
                  q_valid: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Block lists int32 [B, H, ceil(Lq / q_block), top_k] for
    cache_attention.sparse_chunk_attention (ops.select_kv_blocks)."""
    return ops.select_kv_blocks(q, bounds, kv_len, top_k, block, q_block, keep_first, keep_last, q_valid)


def key_mass(q: torch.Tensor, lse: torch.Tensor, cache: dict, kv_len: int, *,
             prior: Optional[torch.Tensor] = None, softmax_scale: Optional[float] = None,
             cache_valid: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention weight of cached keys [0, kv_len) from queries q [B, Lq, Hq, D] with
    log-sum-exps lse [B, Hq, Lq] (of the attention that q ran), onto ``prior``: a new
    fp32 [B, H, kv_len] (ops.attn_key_mass)."""
    codes, scale = _storage(cache, "k")
    return ops.attn_key_mass(q, lse, codes, scale, kv_len, prior,
                             None if softmax_scale is None else float(softmax_scale), cache_valid)


def select_tokens(mass: torch.Tensor, kv_len: int, keep: int, *, keep_first: int = 0, keep_last: int = 0,
                  cache_valid: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The tokens of [0, kv_len) that stay in each head, int32 [B, H, keep]
    (ops.select_kv_tokens)."""
    return ops.select_kv_tokens(mass, kv_len, keep, keep_first, keep_last, cache_valid)


def evict(cache: dict, out: dict, mass: torch.Tensor, kv_len: int, keep: int, *, keep_first: int = 0,
          keep_last: int = 0, cache_valid: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keep ``keep`` of the tokens [0, kv_len) of every head in ``out``, another cache
    of the same heads and format: select_tokens, then codes, scales and mass of the
    chosen ones moved to its rows [0, keep). Returns (idx, mass of the kept tokens),
    int32 and fp32 [B, H, keep]. With fewer valid tokens than ``keep``, idx ends in
    -1 and those rows of ``out`` stay as they are; a batch has as many in every head,
    so ``idx[:, 0] >= 0`` is the validity of out's rows."""
    for c in (cache, out):
        for key in ("k", "v"):
            _storage(c, key)
    if mass.ndim == 3 and mass.shape[2] > cache["k"].shape[1]:
        mass = mass[:, :, :kv_len]
    idx = ops.select_kv_tokens(mass, kv_len, keep, keep_first, keep_last, cache_valid)
    moved = ops.move_kv_tokens_(*(out[n] for n in STORAGE_KEYS), *(cache[n] for n in STORAGE_KEYS), mass, idx)
    return idx, moved


class LayerHistory:
    """Bounds and mass of one layer's cache, and its attention over them.

    ``top_k`` > 0: passes that do not write the cache read ``top_k`` blocks of a
    longer history (the first ``keep_first`` and the last ``keep_last`` of it
    always) and the current chunk; 0: all of it. ``track_mass``: writing passes,
    which read everything, add the weight that each cached key drew to ``mass``.
    A writing pass counts once ``commit`` is called; ``rollback`` forgets it. A pass over
    another number of tokens than ``length``, those accounted for, is refused (bounds and
    mass would be of other keys); one over none starts anew, and ``reset`` takes a
    cache's tokens in."""

    def __init__(self, cache: dict, *, top_k: int = 0, block: int = 64, q_block: int = 128, keep_first: int = 1,
                 keep_last: int = 2, track_mass: bool = False):
        if top_k < 0 or keep_first < 0 or keep_last < 0 or q_block < 1:
            raise ValueError("top_k, keep_first and keep_last must not be negative, q_block must be positive")
        if top_k and keep_first + keep_last > top_k:
            raise ValueError("keep_first + keep_last exceeds top_k")
        self.top_k, self.block, self.q_block = top_k, block, q_block
        self.keep_first, self.keep_last = keep_first, keep_last
        self.track_mass = track_mass
        self.bounds = make_block_bounds(cache, block=block) if top_k else None
        self.mass: Optional[torch.Tensor] = None    # fp32 [B, H, tokens], None: no token yet
        self.length = 0                             # tokens that bounds and mass account for
        self._written = None                        # (mass, start, end) of a pass not committed yet

    def reset(self, cache: dict, kv_len: int) -> None:
        """Account for cache tokens [0, kv_len) as they are, without mass so far."""
        if self.bounds is not None and kv_len:
            update_block_bounds(self.bounds, cache, 0, kv_len, block=self.block)
        codes = cache["k"]
        self.mass = (torch.zeros((codes.shape[0], codes.shape[2], kv_len), dtype=torch.float32, device=codes.device)
                     if self.track_mass and kv_len else None)
        self.length, self._written = kv_len, None

    def attend(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: dict, kv_len: int,
               update_cache: bool) -> torch.Tensor:
        """Attention of one pass over [cache tokens < kv_len | k, v]. On a writing pass
        k and v are in the cache already, from token kv_len on."""
        from .cache_attention import chunk_attention, sparse_chunk_attention
        if kv_len == 0:  # a new roll-out
            self.mass, self.length = None, 0
        elif kv_len != self.length:
            raise ValueError(f"the history accounts for {self.length} tokens, the pass reads {kv_len} (commit or reset)")
        if update_cache:
            end = kv_len + k.shape[1]
            mass = None
            if self.track_mass:
                out, lse = sparse_chunk_attention(q, cache, kv_len, None, k_cur=k, v_cur=v)
                mass = key_mass(q, lse, cache, end, prior=self.mass)
            else:
                out = chunk_attention(q, cache, kv_len, k_cur=k, v_cur=v)
            self._written = (mass, kv_len, end)
            return out
        if self.top_k and -(-kv_len // self.block) > self.top_k:
            idx = select_blocks(q, self.bounds, kv_len, self.top_k, block=self.block, q_block=self.q_block,
                                keep_first=self.keep_first, keep_last=self.keep_last)
            return sparse_chunk_attention(q, cache, kv_len, idx, block=self.block, q_block=self.q_block, k_cur=k,
                                          v_cur=v)[0]
        return chunk_attention(q, cache, kv_len, k_cur=k, v_cur=v)

    def commit(self, cache: dict) -> None:
        """The last writing pass stands: its mass, and the bounds of what it wrote. If the
        bounds cannot be made, nothing has changed and the pass still waits."""
        if self._written is None:
            return
        mass, start, end = self._written
        if self.bounds is not None:
            update_block_bounds(self.bounds, cache, start, end, block=self.block)
        if self.track_mass:
            self.mass = mass
        self.length, self._written = end, None

    def rollback(self) -> None:
        """The last writing pass was refused: nothing of it counts."""
        self._written = None

    def check_evict(self, kv_len: int) -> None:
        """ValueError if ``evict`` would refuse these tokens: for a model that cuts all of
        its layers or none."""
        if not self.track_mass or self.mass is None:
            raise ValueError("eviction needs the mass of the cached tokens (track_mass)")
        if kv_len != self.length:
            raise ValueError(f"the history accounts for {self.length} tokens, not {kv_len}")

    def evict(self, cache: dict, out: dict, kv_len: int, keep: int, *, keep_first: int = 0,
              keep_last: int = 0) -> torch.Tensor:
        """Keep ``keep`` tokens of every head in ``out`` (kv_history.evict by this layer's
        mass), whose bounds and mass take the old ones' place; ``out`` may be of another
        capacity. Returns the kept tokens."""
        self.check_evict(kv_len)
        bounds = self.bounds
        if bounds is not None and bounds.shape[1] != -(-out["k"].shape[1] // self.block):
            bounds = make_block_bounds(out, block=self.block)
        idx, mass = evict(cache, out, self.mass, kv_len, keep, keep_first=keep_first, keep_last=keep_last)
        self.bounds = bounds
        self.length, self._written = min(keep, kv_len), None
        self.mass = mass[:, :, :self.length]
        if self.bounds is not None:
            update_block_bounds(self.bounds, out, 0, self.length, block=self.block)
        return idx
