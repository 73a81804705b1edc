"""Serving with cached keys and values: packed prompts, decode steps behind a prefix
the batch shares, and caches of bounded length.

``CachedAttention`` is an attention layer with grouped heads whose keys and values
live in a ``SequenceCache``; it runs ``ops.prompt_attn``, ``ops.shared_prefix_attn``
and ``ops.cache_evict`` the way a server does:

    layer = CachedAttention(d_model, num_heads, num_kv_heads).to("cuda", torch.bfloat16)
    prefix = layer.encode_prefix(x_prefix)                  # once for every sequence
    cache = layer.new_cache(batch, capacity)
    y = layer.prefill(x_prompts, seq_lens, cache, prefix)   # [sum(seq_lens), d_model]
    y = layer.decode(x_tokens, cache, prefix)               # [batch, d_model], one step
    cache.evict(budget, recent)                             # when it has grown too long

``python -m tiktok_techjam_2026_track3_b200.serving_example`` runs such a session.
"""

from __future__ import annotations

from typing import List, NamedTuple, Optional, Sequence

import torch
import torch.nn as nn

from . import ops

__all__ = ["CachedAttention", "SequenceCache", "SharedPrefix"]


class SharedPrefix(NamedTuple):
    """Keys and values [P, Hkv, hd] that every sequence attends first."""
    k: torch.Tensor
    v: torch.Tensor


class SequenceCache:
    """Keys, values [B, C, Hkv, hd] and accumulated attention weights [B, Hkv, C] of a
    batch of sequences.  The lengths are kept on the device (for the kernels) and on
    the host (so that a full cache is an error before anything is launched)."""

    def __init__(self, batch: int, capacity: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype, device: torch.device) -> None:
        shape = (batch, capacity, num_kv_heads, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self._spare: Optional[tuple] = None   # the pair the next eviction compacts into
        self.key_weights = torch.zeros(batch, num_kv_heads, capacity, dtype=torch.float32, device=device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.host_lengths: List[int] = [0] * batch
        self._rows = torch.arange(batch, device=device)

    @property
    def capacity(self) -> int:
        return self.k.shape[1]

    def _room(self, more: Sequence[int]) -> None:
        if len(more) != len(self.host_lengths):
            raise RuntimeError(f"expected {len(self.host_lengths)} sequences, got {len(more)}")
        for b, (have, add) in enumerate(zip(self.host_lengths, more)):
            if add < 0:
                raise RuntimeError(f"sequence {b} cannot take {add} rows")
            if have + add > self.capacity:
                raise RuntimeError(f"cache of sequence {b} is full: {have} + {add} rows, capacity {self.capacity}")

    def _fit(self, rows: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """k and v are that many rows of this cache's (index assignment would spread a single one)."""
        for t, n in ((k, "k"), (v, "v")):
            if t.shape != (rows, *self.k.shape[2:]) or t.dtype != self.k.dtype:
                raise RuntimeError(f"{n} must be {self.k.dtype} {[rows, *self.k.shape[2:]]}, got {t.dtype} {list(t.shape)}")

    def extend(self, seq_lens: Sequence[int], k: torch.Tensor, v: torch.Tensor) -> None:
        """Append packed rows k, v [sum(seq_lens), Hkv, hd], seq_lens[b] of them to sequence b."""
        lens = [int(n) for n in seq_lens]
        self._room(lens)
        self._fit(sum(lens), k, v)
        dev = self.k.device
        n = torch.tensor(lens, dtype=torch.int64)
        b = torch.repeat_interleave(torch.arange(len(lens)), n)
        at = torch.arange(int(n.sum())) - torch.repeat_interleave(n.cumsum(0) - n, n)
        at = at + torch.tensor(self.host_lengths, dtype=torch.int64)[b]
        b, at = b.to(dev), at.to(dev)
        self.k[b, at], self.v[b, at] = k, v
        self.host_lengths = [x + y for x, y in zip(self.host_lengths, lens)]
        self.lengths = torch.tensor(self.host_lengths, dtype=torch.int32, device=dev)

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """Append one row k, v [B, Hkv, hd] to every sequence."""
        self._room([1] * len(self.host_lengths))
        self._fit(len(self.host_lengths), k, v)
        at = self.lengths.long()
        self.k[self._rows, at], self.v[self._rows, at] = k, v
        self.lengths += 1
        self.host_lengths = [n + 1 for n in self.host_lengths]

    def _drop(self) -> None:
        """Take the last ``append`` back (rows past the lengths may hold anything)."""
        self.lengths -= 1
        self.host_lengths = [n - 1 for n in self.host_lengths]

    def evict(self, budget: int, recent: int) -> torch.Tensor:
        """Keep at most ``budget`` rows per head: the last ``recent`` and the heaviest of
        the others.  Returns the kept rows' indices [B, Hkv, budget] (-1: none)."""
        if budget > self.capacity:
            raise RuntimeError(f"budget {budget} exceeds the capacity {self.capacity}")
        if self._spare is None:
            self._spare = (torch.zeros_like(self.k), torch.zeros_like(self.v))
        kept = ops.cache_evict(self.k, self.v, self.key_weights, self.lengths, budget, recent, out=self._spare)
        (self.k, self.v), self._spare = self._spare, (self.k, self.v)
        self.key_weights = torch.zeros_like(self.key_weights)
        self.key_weights[:, :, :budget] = kept.key_weights
        self.lengths = kept.lengths
        self.host_lengths = [min(n, budget) for n in self.host_lengths]
        return kept.positions


def _join(a: torch.Tensor, lse_a: torch.Tensor, b: torch.Tensor, lse_b: torch.Tensor) -> torch.Tensor:
    """Attention over the union of two key sets from its results over each."""
    w = torch.sigmoid(lse_b - lse_a)[..., None]    # the second set's share
    return torch.lerp(a.float(), b.float(), w).to(a.dtype)


class CachedAttention(nn.Module):
    """Attention layer with ``num_heads`` query heads over ``num_kv_heads`` key / value
    heads, on packed tokens [T, d_model] (no batch dimension)."""

    def __init__(self, d_model: int, num_heads: int, num_kv_heads: int) -> None:
        super().__init__()
        if d_model % num_heads != 0:
            raise ValueError("d_model must be divisible by num_heads")
        if num_heads % num_kv_heads != 0:
            raise ValueError("num_heads must be divisible by num_kv_heads")
        self.num_heads, self.num_kv_heads, self.head_dim = num_heads, num_kv_heads, d_model // num_heads
        self.qkv_proj = nn.Linear(d_model, (num_heads + 2 * num_kv_heads) * self.head_dim)
        self.out_proj = nn.Linear(d_model, d_model)

    def _qkv(self, x: torch.Tensor):
        hq, hkv = self.num_heads, self.num_kv_heads
        packed = ops.linear(x, self.qkv_proj.weight.detach(), self.qkv_proj.bias.detach())
        packed = packed.view(x.shape[0], hq + 2 * hkv, self.head_dim)
        return packed[:, :hq], packed[:, hq:hq + hkv], packed[:, hq + hkv:]

    def _out(self, ctx: torch.Tensor) -> torch.Tensor:
        return ops.linear(ctx.flatten(1), self.out_proj.weight.detach(), self.out_proj.bias.detach())

    def new_cache(self, batch: int, capacity: int) -> SequenceCache:
        w = self.qkv_proj.weight
        return SequenceCache(batch, capacity, self.num_kv_heads, self.head_dim, w.dtype, w.device)

    def plan(self, seq_lens: Sequence[int]) -> ops.PromptPlan:
        return ops.PromptPlan(seq_lens, self.num_heads, self.num_kv_heads, self.head_dim, self.qkv_proj.weight.device)

    def encode_prefix(self, x: torch.Tensor) -> SharedPrefix:
        """Keys and values of prefix tokens x [P, d_model]."""
        _, k, v = self._qkv(x)
        return SharedPrefix(k, v)

    def _no_prefix(self, like: torch.Tensor) -> SharedPrefix:
        none = like.new_empty(0, self.num_kv_heads, self.head_dim)
        return SharedPrefix(none, none)

    def prefill(self, x: torch.Tensor, seq_lens: Sequence[int], cache: SequenceCache,
                prefix: Optional[SharedPrefix] = None, plan: Optional[ops.PromptPlan] = None) -> torch.Tensor:
        """Prompts x [sum(seq_lens), d_model] of the cache's (empty) sequences: each token
        attends the prefix and its own prompt up to itself.  ``plan``, where the caller
        has one, must be of these lengths.  Behind a prefix the two contexts are joined
        as the operators return them, in x's dtype, and rounded once more."""
        if any(cache.host_lengths):
            raise RuntimeError("prefill starts sequences: the cache must be empty")
        lens = tuple(int(n) for n in seq_lens)
        if x.shape[0] != sum(lens):
            raise RuntimeError(f"x holds {x.shape[0]} tokens, seq_lens {sum(lens)}")
        if plan is not None and plan.seq_lens != lens:
            # (one of the same total would attend across the prompts' boundaries)
            raise RuntimeError("the plan was built for other prompt lengths than seq_lens")
        cache._room(lens)
        q, k, v = self._qkv(x)
        plan = self.plan(lens) if plan is None else plan
        ctx, lse = ops.prompt_attn(q, k, v, plan, return_lse=True)
        if prefix is not None and x.shape[0] > 0:
            # every prompt token is one more row over the prefix
            no_rows = k.new_empty(x.shape[0], 0, self.num_kv_heads, self.head_dim)
            none = torch.zeros(x.shape[0], dtype=torch.int32, device=x.device)
            over, lse_over = ops.shared_prefix_attn(q, prefix.k, prefix.v, no_rows, no_rows, none, return_lse=True)
            ctx = _join(ctx, lse, over, lse_over)
        y = self._out(ctx)
        cache.extend(lens, k, v)    # last: a refused call leaves the cache empty
        return y

    def decode(self, x: torch.Tensor, cache: SequenceCache, prefix: Optional[SharedPrefix] = None) -> torch.Tensor:
        """One new token per sequence, x [B, d_model]: appended to the cache, attended, and
        the step's attention weights added to the cache's."""
        q, k, v = self._qkv(x)
        cache.append(k, v)
        try:
            pre = self._no_prefix(k) if prefix is None else prefix
            ctx, key_weights = ops.shared_prefix_attn(q, pre.k, pre.v, cache.k, cache.v, cache.lengths,
                                                      key_weights=cache.key_weights)
            y = self._out(ctx)
        except BaseException:       # a refused call leaves the cache as it was
            cache._drop()
            raise
        cache.key_weights = key_weights
        return y
