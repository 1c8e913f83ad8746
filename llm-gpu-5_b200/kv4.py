"""A key/value cache held in 4 bits, with eviction by accumulated attention weight.

``KV4Cache`` stands in for ``KVCache`` in ``MultiHeadAttention.forward(..., kv_cache=)`` and
``forward_decode``: keys and values are quantised as they enter (4.5 bits per value at head_dim 64
and 128 against 16 or 32), the decode attends over the codes, and, where weights are tracked, every
cached token keeps the attention it has received so far, so that ``evict`` can give up the tokens
that matter least.  The reference has no key/value cache (generate.py:611-628 runs the whole context
again for every token)."""

from __future__ import annotations

import torch

from . import mha_ops as ops


class KV4Cache:
    """4-bit keys and values of B sequences, [B, NH, max_len] rows of D values (16, 32, 64 or 128).

    ``length`` counts the rows in use, ``seen`` the tokens that have entered; they part company
    when ``evict`` gives rows up.  With ``track_weights``, ``weights`` [B, NH, cap] holds each row's
    accumulated attention weight (over the prompt's queries, or its last ``prompt_window`` ones, and
    every decoded token) and ``positions`` its token's position."""

    def __init__(self, B: int, max_len: int, NH: int, D: int, track_weights: bool = False, prompt_window: int | None = None):
        if B <= 0 or max_len <= 0 or NH <= 0:
            raise ValueError(f"KV4Cache: sizes must be positive, got B={B}, max_len={max_len}, NH={NH}")
        if prompt_window is not None and prompt_window <= 0:
            raise ValueError(f"KV4Cache: prompt_window must be positive, got {prompt_window}")
        self.B, self.max_len, self.NH, self.D = B, max_len, NH, D
        self.codes, self.params = ops.kv4_empty(B, NH, max_len, D)
        cap = self.codes.shape[3]
        self.weights = self.positions = None
        if track_weights:
            self.weights = torch.zeros((B, NH, cap), dtype=torch.float32, device="cuda")
            self.positions = torch.zeros((B, NH, cap), dtype=torch.int32, device="cuda")
        self.prompt_window = prompt_window
        self.length = 0
        self.seen = 0

    def store(self, qkv: torch.Tensor, pos: int):
        """Quantise K and V of qkv [B, T, 3C] (the fused projection's output): at pos 0 a new prompt,
        replacing what the cache held; at pos ``length`` the next tokens."""
        B, T, C3 = qkv.shape
        if pos not in (0, self.length):
            raise RuntimeError(f"KV4Cache: tokens go to position 0 or {self.length}, got {pos}")
        if pos + T > self.max_len:
            raise RuntimeError(f"KV4Cache: {pos + T} positions exceed max_len {self.max_len}")
        x = qkv.view(B, T, 3, self.NH, self.D)
        seen = self.seen if pos else 0
        ops.kv4_store(x[:, :, 1], x[:, :, 2], self.codes, self.params, pos, weights=self.weights,
                      positions=self.positions, seen=seen)
        self.length = pos + T
        self.seen = seen + T

    def add_prompt_weights(self, qkv: torch.Tensor, lse: torch.Tensor, dtype):
        """Add the prompt's attention weights (its causal softmax's column sums, from the forward's
        lse) to ``weights``; nothing without ``track_weights``."""
        if self.weights is None:
            return
        B, T, _ = qkv.shape
        x = qkv.view(B, T, 3, self.NH, self.D)
        first = 0 if self.prompt_window is None else max(0, T - self.prompt_window)
        # the tf32 forward truncates its scores' operands on tensor cores only, up to head_dim 32 (the projection's
        # layout always suits them); wider heads run in float32, and so do their weights
        if dtype == "tf32" and self.D > 32:
            dtype = torch.float32
        ops.key_weights(x[:, :, 0], x[:, :, 1], lse, first_query=first, weights=self.weights[:, :, :T], dtype=dtype)

    def attend(self, q: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of one query per sequence, q [B, NH, D], over the rows in use; adds the attention
        weights to ``weights`` when they are tracked."""
        if self.length == 0:
            raise RuntimeError("KV4Cache: the cache is empty")
        return ops.kv4_decode(q, self.codes, self.params, self.length, out=out, weights=self.weights)

    def evict(self, keep: int, recent: int = 0) -> torch.Tensor | None:
        """Give up all but ``keep`` rows per sequence and head: the last ``recent`` tokens stay, then
        those of the largest accumulated weight.  Returns the slots map of ``mha_ops.kv4_evict``, or None
        when the cache holds no more than ``keep`` rows."""
        if self.weights is None:
            raise RuntimeError("KV4Cache.evict() needs track_weights=True")
        if keep <= 0 or not 0 <= recent <= keep:
            raise ValueError(f"KV4Cache.evict: need 0 <= recent <= keep and keep > 0, got keep={keep}, recent={recent}")
        if self.length <= keep:
            return None
        slots = ops.kv4_evict(self.codes, self.params, self.weights, self.positions, self.length, keep, recent=recent,
                              seen=self.seen)
        self.length = keep
        return slots
