"""A KV cache held at a budget of rows: the rows that attention looked at least are dropped as the generation goes on.

The reference keeps every token's row for the whole generation (torch_ffa_api.cpp:65-66).  Here a pair's cache never grows
beyond `budget + slack` rows: every step adds to each row the softmax weight it was given, and when a sequence has filled its
slack the cache is cut back to `budget` rows -- the `recent` newest tokens, the `first` ones of the sequence, and the heaviest of
the rest, for each (batch, head) on its own.

    ffa = EvictingFastForwardAttn(K, V, budget=2048, recent=512, first=4, weights=prompt_weights)
    out = ffa.attention(q, k, v, softmax_scale)      # [B, H, Dh]; every sequence appends at its own length
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch


class EvictingFastForwardAttn:
    """K, V: [B, H, Lp, Dh] prompts, right-padded when `lengths` is given.  weights: [B, H, Lp], what the prompt's own attention
    gave each of its rows (None: nothing, so that of an overlong prompt the first rows stay until steps have told them apart).
    A prompt longer than the budget is cut at once.  slack: rows that may gather before the next cut (1: cut every token)."""

    def __init__(self, K: torch.Tensor, V: torch.Tensor, budget: int, recent: Optional[int] = None, first: int = 0, slack: int = 1,
                 lengths: Optional[Sequence[int]] = None, weights: Optional[torch.Tensor] = None):
        from . import FastForwardAttn

        B, H, Lp, _ = K.shape
        recent = budget // 4 if recent is None else recent
        if budget < 1 or slack < 1 or recent < 0 or first < 0 or recent + first > budget:
            raise ValueError("need budget >= 1, slack >= 1, recent and first >= 0, recent + first <= budget")
        self.lengths = [Lp] * B if lengths is None else [int(n) for n in lengths]
        if len(self.lengths) != B or any(not 0 <= n <= Lp for n in self.lengths):
            raise ValueError("lengths must hold one prompt length of [0, prompt rows] per sequence")
        self.budget, self.recent, self.first, self.slack = budget, recent, first, slack
        self.engine = FastForwardAttn(K, V, max(Lp, budget + slack), False)
        L, dev = self.engine.max_len, K.device
        self.weights = torch.zeros(B, H, L, dtype=torch.float32, device=dev)
        if weights is not None:
            if tuple(weights.shape) != (B, H, Lp):
                raise ValueError("weights must be [batch, heads, prompt rows]")
            self.weights[:, :, :Lp] = weights
        self.positions = torch.arange(L, dtype=torch.int32, device=dev).expand(B, H, L).contiguous()
        self.rows = torch.tensor(self.lengths, dtype=torch.int32, device=dev)
        self.seen = self.rows.clone()   # tokens of each sequence so far, dropped ones included: the next token's position
        self._cut_if_full(budget)

    def _cut_if_full(self, most: int) -> None:
        """Cuts back to the budget once a sequence holds more than `most` rows."""
        if max(self.lengths) <= most:
            return
        self.engine.evict(self.rows, self.weights, self.positions, self.budget, recent=self.recent, first=self.first, max_row=max(self.lengths))
        self.rows.clamp_(max=self.budget)
        self.lengths = [min(n, self.budget) for n in self.lengths]

    def attention(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, softmax_scale: float,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One decode step over the rows that are left, then the cut when a sequence has filled its slack."""
        out = self.engine.attention_accumulate(q, k, v, softmax_scale, self.rows, self.weights, self.positions, self.seen, out=out,
                                               max_row=max(self.lengths))
        self.rows += 1
        self.seen += 1
        self.lengths = [n + 1 for n in self.lengths]
        self._cut_if_full(self.budget + self.slack - 1)
        return out
