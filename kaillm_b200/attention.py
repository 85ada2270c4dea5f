"""What a decode step runs between the q/k/v projection and the output projection, over a paged key-value cache.

The reference leaves this part to vLLM, whose model code calls its linear method; here it is what `sharded.DecoderStack` runs
between its projections when it is given a `StepAttention`:

    total, starts, positions, slots, taken = plan_pages(block_table, seq_lens, new_lens, free_pages, taken, page_size, tokens)
    q = qk_norm_rope_store(qkv, positions, inv_freq, heads, k_cache, v_cache, slots, q_weight=..., k_weight=...)   # every layer
    out = paged_attention(q, k_cache, v_cache, block_table, total)                                                 # every layer

A cache is a pair of tensors [pages, page size, kv heads, head dim] (any order of the first three in memory, so also
`torch.empty(pages, kv_heads, page_size, head_dim).transpose(1, 2)`), dense and 16-byte aligned along the last dimension.  Lengths,
tables, slots and positions stay on the GPU: no call synchronises, and a captured call reads their values at each replay.
None of the operators has a derivative; they refuse inputs that require one.
"""
from __future__ import annotations

import torch

from .ops import PAGED_ATTENTION, PLAN_PAGES, QK_NORM_ROPE, QK_NORM_ROPE_STORE


def qk_norm_rope(qkv: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, num_heads: int, num_kv_heads: int, *,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                 interleaved: bool = False, factor: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotated queries [tokens, num_heads, D] and keys [tokens, num_kv_heads, D] of a merged projection's output `qkv`
    [tokens, (num_heads + 2 * num_kv_heads) * D].

    positions: int32 or int64 [tokens].  inv_freq: float32 [R / 2], R <= D: pair i of a head turns by position * inv_freq[i] (formed
    and reduced in 64 bits); pairs are (i, i + R / 2), or (2i, 2i + 1) if `interleaved`; values from R on are not turned.
    `factor` multiplies the rotated values (the attention factor of scaled rotations).  With q_weight / k_weight [D] (float32 or
    qkv's type) the head is first divided by sqrt(mean of squares + eps) and multiplied by the weight.  fp32 throughout, one
    rounding at the end.  D: even, up to 512."""
    return QK_NORM_ROPE(qkv, positions, inv_freq, num_heads, num_kv_heads, q_weight, k_weight, eps, interleaved, factor)


def qk_norm_rope_store(qkv: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, num_heads: int, k_cache: torch.Tensor,
                       v_cache: torch.Tensor, slots: torch.Tensor, *, q_weight: torch.Tensor | None = None,
                       k_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False,
                       factor: float = 1.0) -> torch.Tensor:
    """`qk_norm_rope` that returns the queries and writes the rotated keys and the values of token t into slot slots[t] of the caches
    (slot = page * page size + place; int32 or int64; a slot outside the cache, -1 for instance, is skipped).  Slots should be
    distinct: one that is named twice holds values of either token.  The caches must not overlap each other or qkv."""
    return QK_NORM_ROPE_STORE(qkv, positions, inv_freq, num_heads, k_cache, v_cache, slots, q_weight, k_weight, eps, interleaved, factor)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, *,
                    scale: float | None = None, window: int = 0, softcap: float = 0.0, return_lse: bool = False):
    """Attention of one token per sequence, q [batch, heads, D], over the first seq_lens[b] cached tokens (the last `window` of them
    if window > 0): [batch, heads, D], and with return_lse the fp32 log of the sum of exponentials [batch, heads].

    scale (positive): 1 / sqrt(D) by default.  softcap > 0: scores become softcap * tanh(score / softcap).  block_table int32 [batch, pages]:
    token j of sequence b is place j % page size of page block_table[b, j // page size]; entries outside the cache count as absent.
    A sequence without visible tokens gives zeros (lse -inf).  The token's own key has to be in the cache
    (`qk_norm_rope_store` first) and counted in seq_lens.  D: a multiple of 16 up to 256; float32, float16 or bfloat16.

    Scores, the softmax's maximum and sums and the sums of the values are fp32; for 16-bit types the weights enter the product with the
    values with 22 (float16) or 17 bits (bfloat16).  A visible value that is not finite spoils its column of the output: for 16-bit types
    an infinity too gives NaN.  Keys and values that no sequence sees may hold anything."""
    out, lse = PAGED_ATTENTION(q, k_cache, v_cache, block_table, seq_lens, q.shape[-1] ** -0.5 if scale is None else scale, window, softcap,
                               return_lse)
    return (out, lse) if return_lse else out


def plan_pages(block_table: torch.Tensor, seq_lens: torch.Tensor, new_lens: torch.Tensor, free_pages: torch.Tensor, taken: torch.Tensor,
               page_size: int, num_tokens: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Room in the cache for new_lens[r] more tokens of each request: (total_lens [R], starts [R + 1], positions [num_tokens], slots
    [num_tokens] int64, taken [1]); everything else int32.

    Request r holds ceil(seq_lens[r] / page_size) pages, named in its row of block_table [R, pages]; what it needs more is taken from
    free_pages in the order of the requests, from index taken[0] on, and entered into block_table in place.  `taken` comes back
    raised by the pages asked for; above len(free_pages) the list has run out and the tokens concerned have slot -1, as have
    tokens beyond the table's width and the padding behind the last of the num_tokens entries.  num_tokens must be at least
    the sum of new_lens."""
    return PLAN_PAGES(block_table, seq_lens, new_lens, free_pages, taken, page_size, num_tokens)


class StepAttention:
    """The attention of a decode step of `sharded.DecoderStack`: one new token for each of m sequences over paged caches.

    caches: per layer a pair (k_cache, v_cache) [pages, page size, kv heads, head dim].  block_table int32 [m, pages per sequence],
    seq_lens int32 [m] (tokens in the caches), free_pages int32 and taken int32 [1] are the program's own tensors; every step moves
    them on in place, so a captured step does so at each replay.  q_weights / k_weights: per layer the norm weights of queries and
    keys, or None.  The other arguments are those of `qk_norm_rope_store` and `paged_attention`.

    A sequence whose row of block_table is full, or for which free_pages has run out, has no place for its new token: seq_lens counts
    it, but its key and value are in no cache, and the outputs from then on are without it.  A step cannot stop for that (it does not
    look at the GPU's values), so `dropped` [m] turns to -1 for such a sequence and stays so, and `check` raises.  A program that has
    dealt with it (ended the sequence, or started it again with more pages) sets its entry of `dropped` back to 0."""

    def __init__(self, caches, num_heads: int, inv_freq: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                 free_pages: torch.Tensor, taken: torch.Tensor, *, q_weights=None, k_weights=None, eps: float = 1e-6,
                 interleaved: bool = False, factor: float = 1.0, scale: float | None = None, window: int = 0, softcap: float = 0.0):
        self.caches = [tuple(pair) for pair in caches]
        if not self.caches or any(k.shape != self.caches[0][0].shape or v.shape != k.shape for k, v in self.caches):
            raise ValueError("caches must be pairs of tensors of one shape, one pair per layer")
        for name, w in (("q_weights", q_weights), ("k_weights", k_weights)):
            if w is not None and len(w) != len(self.caches):
                raise ValueError(f"{name} must hold one tensor per layer")
        self.num_heads, self.inv_freq = num_heads, inv_freq
        self.page_size, self.num_kv_heads, self.head_dim = self.caches[0][0].shape[1:]
        self.block_table, self.seq_lens, self.free_pages, self.taken = block_table, seq_lens, free_pages, taken
        self.q_weights, self.k_weights = (w if w is not None else [None] * len(self.caches) for w in (q_weights, k_weights))
        self.eps, self.interleaved, self.factor, self.scale, self.window, self.softcap = eps, interleaved, factor, scale, window, softcap
        self.one_each = torch.ones_like(seq_lens)
        with torch.inference_mode(False):                # steps may write it in or outside of that mode
            self.dropped = torch.zeros_like(seq_lens, dtype=torch.int64)
        self.positions = self.slots = None

    def begin_step(self) -> None:
        """Room for one more token of every sequence; seq_lens counts it from here on."""
        total, _, self.positions, self.slots, taken = plan_pages(self.block_table, self.seq_lens, self.one_each, self.free_pages, self.taken,
                                                                 self.page_size, self.seq_lens.shape[0])
        self.seq_lens.copy_(total)
        self.taken.copy_(taken)
        torch.minimum(self.dropped, self.slots, out=self.dropped)       # a slot is -1 where there is no page

    def check(self) -> None:
        """Synchronises; raises if a sequence has had no room for a token, or if a bounded wait inside `paged_attention` ran out on this
        device (its outputs are then undefined)."""
        from . import capi

        status = capi.paged_attention_status(device=self.seq_lens.device)
        if status:
            raise RuntimeError(f"paged attention: kernel status {status} (a bounded wait ran out)")
        lost = self.dropped.nonzero().flatten().tolist()
        if lost:
            raise RuntimeError(f"no page for new tokens of the sequences {lost}: their rows of block_table are full, or free_pages has run out")

    def layer(self, index: int, qkv: torch.Tensor) -> torch.Tensor:
        """The attention output [m, num_heads * head dim] of layer `index` for this step's merged projection."""
        k_cache, v_cache = self.caches[index]
        q = qk_norm_rope_store(qkv, self.positions, self.inv_freq, self.num_heads, k_cache, v_cache, self.slots, q_weight=self.q_weights[index],
                               k_weight=self.k_weights[index], eps=self.eps, interleaved=self.interleaved, factor=self.factor)
        out = paged_attention(q, k_cache, v_cache, self.block_table, self.seq_lens, scale=self.scale, window=self.window, softcap=self.softcap)
        return out.flatten(1)
