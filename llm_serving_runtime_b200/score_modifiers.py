"""Changed attention scores for ``paged_attention_decode`` (``pa_decode_ext``).

    mods = ScoreModifiers(softcap=50.0, window=4096)
    out = paged_attention_decode(query, k_cache, v_cache, block_tables, context_lens,
                                 scale, score_modifiers=mods)

For the query token at position i (``context_lens[b] + t``) and the key at j:

* ``softcap``       s = softcap * tanh(s / softcap), applied to s = scale * q.k
* ``alibi_slopes``  float32 [num_q_heads]: s -= slope[h] * |i - j|, after the cap
* ``window``        keys with i - j >= window are hidden (a window of 1: itself)
* ``key_starts``    int32 [batch, q_len] or [batch]: keys before it are hidden,
                    e.g. the start of the token's document in a packed sequence
* ``prefix_lens``   int32 [batch]: keys before it are seen by every token of the
                    row, also by earlier ones (a prefix language model)

All of them may be given together; the masks intersect, except that a prefix
lifts the causal limit.  A token that sees no key gets a zero row.  What a token
does not see cannot reach its row (not even as NaN), and blocks before the first
key that any of a sequence's tokens sees are never read, so a sliding window's old
blocks may be recycled while their table entries stay.

The tensors are read on the device at the call (at the replay, in a captured
graph), so they may be rewritten in place between steps.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib

__all__ = ["ScoreModifiers"]


@dataclass
class ScoreModifiers:
    softcap: float = 0.0
    window: int = 0
    alibi_slopes: torch.Tensor | None = None
    key_starts: torch.Tensor | None = None
    prefix_lens: torch.Tensor | None = None

    def to_args(self, batch: int, num_q_heads: int, q_len: int, device: torch.device) -> _lib.ScoreModifiersArgs:
        """The C arguments for a call of this shape; ValueError where they do not fit it."""
        a = _lib.ScoreModifiersArgs()
        if self.softcap != 0.0 and not 1e-30 < self.softcap < 1e30:
            raise ValueError(f"softcap must be 0 (none) or in (1e-30, 1e30), got {self.softcap}")
        if not 0 <= self.window < 2**31:
            raise ValueError(f"window must be 0 (none) or positive, got {self.window}")
        a.softcap, a.window = float(self.softcap), int(self.window)
        if self.alibi_slopes is not None:
            s = self.alibi_slopes
            if s.dtype != torch.float32 or tuple(s.shape) != (num_q_heads,) or s.device != device \
                    or not s.is_contiguous():
                raise ValueError(f"alibi_slopes must be a contiguous float32 [num_q_heads={num_q_heads}] on {device}")
            a.alibi_slopes = s.data_ptr()
        if self.key_starts is not None:
            k = self.key_starts
            if k.dtype != torch.int32 or k.device != device or tuple(k.shape) not in ((batch,), (batch, q_len)):
                raise ValueError(f"key_starts must be int32 [batch={batch}] or [batch, q_len={q_len}] on {device}")
            a.key_starts = k.data_ptr()
            a.key_starts_stride_b = k.stride(0)
            a.key_starts_stride_t = k.stride(1) if k.dim() == 2 else 0
        if self.prefix_lens is not None:
            p = self.prefix_lens
            if p.dtype != torch.int32 or tuple(p.shape) != (batch,) or p.device != device or not p.is_contiguous():
                raise ValueError(f"prefix_lens must be a contiguous int32 [batch={batch}] on {device}")
            a.prefix_lens = p.data_ptr()
        return a

    def astuple(self) -> tuple:
        return self.softcap, self.window, self.alibi_slopes, self.key_starts, self.prefix_lens

    def rows(self, lo: int, hi: int) -> "ScoreModifiers":
        """The modifiers of batch rows [lo, hi)."""
        return ScoreModifiers(
            softcap=self.softcap, window=self.window, alibi_slopes=self.alibi_slopes,
            key_starts=None if self.key_starts is None else self.key_starts[lo:hi],
            prefix_lens=None if self.prefix_lens is None else self.prefix_lens[lo:hi],
        )
