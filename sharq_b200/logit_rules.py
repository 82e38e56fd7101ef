"""What a decoder's logits go through before a token is chosen (SharqDecoder.prefill and decode with rules), for ops.adjust_logits.

The reference leaves this to HuggingFace's generation loop.  The history is kept on the device, so that a captured decode step goes on from token to token.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import ops


@dataclass
class LogitRules:
    """Penalties, biases and a mask, one row per row of logits; see ops.adjust_logits for their meaning."""
    tokens: Optional[torch.Tensor] = None          # int32 or int64 [rows, width]: every row's history
    lengths: Optional[torch.Tensor] = None         # int32 [rows]
    prompt_lengths: Optional[torch.Tensor] = None  # int32 [rows]
    repetition: Optional[torch.Tensor] = None      # float32 [rows]
    presence: Optional[torch.Tensor] = None
    frequency: Optional[torch.Tensor] = None
    bias: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]] = None  # offsets int32 [rows + 1], ids int32, values float32
    mask: Optional[torch.Tensor] = None            # int32 [rows, ceil(vocab / 32)], a bit per token

    def check_rows(self, rows: int) -> None:
        """Refuses rules of another number of rows, ahead of a step that would have changed its cache when adjust_logits refuses them."""
        held = {name: getattr(self, name) for name in ("tokens", "lengths", "prompt_lengths", "repetition", "presence", "frequency", "mask")}
        for name, t in held.items():
            if t is not None and t.shape[:1] != (rows,):
                raise ValueError(f"{name} of the rules must have a row for each of the {rows} rows of logits, not shape {tuple(t.shape)}")
        if self.bias is not None and self.bias[0].shape != (rows + 1,):
            raise ValueError(f"the biases' offsets must be {rows + 1} for {rows} rows of logits, not shape {tuple(self.bias[0].shape)}")

    def apply_(self, logits: torch.Tensor) -> torch.Tensor:
        """The logits [rows, vocab], changed in place."""
        return ops.adjust_logits(logits, self.tokens, self.lengths, self.prompt_lengths, self.repetition, self.presence, self.frequency, self.bias,
                                 self.mask, out=logits)

    def append_(self, token_ids: torch.Tensor) -> None:
        """One more token [rows] of every history.  Where there is no room the last place is overwritten and the length, which adjust_logits
        reports then, goes on."""
        if self.tokens is None or self.tokens.shape[1] == 0:
            raise ValueError("there is no history to append to")
        at = self.lengths.long().clamp(0, self.tokens.shape[1] - 1)
        self.tokens.scatter_(1, at[:, None], token_ids.to(self.tokens.dtype)[:, None])
        self.lengths += 1
