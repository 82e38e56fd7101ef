"""Paged key/value cache of a decoder stack (SharqDecoder.new_cache), for ops.rope_append_paged and ops.paged_attention.

The reference leaves the cache to HuggingFace's layers (model/qLlamaLayer.py:143-160).  Pages of `page_size` tokens are handed out as
sequences grow, so a batch of short and long sequences takes the memory of its tokens; a cache of torch.float8_e4m3fn values takes half of it.
The page numbers and lengths are kept on the host, where pages are handed out, and on the device, where the kernels read them.  With on_device they
are handed out there too (ops.plan_paged_step), and the host knows none of them: a captured decode step then grows its sequences by itself.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import ops


@dataclass
class LayerCache:
    """What one layer's attention needs for one step.  lengths is None while prompts are appended: their attention reads the prompt."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor]
    v_scale: Optional[torch.Tensor]
    table: torch.Tensor
    positions: torch.Tensor
    sequences: Optional[torch.Tensor]
    lengths: Optional[torch.Tensor]
    cos: torch.Tensor
    sin: torch.Tensor


class PagedKVCache:
    def __init__(self, layers: int, kv_heads: int, head_dim: int, sequences: int, max_tokens: int, cos: torch.Tensor, sin: torch.Tensor,
                 page_size: int = 64, pages: Optional[int] = None, dtype: torch.dtype = torch.bfloat16,
                 k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None, on_device: bool = False):
        """Room for `sequences` sequences of up to max_tokens tokens in `pages` pages (default: enough for all of them).  cos, sin:
        rotary tables [>= max_tokens, head_dim].  k_scale, v_scale: float32 [layers, kv_heads] of a float8_e4m3fn cache, default 1.
        on_device: pages are handed out by plan(), not by reserve() and advance()."""
        if min(layers, kv_heads, head_dim, sequences, max_tokens, page_size) < 1:
            raise ValueError("sizes of the cache must be positive")
        if cos.shape[0] < max_tokens or cos.shape != sin.shape or cos.shape[1] != head_dim:
            raise ValueError("the rotary tables must be shaped [>= max_tokens, head_dim]")
        if dtype not in (torch.bfloat16, torch.float8_e4m3fn):
            raise ValueError(f"a cache holds torch.bfloat16 or torch.float8_e4m3fn, not {dtype}")
        if dtype == torch.bfloat16 and (k_scale is not None or v_scale is not None):
            raise ValueError("k_scale and v_scale belong to a torch.float8_e4m3fn cache")
        self.max_tokens, self.page_size, self.sequences, self.on_device = max_tokens, page_size, sequences, on_device
        most = -(-max_tokens // page_size)
        pages = sequences * most if pages is None else pages
        device = cos.device
        self.k = torch.empty((layers, pages, kv_heads, page_size, head_dim), dtype=dtype, device=device)
        self.v = torch.empty_like(self.k)
        self.k_scale = self.v_scale = None
        if dtype == torch.float8_e4m3fn:
            given = [torch.ones((layers, kv_heads)) if s is None else s for s in (k_scale, v_scale)]
            if any(tuple(s.shape) != (layers, kv_heads) for s in given):
                raise ValueError("k_scale and v_scale must be shaped [layers, kv_heads]")
            self.k_scale, self.v_scale = (s.to(device, torch.float32).contiguous() for s in given)
        self.cos, self.sin = cos, sin
        self.table = torch.zeros((sequences, most), dtype=torch.int32, device=device)
        self.lengths = [0] * sequences
        self.device_lengths = torch.zeros(sequences, dtype=torch.int32, device=device)
        self._held: list[list[int]] = [[] for _ in range(sequences)]
        self._free = list(range(pages - 1, -1, -1))
        if on_device:
            self.lengths = None
            self.free_pages = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device)
            self.free_count = torch.full((1,), pages, dtype=torch.int32, device=device)

    def plan(self, counts: torch.Tensor, rows: int, released: Optional[torch.Tensor] = None):
        """counts[i] (int32, on the device) more tokens for every sequence i, which with released (bool) gives back what it holds first ->
        (offsets, positions, sequences) of the `rows` rows of the step, see ops.plan_paged_step.  Where the pages do not suffice, which reserve() raises,
        check_device_errors does."""
        if not self.on_device:
            raise RuntimeError("the pages of this cache are handed out on the host: reserve() and advance()")
        if released is not None:  # what waited for its prompt (length -1) holds nothing
            self.device_lengths.masked_fill_(released.bool() & (self.device_lengths == -1), 0)
        return ops.plan_paged_step(self.table, self.device_lengths, counts, self.free_pages, self.free_count, self.page_size, rows, released,
                                   self.max_tokens, strict=True)

    def step_places(self, which: Sequence[int], tokens: int, restart: bool = False):
        """plan() of `tokens` new tokens of every sequence in `which` -> (positions, sequences), int32, in the order of `which`.  restart: they begin anew, and
        those for which the pages do not suffice are left with length -1: no token is taken for them until they begin anew once more, or are freed."""
        device, everyone = self.table.device, list(which) == list(range(self.sequences))
        if everyone:
            chosen = torch.ones(self.sequences, dtype=torch.int32, device=device)
        else:
            at = torch.tensor(list(which), device=device)
            chosen = torch.zeros(self.sequences, dtype=torch.int32, device=device).index_fill_(0, at, 1)
        offsets, positions, sequences = self.plan(chosen * tokens, len(which) * tokens, chosen.bool() if restart else None)
        if restart and tokens > 0:
            self.device_lengths.masked_fill_(chosen.bool() & (self.device_lengths == 0), -1)
        if list(which) != sorted(which):
            row = (offsets[at][:, None] + torch.arange(tokens, device=device)).reshape(-1)
            positions, sequences = positions[row], sequences[row]
        return positions, sequences

    def _by_host(self) -> None:
        if self.on_device:
            raise RuntimeError("the pages of this cache are handed out on the device: plan()")

    def reserve(self, counts: Sequence[int]) -> None:
        """Pages for counts[i] more tokens of sequence i.  Raises RuntimeError, and changes nothing, where a sequence would pass
        max_tokens or the pages do not suffice."""
        self._by_host()
        if len(counts) != self.sequences or min(counts) < 0:
            raise ValueError("one count of tokens per sequence")
        want = [n + more for n, more in zip(self.lengths, counts)]
        if max(want) > self.max_tokens:
            raise RuntimeError(f"a sequence of {max(want)} tokens does not fit a cache of {self.max_tokens} per sequence")
        need = [max(0, -(-n // self.page_size) - len(held)) for n, held in zip(want, self._held)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"the cache has {len(self._free)} free pages, {sum(need)} are needed")
        for i, n in enumerate(need):
            if n:
                new = [self._free.pop() for _ in range(n)]
                at = len(self._held[i])
                self._held[i] += new
                self.table[i, at:at + n] = torch.tensor(new, dtype=torch.int32, device=self.table.device)

    def advance(self, counts: Sequence[int]) -> None:
        """The tokens that were reserved and appended now belong to their sequences."""
        self._by_host()
        if len(counts) != self.sequences or any(n + more > len(held) * self.page_size for n, more, held in zip(self.lengths, counts, self._held)):
            raise ValueError("tokens must be reserved before they are counted")
        self.lengths = [n + more for n, more in zip(self.lengths, counts)]
        if len(set(counts)) == 1:
            self.device_lengths += counts[0]
        else:
            self.device_lengths += torch.tensor(list(counts), dtype=torch.int32, device=self.table.device)

    def free(self, sequence: int) -> None:
        """Gives the pages of a sequence back; it is empty then, and another prompt may take its place (SharqDecoder.prefill with sequences)."""
        if self.on_device:
            ended = torch.zeros(self.sequences, dtype=torch.int32, device=self.table.device)
            ended[range(self.sequences)[sequence]] = 1  # a number outside is an IndexError here, too
            self.plan(torch.zeros_like(ended), 0, ended.bool())
            return
        self._free += reversed(self._held[sequence])
        self._held[sequence] = []
        self.lengths[sequence] = 0
        self.device_lengths[sequence] = 0

    def chosen(self, sequences: Optional[Sequence[int]]) -> list[int]:
        """The sequences that a step is for: all of them, or those listed, each once."""
        which = list(range(self.sequences)) if sequences is None else [int(i) for i in sequences]
        if not which or len(set(which)) != len(which) or not all(0 <= i < self.sequences for i in which):
            raise ValueError(f"sequences must be different numbers below {self.sequences}, got {which}")
        return which

    def counts(self, which: Sequence[int], tokens: int) -> list[int]:
        """For reserve and advance: `tokens` of every sequence in `which`, none of the others."""
        listed = set(which)
        return [tokens if i in listed else 0 for i in range(self.sequences)]

    def prompt_step(self, tokens: int, sequences: Optional[Sequence[int]] = None):
        """(positions, sequences) int32 of `tokens` new tokens of every sequence, or of those listed, sequence after sequence."""
        self._by_host()
        device = self.table.device
        first, which = self.device_lengths, torch.arange(self.sequences, dtype=torch.int32, device=device)
        if sequences is not None:
            which = torch.tensor(self.chosen(sequences), dtype=torch.int32, device=device)
            first = first[which.long()]
        positions = (first[:, None] + torch.arange(tokens, dtype=torch.int32, device=device)).reshape(-1)
        return positions, which.repeat_interleave(tokens)

    def held_table(self, rows: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The page table cut to what the longest sequence holds, as far as the host knows, of all sequences or of those in rows (int64, device).  A row of no
        sequence has no pages, which the kernels report."""
        table = self.table if self.on_device else self.table[:, :max(1, max(len(h) for h in self._held))]
        if rows is None:
            return table
        there = (rows >= 0) & (rows < self.sequences)
        return torch.where(there[:, None], table[rows.clamp(0, self.sequences - 1)], -1)

    def layer(self, index: int, positions: torch.Tensor, sequences: Optional[torch.Tensor], lengths: Optional[torch.Tensor],
              table: Optional[torch.Tensor] = None) -> LayerCache:
        """Layer `index` for a step.  table: the rows of the page table that belong to the step's rows, default held_table()."""
        return LayerCache(self.k[index], self.v[index], None if self.k_scale is None else self.k_scale[index],
                          None if self.v_scale is None else self.v_scale[index], self.held_table() if table is None else table, positions,
                          sequences, lengths, self.cos, self.sin)
