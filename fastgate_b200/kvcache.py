"""Paged key/value cache held in 4 bits: the pool and its bookkeeping around the cache operators.

    cache = KVCacheInt4(num_pages=4096, kv_heads=8, head_dim=128, page_size=64)
    table = rotation_table(max_positions, head_dim)              # cos/sin, fp32
    # one step: q, k, v are column ranges of a fused QKV projection, viewed [tokens, heads, head_dim]
    slots = cache.slots(block_table, sequence_of_token, positions)
    cache.append(k, v, slots, cos_sin=table, positions=positions, q=q)        # q is rotated in place
    cache.attend(q, block_table, seq_lens, out)                  # one new token per sequence
    cache.attend(q, block_table, seq_lens, out, q_starts=starts) # several

Which page belongs to which sequence is the caller's: `block_table` is an int32 tensor [batch, pages], row b
naming the pages of sequence b in order.  Indices that lie on the device are checked by the kernels; `check()`
raises if one was out of range.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _C, capi


def rotation_table(positions: int, head_dim: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """cos_sin [positions, head_dim] fp32 for `append`: the cosines of the head_dim/2 angles p * base^(-2i/head_dim),
    then their sines.  The angles are formed in 64 bits: at far positions 32 bits lose whole digits of them."""
    inv = float(base) ** (-torch.arange(0, head_dim, 2, dtype=torch.float64, device=device) / head_dim)
    a = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], dim=1).float()


class KVCacheInt4:
    """A pool of `num_pages` pages of `page_size` rows (a multiple of 16) for `kv_heads` heads of 64 or 128 channels:
    page_size * (head_dim + 8) bytes per page and head, keys and values together."""

    def __init__(self, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device="cuda"):
        if head_dim not in (64, 128):
            raise ValueError("fastgate_b200: head_dim must be 64 or 128")
        if page_size < 16 or page_size % 16 or page_size > 1 << 20:
            raise ValueError("fastgate_b200: page_size must be a multiple of 16, at most 2^20")
        if num_pages < 1 or kv_heads < 1:
            raise ValueError("fastgate_b200: num_pages and kv_heads must be positive")
        self.page_size, self.kv_heads, self.head_dim = page_size, kv_heads, head_dim
        self.pages = torch.zeros(num_pages, kv_heads, page_size * (head_dim + 8), dtype=torch.uint8, device=device)
        self._status = torch.zeros(1, dtype=torch.int32, device=device)

    def slots(self, block_table: torch.Tensor, sequence: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """Slot of each row: page block_table[sequence, position // page_size], row position % page_size.  A negative
        position (a padding row) gets slot -1; a row that the table has no page for, the slot behind the last one, which
        append and read leave out and check() reports."""
        rows, width = block_table.shape
        if rows == 0 or width == 0:  # no page at all
            return torch.where(positions >= 0, self.pages.shape[0] * self.page_size, -1).long()
        seq, at = sequence.long(), positions.long().clamp(min=0)
        nth = at // self.page_size
        page = block_table[seq.clamp(0, rows - 1), nth.clamp(max=width - 1)].long()
        known = (seq >= 0) & (seq < rows) & (nth < width) & (page >= 0)
        slot = torch.where(known, page * self.page_size + at % self.page_size, self.pages.shape[0] * self.page_size)
        return torch.where(positions >= 0, slot, -1)

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, cos_sin: Optional[torch.Tensor] = None,
               positions: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
               interleaved: bool = False) -> None:
        """Rows k, v [tokens, kv_heads, head_dim] into `slots`; k and q turned by the angles of `positions` first."""
        _C.kv_append_int4(k, v, self.pages, slots, self.page_size, cos_sin, positions, q, q_out, interleaved, self._status)

    def read(self, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """The rows of `slots` as fp16 (rows of negative slots are zeros)."""
        k = torch.zeros(slots.shape[0], self.kv_heads, self.head_dim, dtype=torch.float16, device=self.pages.device)
        v = torch.zeros_like(k)
        _C.kv_read_int4(self.pages, slots, k, v, self.page_size, self._status)
        return k, v

    def attend(self, q: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, out: torch.Tensor,
               q_starts: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> None:
        """out = attention of q [tokens, q_heads, head_dim] over the cached rows of each sequence (see kv_attention_int4)."""
        _C.kv_attention_int4(q, self.pages, block_table, seq_lens, out, self.page_size, q_starts, scale, self._status)

    def check(self) -> None:
        """Raises if a call since the last check, on whatever stream, met an index out of range (waits for the device)."""
        wait = torch.cuda.synchronize if self._status.is_cuda else lambda device: None
        wait(self._status.device)
        status = int(self._status.item())
        if status:
            self._status.zero_()
            wait(self._status.device)  # calls that follow on other streams report into a cleared word
            raise RuntimeError(f"fastgate_b200: {capi.status_str(status)}")
