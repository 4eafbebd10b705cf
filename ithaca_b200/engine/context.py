"""What one step tells the kernels: which tokens, whose they are, where they sit.

All of it is small int32 data.  It is assembled on the host into one pinned
buffer and reaches the device in one copy; the fields below are views of that
device buffer.  Positions are implied by the cache: token k of a sequence sits at
the sequence's length before the step plus k.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch


@dataclass
class StepContext:
    n_tokens: int
    n_seqs: int
    n_logit_rows: int
    token_ids: torch.Tensor            # [T]
    token_seq: torch.Tensor            # [T] index of the token's sequence in this step
    token_pos: torch.Tensor            # [T] absolute position
    cu_seqlens: torch.Tensor           # [B + 1] first token of each sequence
    slots: torch.Tensor                # [B]
    kv_lens: torch.Tensor              # [B] positions each sequence holds after this step
    logit_rows: torch.Tensor           # [R] token indices whose logits are wanted
    tables: List[torch.Tensor]         # per key/value group: [B, pages] block table
    is_decode: bool                    # every sequence brings exactly one token
    max_new: int
    max_kv_len: int
    kv_len_bound: int = 0              # no sequence is longer than this (sizes grids; >= max_kv_len)
    replayed: bool = False             # captured, and replayed for other lengths than this step's: only the bound counts
    host_slots: List[int] = field(default_factory=list)
    host_n_new: List[int] = field(default_factory=list)
    host_kv_lens: List[int] = field(default_factory=list)
    shared: dict = field(default_factory=dict)     # what the layers of one step compute once and share (rotary tables)
    sharing: List[Optional["Sharing"]] = field(default_factory=list)     # per key/value group: who shares pages (decode steps of forked sequences; else empty)


@dataclass
class Sharing:
    """Neighbouring sequences of a decode step that share their first pages: group i are the sequences starts[i] <= b < starts[i + 1]."""
    starts: List[int]
    pages: List[int]                   # per sequence: pages it shares with its whole group
    shared_bound: int                  # the most pages a group shares
    own_bound: int                     # the most pages a sequence has to itself
    most: int = 0                      # no group is larger
    starts_dev: Optional[torch.Tensor] = None
    pages_dev: Optional[torch.Tensor] = None

    @property
    def n_groups(self) -> int:
        return len(self.starts) - 1

    @property
    def max_members(self) -> int:
        return self.most

    def pad(self, n_groups: int) -> None:
        """Empty groups behind the others, until there are so many."""
        self.starts += [self.starts[-1]] * (n_groups - self.n_groups)


def find_sharing(table: np.ndarray, n_pages: Sequence[int]) -> Optional[Sharing]:
    """``table`` [B, columns]: the block table of a decode step's sequences, ``n_pages``: how many pages each has.  The same page in the same column of
    neighbouring rows is shared (and full).  Cuts the rows into groups so that the most page readings are saved: m rows that have s first pages in
    common save (m - 1) s.  None if nothing is shared."""
    B = table.shape[0]
    if B < 2:
        return None
    other = (table[1:] != table[:-1]) | (table[1:] < 0)
    first = other.argmax(axis=1)                                   # 0 where there is none, too
    common = np.where(other[np.arange(B - 1), first], first, table.shape[1])
    if not common.any():
        return None
    starts, pages, lo, common = [], [], 0, common.tolist() + [0]
    for hi, c in enumerate(common, 1):
        if c:
            continue
        # rows lo .. hi - 1 are a run whose neighbours all have pages in common
        for a, b, s in _cut_run(common[lo:hi - 1]):
            starts.append(lo + a)
            pages += [s] * (b - a)
        lo = hi
    starts.append(B)
    return Sharing(starts, pages, max(pages), max(n - s for n, s in zip(n_pages, pages)), max(b - a for a, b in zip(starts, starts[1:])))


def _cut_run(c: List[int]) -> List[Tuple[int, int, int]]:
    """``c``: the pages that each of a run's len(c) + 1 rows has in common with the next.  The groups (first row, row behind the last, pages in common) that save
    the most; of equal ways the larger group."""
    m = len(c) + 1
    if len(set(c)) < 2:
        return [(0, m, c[0] if c else 0)]
    # What a cut within a stretch of equal numbers saves is linear in where it lies: only its two ends need looking at
    at = [0] + [j for j in range(1, m) if j == 1 or j == m - 1 or c[j - 1] != c[j - 2] or c[j - 1] != c[j]] + [m]
    least = [min(c[i:j]) if j < m else 0 for i, j in zip(at, at[1:])]                   # of the rows between two of them, with the cut's own
    best, cuts = [0], [(0, 0)]
    for y in range(1, len(at)):
        most, cut, low = best[y - 1], (y - 1, 0), 0
        if at[y] - at[y - 1] > 1:
            low = min(c[at[y - 1]:at[y] - 1])
            most, cut = most + (at[y] - at[y - 1] - 1) * low, (y - 1, low)
        for x in range(y - 2, -1, -1):
            low = min(low or least[x], least[x])
            gain = best[x] + (at[y] - at[x] - 1) * low
            if gain >= most:
                most, cut = gain, (x, low)
        best.append(most)
        cuts.append(cut)
    groups, y = [], len(at) - 1
    while y:
        x, low = cuts[y]
        groups.append((at[x], at[y], low))
        y = x
    return groups[::-1]


def field_offsets(sizes):
    """Where each field of a step's description starts in the packed int32 buffer: every field on a
    16-byte boundary.  Returns (offsets, sizes, total length)."""
    offs, total = [], 0
    for n in sizes:
        offs.append(total)
        total += (n + 3) // 4 * 4
    return offs, list(sizes), max(total, 4)


class ContextBuilder:
    """Reusable pinned staging so that a step costs one host-to-device copy."""

    def __init__(self, device: str):
        self.device = device
        self.last_upload_bytes = 0
        self._pinned: Optional[torch.Tensor] = None
        self._copied: Optional[torch.cuda.Event] = None      # the last upload from the staging buffer

    def _staging(self, n: int) -> torch.Tensor:
        if self._pinned is None or self._pinned.numel() < n:
            cap = max(4096, 1 << (n - 1).bit_length())
            self._pinned = torch.empty(cap, dtype=torch.int32).pin_memory()
        return self._pinned

    def build(self, slots: Sequence[int], tokens: Sequence[Sequence[int]], start: Sequence[int],
              want: Sequence[Sequence[int]], tables: Sequence[np.ndarray],
              into: Optional[torch.Tensor] = None, sharing: Sequence[Optional[Sharing]] = ()) -> StepContext:
        """``start[b]``: positions sequence b holds before the step.  ``tables[g]``: the
        [B, pages] block table of group g (pages already reserved for the new tokens).
        ``into``: a device buffer to fill instead of a fresh one (its layout must be the
        same as at its first use; CUDA graphs replay on it).  ``sharing``: per group, who shares pages."""
        B = len(slots)
        n_new = [len(t) for t in tokens]
        T = int(sum(n_new))
        cu = np.zeros(B + 1, dtype=np.int32)
        cu[1:] = np.cumsum(n_new)
        token_ids = np.fromiter((x for t in tokens for x in t), dtype=np.int32, count=T)
        token_seq = np.repeat(np.arange(B, dtype=np.int32), n_new)
        token_pos = (np.arange(T, dtype=np.int32) - cu[token_seq] + np.asarray(start, dtype=np.int32)[token_seq])
        rows = np.fromiter((cu[b] + w for b in range(B) for w in want[b]), dtype=np.int32)
        kv_lens = np.asarray(start, dtype=np.int32) + np.asarray(n_new, dtype=np.int32)
        parts = [token_ids, token_seq, token_pos, cu, np.asarray(slots, dtype=np.int32), kv_lens, rows]
        parts += [np.ascontiguousarray(t, dtype=np.int32).reshape(-1) for t in tables]
        parts += [np.asarray(x, dtype=np.int32) for s in sharing if s is not None for x in (s.starts, s.pages)]
        offs, sizes, total = field_offsets([p.size for p in parts])
        if self._copied is not None:
            self._copied.synchronize()                        # the staging buffer is free again
        stage = self._staging(total)
        sn = stage.numpy()
        for p, o in zip(parts, offs):
            sn[o:o + p.size] = p
        if into is None:
            dev = torch.empty(total, dtype=torch.int32, device=self.device)
        else:
            if into.numel() < total:
                raise ValueError("the context buffer is too small for this step")
            dev = into
        dev[:total].copy_(stage[:total], non_blocking=True)
        if self._copied is None:
            self._copied = torch.cuda.Event()
        self._copied.record()
        self.last_upload_bytes = total * 4

        def view(i):
            return dev[offs[i]:offs[i] + sizes[i]]

        at = 7 + len(tables)
        for s in sharing:
            if s is not None:
                s.starts_dev, s.pages_dev, at = view(at), view(at + 1), at + 2
        tabs = [view(7 + g).view(B, tables[g].shape[1]) for g in range(len(tables))]
        return StepContext(
            n_tokens=T, n_seqs=B, n_logit_rows=int(rows.size), token_ids=view(0), token_seq=view(1),
            token_pos=view(2), cu_seqlens=view(3), slots=view(4), kv_lens=view(5), logit_rows=view(6), tables=tabs,
            is_decode=all(n == 1 for n in n_new), max_new=max(n_new) if n_new else 0,
            max_kv_len=int(kv_lens.max()) if B else 0, kv_len_bound=int(kv_lens.max()) if B else 0, host_slots=list(slots), host_n_new=n_new,
            host_kv_lens=[int(x) for x in kv_lens], sharing=list(sharing))
