"""KV cache in pages that sequences share (no counterpart in the reference, whose cache is one contiguous
slice per batch row: packages/model-utils/src/kv-cache.ts:92-309).

All layers' keys and values live in one pool [layers, 2, pages, kv heads, page size, head dim]; a page table
says which pages each of up to max_sequences rows holds, in which order, and a reference count per page how
many entries hold it.  Rows grow (reserve), take over other rows' pages (fork: beams, or an answer forked off a
prompt) and give theirs back (free) by device kernels that only touch the table and the counts; a page is
copied when a row grows into one that others hold, too, and when the pool is compacted.

The host keeps each row's length in step, so that a call that does not fit is refused before anything is
enqueued; whether enough pages are free is known on the device, and read back by reserve(check=True).
"""
from __future__ import annotations

from typing import Optional, Sequence

import numpy as np

from .. import functional as F
from ..tensor import Tensor


class PagedKVCache:
    def __init__(self, num_layers: int, num_kv_heads: int, head_dim: int, num_pages: int, max_sequences: int,
                 max_seq_len: int, page_size: int = 16, dtype: str = "bfloat16"):
        if num_pages < 1 or max_sequences < 1 or max_seq_len < 1:
            raise ValueError(f"PagedKVCache: {num_pages} pages, {max_sequences} sequences of {max_seq_len} rows")
        if max_sequences > 2048 or max_seq_len > 1 << 30:
            raise ValueError(f"PagedKVCache: {max_sequences} sequences of {max_seq_len} rows, at most 2048 of 2^30")
        if page_size < 16 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError(f"PagedKVCache: page size {page_size} is not a power of two from 16 to 4096")
        self.num_layers, self.page_size, self.num_pages = num_layers, page_size, num_pages
        self.max_sequences, self.max_seq_len = max_sequences, max_seq_len
        self.width = -(-max_seq_len // page_size)
        self.pages = F.zeros((num_layers, 2, num_pages, num_kv_heads, page_size, head_dim), dtype)
        pool = (num_pages, num_kv_heads, page_size, head_dim)
        self._pools = []
        for i in range(num_layers):
            both = F.narrow(self.pages, 0, i, 1)
            k, v = F.narrow(both, 1, 0, 1), F.narrow(both, 1, 1, 1)
            self._pools.append((F.view(k, pool), F.view(v, pool)))
            for t in (both, k, v):
                t.dispose()
        # the state, and a second set that fork and compact write to: they change places
        self.state = self._new_state()
        self._other = self._new_state()
        self.lens = np.zeros(max_sequences, np.int64)
        self._unchecked = 0   # reserves whose success the host has not looked at
        self._moves = F.zeros((max_sequences, 2), "int32")
        self._info = F.zeros((3,), "int32")

    def _new_state(self):
        table = Tensor(np.full((self.max_sequences, self.width), -1, np.int32), dtype="int32")
        return table, F.zeros((self.max_sequences,), "int32"), F.zeros((self.num_pages,), "int32")

    @property
    def page_table(self) -> Tensor:
        return self.state[0]

    @property
    def kv_lens(self) -> Tensor:
        return self.state[1]

    @property
    def page_refs(self) -> Tensor:
        return self.state[2]

    @property
    def reserve_info(self) -> Tensor:
        """What the last reserve has left (int32 [3], on the device), for paged_kv_write: a step that lacked pages then
        writes nothing over the cached rows."""
        return self._info

    def layer(self, i: int):
        """(keys, values) of layer i: its two pools [pages, kv heads, page size, head dim]."""
        return self._pools[i]

    def free_pages(self) -> int:
        """Pages that no row holds (waits for the device)."""
        return int((self.page_refs.numpy() <= 0).sum())

    def _check_counts(self, counts) -> np.ndarray:
        n = np.asarray(counts, np.int64).reshape(-1)
        if n.shape != self.lens.shape or (n < 0).any():
            raise ValueError(f"PagedKVCache: counts must be {self.max_sequences} numbers of new rows, got {list(np.shape(counts))}")
        over = np.flatnonzero(self.lens + n > self.max_seq_len)
        if len(over):
            raise ValueError(f"Cache overflow: sequence {over[0]} has {self.lens[over[0]]} rows and {n[over[0]]} new ones, "
                             f"but maxSeqLen is {self.max_seq_len}")
        return n

    def enqueue_reserve(self, counts: Tensor) -> None:
        """reserve() for counts on the device (int32 [max_sequences]) and without the host's part: for a captured step,
        whose caller advances `lens` at each replay, hands reserve_info to paged_kv_write, and asks check_info() after each
        replay whether the pages sufficed."""
        F.pages_reserve(*self.state, counts, self.page_size, out=(self._moves, self._info))
        F.pages_copy(self.pages, self._moves, self._info)

    def check_info(self) -> None:
        """Raises if the last reserve lacked pages, or one before it that reserve(check=False) left unchecked (waits for
        the device).  `lens` are then the device's: a reserve that lacked pages has changed nothing."""
        _, missing, too_long = self._info.numpy().tolist()
        unchecked, self._unchecked = self._unchecked, 0
        if not missing and not too_long and unchecked < 2:
            return
        lens = self.kv_lens.numpy().astype(np.int64)   # (info speaks of the last reserve alone)
        same, self.lens = np.array_equal(lens, self.lens), lens
        if missing:
            raise RuntimeError(f"PagedKVCache: {missing} pages are missing ({self.num_pages} of {self.page_size} rows in all)")
        if too_long:
            raise RuntimeError(f"PagedKVCache: {too_long} rows are too long for the page table")
        if not same:
            raise RuntimeError(f"PagedKVCache: pages were missing for a reserve before the last ({self.num_pages} of "
                               f"{self.page_size} rows in all)")

    def reserve(self, counts: Sequence[int], check: bool = True) -> None:
        """Makes room for counts[s] new rows behind each sequence's cached ones, which kv_lens then includes.  Pages
        that a sequence grows into are its own afterwards.  check: raise if the pool has too few free pages (nothing
        has changed then); without it the caller hands reserve_info to what it enqueues (paged_kv_write) and calls
        check_info() later, until which `lens` counts on the pages."""
        if check and self._unchecked:
            self.check_info()   # before anything is enqueued behind it
        n = self._check_counts(counts)
        t = Tensor(n.astype(np.int32), dtype="int32")
        self.enqueue_reserve(t)
        t.dispose()
        self.lens += n
        self._unchecked += 1
        if check:
            self.check_info()

    def enqueue_fork(self, parents: Tensor) -> None:
        """fork() for parents on the device, without the host's part."""
        F.pages_fork(*self.state, parents, out=self._other)
        self.state, self._other = self._other, self.state

    def fork(self, parents: Sequence[int]) -> None:
        """Sequence s takes over the rows of sequence parents[s] (itself: unchanged; -1: none, its pages are given
        back).  Rows are shared, not copied."""
        p = np.asarray(parents, np.int64).reshape(-1)
        if p.shape != self.lens.shape or (p < -1).any() or (p >= self.max_sequences).any():
            raise ValueError(f"PagedKVCache: parents must be {self.max_sequences} sequence numbers or -1")
        t = Tensor(p.astype(np.int32), dtype="int32")
        self.enqueue_fork(t)
        t.dispose()
        self.lens = np.where(p < 0, 0, self.lens[p])

    def free(self, sequences: Sequence[int]) -> None:
        """Gives back the pages of these sequences."""
        s = np.asarray(list(sequences), np.int64)
        if (s < 0).any() or (s >= self.max_sequences).any():
            raise ValueError(f"PagedKVCache: sequences outside [0, {self.max_sequences})")
        parents = np.arange(self.max_sequences)
        parents[s] = -1
        self.fork(parents)

    def reset(self) -> None:
        self.free(range(self.max_sequences))

    def compact(self) -> int:
        """Moves the pages in use to the front of the pool; returns how many there are (waits for the device)."""
        table, _, refs = self.state
        o_table, o_lens, o_refs = self._other
        _, _, moves, info = F.pages_compact(table, refs, out=(o_table, o_refs, *self._compact_out()))
        F.pages_copy(self.pages, moves, info)
        F.copy_(o_lens, self.kv_lens)
        self.state, self._other = self._other, self.state
        live = int(info.numpy()[1])
        moves.dispose()
        info.dispose()
        return live

    def _compact_out(self):
        return F.zeros((max(1, self.num_pages // 2), 2), "int32"), F.zeros((2,), "int32")

    def dispose(self) -> None:
        for k, v in self._pools:
            k.dispose()
            v.dispose()
        self._pools = []
        for t in (*self.state, *self._other, self._moves, self._info, self.pages):
            t.dispose()
