"""The cache on the device: page pools per group, page tables, fixed-size state.

Layout of one group: keys and values ``[entries, pages, PAGE, n_kv_heads,
head_dim]`` in the compute dtype (the values ``[..., value_dim]`` where a group's
value heads have a size of their own), and one page table ``[slots, max_pages]``
(int32) shared by the group's entries; a group whose values are the leading part of its key
rows (a latent that serves as both) has the one pool.  Position p of the sequence in slot s is
row p % cap; its page is ``page_table[s, row // PAGE]``.  Nothing is cleared
when a slot is reused: every read is bounded by the sequence's length.

With ``kv_dtype`` torch.float8_e4m3fn the groups whose mixers can work from 8-bit codes hold those,
and beside each pool one 32-bit power-of-two scale for each page and kv head: a value is code *
scale.  A window's ring then has a page more than the window takes, so that the page being filled
never holds keys that are still seen and its scale is that of its own tokens alone.  Latent
groups (values that lead the key rows) stay in the compute dtype.

Fixed-size state is ``[entries, slots, numel]`` in 32-bit and is zeroed when a
slot is acquired.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from ..parts.base import KVRequest, StateRequest
from .book import PAGE, CacheBook, CacheError, CacheFull, GroupGeometry, plan_groups, round_up


@dataclass
class KVView:
    """What an attention layer needs to reach its keys and values."""
    k_pool: torch.Tensor          # [pages, PAGE, nkv, hd] of this entry
    v_pool: torch.Tensor
    page_table: torch.Tensor      # [slots, max_pages] int32
    page: int
    cap: int
    window: Optional[int]
    k_scale: Optional[torch.Tensor] = None    # [pages, nkv] float32 of an entry held as codes
    v_scale: Optional[torch.Tensor] = None


@dataclass
class StateView:
    state: torch.Tensor           # [slots, numel] float32 of this entry


class Cache:
    def __init__(self, requests: Sequence[object], max_tokens: int, max_seq_len: int,
                 n_slots: int, dtype: torch.dtype, device: torch.device,
                 kv_dtype: Optional[torch.dtype] = None):
        # an entry asks for keys and values, for fixed-size state, for both (a tuple of the
        # two requests) or for nothing
        self.requests = list(requests)
        self.dtype, self.device = dtype, device

        def pick(r, kind):
            for x in (r if isinstance(r, (tuple, list)) else (r,)):
                if isinstance(x, kind):
                    return x
            return None
        kv_requests = [pick(r, KVRequest) for r in self.requests]
        state_requests = [pick(r, StateRequest) for r in self.requests]
        max_seq_len = max(1, min(max_seq_len, round_up(max_tokens, PAGE)))
        self.max_seq_len = max_seq_len
        self.max_tokens = max_tokens
        if kv_dtype not in (None, dtype, torch.float8_e4m3fn):
            raise CacheError(f"the cache holds the compute dtype ({dtype}) or float8_e4m3fn, not "
                             f"{kv_dtype}")
        groups, self.where = plan_groups(kv_requests, max_tokens, max_seq_len, n_slots,
                                         codes=kv_dtype == torch.float8_e4m3fn)
        if kv_dtype == torch.float8_e4m3fn and not any(g.codes for g in groups):
            raise CacheError("no layer of this model holds keys and values that 8-bit codes can stand "
                             "for")
        self.codes = any(g.codes for g in groups)      # whether any entry is held in 8 bits
        self.book = CacheBook(groups, n_slots, max_seq_len)
        self.n_slots = n_slots
        self.k_pools: List[torch.Tensor] = []
        self.v_pools: List[torch.Tensor] = []
        self.tables: List[torch.Tensor] = []
        self.scales: List[Optional[torch.Tensor]] = []     # [2, entries, pages, nkv], or None
        for g in groups:
            shape = (len(g.entries), g.n_pages, PAGE, g.n_kv_heads)

            def pool(dim):
                if not g.codes:
                    return torch.zeros(shape + (dim,), dtype=dtype, device=device)
                return torch.zeros(shape + (dim,), dtype=torch.uint8, device=device).view(kv_dtype)
            self.k_pools.append(pool(g.head_dim))
            # (a group whose values lead its key rows has one pool under both names)
            self.v_pools.append(self.k_pools[-1] if g.values_in_keys else pool(g.v_dim))
            self.scales.append(torch.ones((2, len(g.entries), g.n_pages, g.n_kv_heads),
                                          dtype=torch.float32, device=device) if g.codes else None)
            self.tables.append(torch.zeros((n_slots, g.max_pages), dtype=torch.int32,
                                           device=device))
        # fixed-size state: one tensor per distinct size
        self.state_where: Dict[int, Tuple[int, int]] = {}
        sizes: Dict[int, List[int]] = {}
        for entry, r in enumerate(state_requests):
            if r is not None:
                sizes.setdefault(r.numel, []).append(entry)
        self.states: List[torch.Tensor] = []
        for numel, entries in sizes.items():
            for i, e in enumerate(entries):
                self.state_where[e] = (len(self.states), i)
            self.states.append(torch.zeros((len(entries), n_slots, numel), dtype=torch.float32,
                                           device=device))

    # ------------------------------------------------------------- lifecycle
    def acquire(self) -> int:
        s = self.book.acquire()
        for st in self.states:
            st[:, s].zero_()
        return s

    def reserve(self, slot: int, new_len: int) -> None:
        self.book.reserve(slot, new_len)

    def trim(self, slot: int) -> None:
        self.book.trim(slot)

    def release(self, slot: int) -> None:
        self.book.release(slot)

    def flush(self) -> None:
        """Copy changed page-table rows to the device (on the current stream).

        Every flush stages its rows in pinned memory of its own: a copy that has
        not run yet must not see what a later flush writes for the same slot (a
        slot released and taken again with no read in between).  The pinned
        allocator hands a block out again only after the copies from it have run."""
        if not self.book.dirty:
            return
        pinned = self.device.type == "cuda"
        for s in sorted(self.book.dirty):
            pages = self.book.pages.get(s)
            if pages is None:
                continue
            for gi, plist in enumerate(pages):
                if not plist:
                    continue
                row = torch.tensor(plist, dtype=torch.int32)
                if pinned:
                    row = row.pin_memory()
                self.tables[gi][s, :len(plist)].copy_(row, non_blocking=True)
        self.book.dirty.clear()

    # ----------------------------------------------------------------- views
    def kv_view(self, entry: int) -> KVView:
        if entry not in self.where:
            raise CacheError(f"cache entry {entry} holds no keys and values")
        gi, li = self.where[entry]
        g = self.book.groups[gi]
        sc = self.scales[gi]
        return KVView(self.k_pools[gi][li], self.v_pools[gi][li], self.tables[gi], PAGE, g.cap,
                      g.window, *((sc[0, li], sc[1, li]) if sc is not None else ()))

    def state_view(self, entry: int) -> StateView:
        if entry not in self.state_where:
            raise CacheError(f"cache entry {entry} holds no fixed-size state")
        ti, li = self.state_where[entry]
        return StateView(self.states[ti][li])

    def bytes_held(self) -> int:
        n = 0
        seen = set()
        scales = [s for s in self.scales if s is not None]
        for t in self.k_pools + self.v_pools + self.states + self.tables + scales:
            if t.data_ptr() in seen:
                continue
            seen.add(t.data_ptr())
            n += t.numel() * t.element_size()
        return n
