"""A key/value cache in pages, and what moves and shares them.

A sequence lives in a slot: its row of ``page_tables`` names its pages in
order, ``lengths`` its tokens.  Sequences that continue one another share
their full pages (``ref_counts`` says by how many a page is held); a
part-filled page belongs to one sequence, so nothing shared is ever written.

All state is on the cache's device and no call waits for it, so calls may be
captured into a graph where slots, pages and counts are tensors on that device;
lists are checked by the host and copied there, which waits and cannot be
captured.  A call that the host can see to be wrong raises; one that only the
tables show to be impossible (no page left, a slot out of range in a device
tensor, a target named twice) changes nothing and is reported by the next
``check()``.  Two exceptions: ``write`` leaves out the tokens it has no place
for, or only one in a shared page (where an ``extend`` before it could not be
carried out), and ``free`` and ``copy_pages`` leave out what is out of range.

On the GPU this is ``ops/csrc/paged_cache.hip``; on the CPU the same in torch.
"""

from __future__ import annotations

from typing import Optional, Sequence, Union

import torch
from torch.autograd import forward_ad

from ... import ops as _ops

Slots = Union[Sequence[int], torch.Tensor]

BAD_SLOT, NO_PAGE, BAD_PAGE, TOO_LONG, SHARED = 1, 2, 4, 8, 16
# of a sequence: sums of places and a few thousand stay below 2^31
MOST_TOKENS = (1 << 31) - 8192
_MESSAGES = {
    BAD_SLOT: "a slot out of range, or named twice",
    NO_PAGE: "no free page left",
    BAD_PAGE: "a page out of the pool",
    TOO_LONG: "a sequence longer than its table",
    SHARED: "a token for a page that several sequences hold",
}


class PagedKVCache:
    def __init__(self, num_layers: int, num_pages: int, page_size: int,
                 num_query_groups: int, head_dim: int, max_slots: int,
                 max_sequence_length: int, dtype=torch.bfloat16,
                 device="cuda"):
        for name, x in (("num_layers", num_layers), ("num_pages", num_pages),
                        ("num_query_groups", num_query_groups),
                        ("head_dim", head_dim), ("max_slots", max_slots),
                        ("max_sequence_length", max_sequence_length)):
            if x < 1:
                raise ValueError(f"PagedKVCache: {name} must be positive")
        if page_size < 16 or page_size % 16:
            raise ValueError("PagedKVCache: page_size must be a multiple of "
                             "16 tokens")
        width = -(-max_sequence_length // page_size)
        ints = dict(dtype=torch.int32, device=device)
        # zeros: what no token was written to is finite
        self._set(torch.zeros(num_layers, 2, num_pages, num_query_groups,
                              page_size, head_dim, dtype=dtype,
                              device=device),
                  torch.zeros(num_pages, **ints),
                  torch.full((max_slots, width), -1, **ints),
                  torch.zeros(max_slots, **ints))

    @classmethod
    def from_state(cls, pages: torch.Tensor, ref_counts: torch.Tensor,
                   page_tables: torch.Tensor, lengths: torch.Tensor
                   ) -> "PagedKVCache":
        """A cache of tensors that are there already (taken as they are, not
        copied): pages [layers, 2, P, groups, page, d], int32 ref_counts [P],
        page_tables [slots, W] and lengths [slots]."""
        cache = cls.__new__(cls)
        cache._set(pages, ref_counts, page_tables, lengths)
        return cache

    def _set(self, pages, ref_counts, page_tables, lengths):
        if pages.dim() != 6 or pages.shape[1] != 2 or not \
                pages.is_contiguous():
            raise ValueError("PagedKVCache: pages must be a contiguous "
                             "[layers, 2, P, groups, page, d]")
        if pages.shape[4] < 16 or pages.shape[4] % 16 or \
                pages.shape[5] * pages.element_size() % 16:
            raise ValueError("PagedKVCache: pages hold a multiple of 16 "
                             "tokens, each head a multiple of 16 bytes")
        for name, t, dim in (("ref_counts", ref_counts, 1),
                             ("page_tables", page_tables, 2),
                             ("lengths", lengths, 1)):
            if t.dtype != torch.int32 or t.dim() != dim or \
                    t.device != pages.device or not t.is_contiguous():
                raise ValueError(f"PagedKVCache: {name} must be a contiguous "
                                 "int32 tensor on the pages' device")
        if ref_counts.shape[0] != pages.shape[2] or \
                lengths.shape[0] != page_tables.shape[0]:
            raise ValueError("PagedKVCache: the tensors' sizes do not fit "
                             "each other")
        if page_tables.shape[1] * pages.shape[4] > MOST_TOKENS:
            raise ValueError("PagedKVCache: a sequence of 2^31 tokens, or "
                             "8191 fewer, does not fit its length")
        self.pages = pages
        self.ref_counts = ref_counts
        self.page_tables = page_tables
        self.lengths = lengths
        self.status = torch.zeros(1, dtype=torch.int32, device=pages.device)
        self.page_size = pages.shape[4]
        self.max_slots = lengths.shape[0]
        self.num_pages = pages.shape[2]

    # ----------------------------------------------------------- reading it
    @property
    def state(self):
        return (self.pages, self.ref_counts, self.page_tables, self.lengths,
                self.status)

    def keys(self, layer: int) -> torch.Tensor:
        """[P, groups, page, d]"""
        return self.pages[layer, 0]

    def values(self, layer: int) -> torch.Tensor:
        return self.pages[layer, 1]

    def free_pages(self) -> int:
        """Pages that no sequence holds.  Waits for the device."""
        return int((self.ref_counts == 0).sum())

    def check(self):
        """Raises if a call since the last check could not be carried out.
        Waits for the device."""
        code = int(self.status)
        if code:
            self.status.zero_()
            raise RuntimeError("PagedKVCache: " + "; ".join(
                m for bit, m in _MESSAGES.items() if code & bit))

    # -------------------------------------------------------------- helpers
    def _list(self, name: str, x: Slots, below: int,
              once: bool) -> torch.Tensor:
        """Slots or pages as an int32 tensor on the device; the host checks
        what it can see."""
        if isinstance(x, torch.Tensor):
            if x.dim() != 1 or x.dtype not in (torch.int32, torch.int64) or \
                    x.device != self.pages.device:
                raise ValueError(f"PagedKVCache: {name} must be a list or an "
                                 "int32 or int64 [n] on the cache's device")
            return self._int32(x)
        x = [int(i) for i in x]
        if any(i < 0 or i >= below for i in x):
            raise ValueError(f"PagedKVCache: {name} out of range: {x}")
        if once and len(set(x)) < len(x):
            raise ValueError(f"PagedKVCache: {name} named twice: {x}")
        return torch.tensor(x, dtype=torch.int32, device=self.pages.device)

    @staticmethod
    def _int32(x: torch.Tensor) -> torch.Tensor:
        """What does not fit 32 bits stays out of every range."""
        if x.dtype != torch.int32:
            x = x.clamp(-1 << 31, (1 << 31) - 1).int()
        return x.contiguous()

    @property
    def _native(self) -> bool:
        return self.pages.is_cuda

    # ------------------------------------------------------------ operators
    def load_tables(self, ref_counts: torch.Tensor, page_tables: torch.Tensor,
                    lengths: torch.Tensor):
        """Takes over the bookkeeping of a scheduler that keeps its own."""
        for name, to, x in (("ref_counts", self.ref_counts, ref_counts),
                            ("page_tables", self.page_tables, page_tables),
                            ("lengths", self.lengths, lengths)):
            if x.shape != to.shape:
                raise ValueError(f"PagedKVCache: {name} must be "
                                 f"{tuple(to.shape)}")
            to.copy_(x)

    def fork(self, src: Slots, dst: Slots):
        """Slot dst[i] becomes a copy of what slot src[i] held before the
        call, for all i at once: full pages are shared, the tokens of a
        part-filled one are copied to the lowest free page.  What dst[i] held
        is freed after that.  dst names no slot twice; src[i] == dst[i] keeps
        the slot as it is."""
        src = self._list("src", src, self.max_slots, False)
        dst = self._list("dst", dst, self.max_slots, True)
        if src.numel() != dst.numel() or src.numel() > self.max_slots:
            raise ValueError("PagedKVCache: fork: src and dst must name as "
                             "many slots, at most all")
        if self._native:
            _ops.get_ops().cache_fork(*self.state, src, dst)
        else:
            self._fork_plain(src.tolist(), dst.tolist())

    def free(self, slots: Slots):
        """Empties the slots; pages that nobody else holds become free."""
        slots = self._list("slots", slots, self.max_slots, False)
        if self._native:
            _ops.get_ops().cache_free(*self.state, slots)
            return
        for s in slots.tolist():
            if 0 <= s < self.max_slots:
                self._drop(s)
            else:
                self._fail(BAD_SLOT)

    def compact(self):
        """Moves the pages in use to the front of the pool: each that lies
        behind as many places as there are pages in use goes to the next free
        place before them, in order."""
        if self._native:
            _ops.get_ops().cache_compact(*self.state)
            return
        live = self.ref_counts > 0
        n = int(live.sum())
        holes = torch.nonzero(~live[:n]).flatten()
        movers = torch.nonzero(live[n:]).flatten() + n
        place = torch.arange(self.num_pages, dtype=torch.int32)
        place[movers] = holes.int()
        self.pages[:, :, holes] = self.pages[:, :, movers]
        self.ref_counts[holes] = self.ref_counts[movers]
        self.ref_counts[movers] = 0
        held = (self.page_tables >= 0) & (self.page_tables < self.num_pages)
        self.page_tables[held] = place[self.page_tables[held].long()]

    def copy_pages(self, src: Slots, dst: Slots):
        """Page dst[i] gets the content of page src[i], in all layers.  dst
        names no page twice, nor one of src: a list is checked for that, a
        tensor is not."""
        if not isinstance(src, torch.Tensor) and \
                not isinstance(dst, torch.Tensor) and \
                set(map(int, src)) & set(map(int, dst)):
            raise ValueError("PagedKVCache: copy_pages: a page is both "
                             "source and target")
        src = self._list("src", src, self.num_pages, False)
        dst = self._list("dst", dst, self.num_pages, True)
        if src.numel() != dst.numel():
            raise ValueError("PagedKVCache: copy_pages: src and dst must "
                             "name as many pages")
        if self._native:
            _ops.get_ops().cache_copy(*self.state, src, dst)
            return
        fine = (src >= 0) & (src < self.num_pages) & (dst >= 0) & \
            (dst < self.num_pages)
        if not bool(fine.all()):
            self._fail(BAD_PAGE)
        self.pages[:, :, dst[fine].long()] = self.pages[:, :,
                                                        src[fine].long()]

    def extend(self, slots: Slots, num_tokens: Union[int, Slots] = 1):
        """Makes the sequences longer by ``num_tokens`` (one number, or one
        for each), with pages for them, lowest free ones first; ``write``
        fills them, layer by layer.  No slot is named twice."""
        slots = self._list("slots", slots, self.max_slots, True)
        counts, each = None, 0
        if isinstance(num_tokens, int):
            if num_tokens < 0 or num_tokens >= 1 << 30:
                raise ValueError("PagedKVCache: extend: num_tokens out of "
                                 "range")
            each = num_tokens
        else:
            counts = self._list("num_tokens", num_tokens, 1 << 30, False)
            if counts.numel() != slots.numel():
                raise ValueError("PagedKVCache: extend: one number of tokens "
                                 "for each slot")
        if slots.numel() > self.max_slots:
            raise ValueError("PagedKVCache: extend: more slots than there "
                             "are")
        if self._native:
            _ops.get_ops().cache_extend(*self.state, slots, counts, each)
        else:
            self._extend_plain(slots.tolist(),
                               counts.tolist() if counts is not None
                               else [each] * slots.numel())

    def write(self, layer: int, key: torch.Tensor, value: torch.Tensor,
              slots: Slots, cu_seqlens: Optional[torch.Tensor] = None):
        """Puts key and value [tokens, groups, d] in the last places of the
        slots' sequences: one token each, or tokens cu_seqlens[i] to
        cu_seqlens[i + 1] as the last of slots[i].  No slot is named twice.
        The cache holds values: no derivative goes through it."""
        slots = self._list("slots", slots, self.max_slots, True)
        if not 0 <= layer < self.pages.shape[0]:
            raise ValueError(f"PagedKVCache: no layer {layer}")
        if key.dim() != 3 or value.shape != key.shape or \
                key.shape[1:] != (self.pages.shape[3], self.pages.shape[5]) \
                or key.dtype != self.pages.dtype or \
                value.dtype != self.pages.dtype or \
                key.device != self.pages.device or \
                value.device != self.pages.device:
            raise ValueError("PagedKVCache: write: key and value must be "
                             "[tokens, groups, d] of the cache's type and "
                             "device")
        if cu_seqlens is None:
            if key.shape[0] != slots.numel():
                raise ValueError("PagedKVCache: write: one token for each "
                                 "slot")
        elif cu_seqlens.dim() != 1 or \
                cu_seqlens.numel() != slots.numel() + 1 or \
                cu_seqlens.device != self.pages.device:
            raise ValueError("PagedKVCache: write: cu_seqlens must be "
                             "[slots + 1] on the cache's device")
        else:
            cu_seqlens = self._int32(cu_seqlens)
        if self._native:
            _ops.get_ops().cache_write(*self.state, layer, key, value, slots,
                                       cu_seqlens)
        else:
            self._write_plain(layer, key, value, slots.tolist(), cu_seqlens)

    # ------------------------------------------------------- the same in torch
    def _fail(self, code: int):
        self.status |= code

    def _lowest_free(self, n: int):
        free = torch.nonzero(self.ref_counts == 0).flatten()
        return None if free.numel() < n else free[:n].tolist()

    def _drop(self, slot: int):
        for p in self.page_tables[slot].tolist():
            if 0 <= p < self.num_pages:
                self.ref_counts[p] -= 1
        self.page_tables[slot] = -1
        self.lengths[slot] = 0

    def _fork_plain(self, src, dst):
        code, plan, copies = 0, [], 0
        if len(set(dst)) < len(dst):
            code |= BAD_SLOT
        for s, t in zip(src, dst):
            if not (0 <= s < self.max_slots and 0 <= t < self.max_slots):
                code |= BAD_SLOT
                continue
            n = int(self.lengths[s])
            if n < 0 or -(-n // self.page_size) > self.page_tables.shape[1]:
                code |= TOO_LONG
                continue
            row, copy = self.page_tables[s].clone(), None
            if s != t and n % self.page_size:
                copy = int(row[n // self.page_size])
                copies += 1
                if not 0 <= copy < self.num_pages:
                    code |= BAD_PAGE
            plan.append((t, n, row, copy, s == t))
        fresh = self._lowest_free(copies)
        if fresh is None:
            code |= NO_PAGE
        if code:
            self._fail(code)
            return
        rows = []
        for t, n, row, copy, same in plan:
            if same:
                continue
            full, part = divmod(n, self.page_size)
            row[full:] = -1
            if copy is not None:
                new = fresh.pop(0)
                row[full] = new
                self.pages[:, :, new, :, :part] = \
                    self.pages[:, :, copy, :, :part]
            rows.append((t, n, row))
        for t, n, row in rows:
            for p in row.tolist():
                if 0 <= p < self.num_pages:
                    self.ref_counts[p] += 1
        for t, n, row in rows:
            self._drop(t)
            self.page_tables[t] = row
            self.lengths[t] = n

    def _extend_plain(self, slots, counts):
        code, need, plan = 0, 0, []
        if len(set(slots)) < len(slots):
            code |= BAD_SLOT
        for s, c in zip(slots, counts):
            if not 0 <= s < self.max_slots or c < 0:
                code |= BAD_SLOT
                continue
            n = int(self.lengths[s])
            if n < 0 or n + c > self.page_tables.shape[1] * self.page_size:
                code |= TOO_LONG
                continue
            have = -(-n // self.page_size)
            more = -(-(n + c) // self.page_size) - have
            need += more
            plan.append((s, c, have, more))
        if code:
            self._fail(code)
            return
        fresh = self._lowest_free(need)
        if fresh is None:
            self._fail(NO_PAGE)
            return
        for s, c, have, more in plan:
            for j in range(more):
                p = fresh.pop(0)
                self.page_tables[s, have + j] = p
                self.ref_counts[p] = 1
            self.lengths[s] += c

    def _write_plain(self, layer, key, value, slots, cu):
        cu = list(range(len(slots) + 1)) if cu is None else cu.tolist()
        key, value = (forward_ad.unpack_dual(x.detach()).primal
                      for x in (key, value))
        for s, a, b in zip(slots, cu[:-1], cu[1:]):
            for t in range(max(a, 0), min(b, key.shape[0])):
                if not 0 <= s < self.max_slots:
                    self._fail(BAD_SLOT)
                    continue
                at = int(self.lengths[s]) - (b - t)
                if at < 0 or at // self.page_size >= \
                        self.page_tables.shape[1]:
                    self._fail(TOO_LONG)
                    continue
                page = int(self.page_tables[s, at // self.page_size])
                if not 0 <= page < self.num_pages:
                    self._fail(BAD_PAGE)
                    continue
                if int(self.ref_counts[page]) > 1:
                    self._fail(SHARED)
                    continue
                self.pages[layer, 0, page, :, at % self.page_size] = key[t]
                self.pages[layer, 1, page, :, at % self.page_size] = value[t]
