"""Pages, block tables and state slots: the host side of the cache manager.

Nothing here touches a device.  A page is `page_size` consecutive positions of
one request in every layer of one group; a block table maps a request's block
number (position // page_size) to a page id, or -1 where no page is held
(before the first, or behind a window).  Pages are handed out from a LIFO
stack, so a page that was just given back is the next one used.

Requests may hold pages in common: fork() opens a request that goes on from
where another stands, adopt() makes open requests go on from others.  Full
pages are shared (a page goes back to its pool when its last holder gives it
up); the page a request is in the middle of is always its own, since it will be
written, so a fork takes a new page for it and names the copy to make.

The reference keeps a contiguous cache per sequence slot
(engine/include/model.h:106-110) and so never runs out in mid-request; its
unused kv_cache.c names the vocabulary only (block, block table, unmapped =
all-ones).  The paging here is this engine's own.
"""
from __future__ import annotations

import itertools
from dataclasses import dataclass, field
from typing import Dict, Hashable, List, Optional, Sequence

UNMAPPED = -1


class CacheError(RuntimeError):
    """A misuse of the cache manager: a page freed twice, a foreign page, an unknown request."""


class OutOfPages(CacheError):
    """The pool cannot give the pages a step needs; nothing was changed."""


class PagePool:
    """`num_pages` page ids with an owner tag each, and further holders where a page is shared.  alloc, share and free are O(1)."""

    def __init__(self, num_pages: int):
        if num_pages < 1:
            raise CacheError("a page pool needs at least one page")
        self.num_pages = num_pages
        self._free: List[int] = list(range(num_pages - 1, -1, -1))  # pop() gives 0 first
        self._owner: List[Optional[Hashable]] = [None] * num_pages
        self._more: Dict[int, Dict[Hashable, None]] = {}            # shared pages: who holds them besides the owner

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def alloc(self, owner: Hashable) -> int:
        if owner is None:
            raise CacheError("a page needs an owner")
        if not self._free:
            raise OutOfPages("no free page")
        page = self._free.pop()
        self._owner[page] = owner
        return page

    def free(self, page: int, owner: Hashable) -> None:
        if not (0 <= page < self.num_pages):
            raise CacheError(f"page {page} is not in the pool")
        if self._owner[page] is None:
            raise CacheError(f"page {page} is freed twice")
        more = self._more.get(page)
        if self._owner[page] != owner:
            if more is None or owner not in more:
                raise CacheError(f"page {page} belongs to {self._owner[page]!r}, not to {owner!r}")
            del more[owner]
        elif more is not None:
            self._owner[page] = more.popitem()[0]
        else:
            self._owner[page] = None
            self._free.append(page)
            return
        if not more:
            del self._more[page]

    def share(self, page: int, owner: Hashable) -> None:
        """`owner` holds the page too, until it frees it."""
        if owner is None:
            raise CacheError("a page needs an owner")
        if not (0 <= page < self.num_pages) or self._owner[page] is None:
            raise CacheError(f"page {page} is held by nobody")
        if owner == self._owner[page] or owner in self._more.get(page, ()):
            raise CacheError(f"page {page} is held by {owner!r} already")
        self._more.setdefault(page, {})[owner] = None

    def holders(self, page: int) -> List[Hashable]:
        """Who holds the page (nobody: it is free)."""
        return [] if self._owner[page] is None else [self._owner[page], *self._more.get(page, ())]

    def is_shared(self, page: int) -> bool:
        return page in self._more

    @property
    def has_shared(self) -> bool:
        """Whether any page has several holders."""
        return bool(self._more)

    def owner(self, page: int) -> Optional[Hashable]:
        return self._owner[page]

    def check(self) -> None:
        """Every page is either free exactly once or owned; raises otherwise."""
        seen = set()
        for p in self._free:
            if p in seen:
                raise CacheError(f"page {p} is on the free list twice")
            if self._owner[p] is not None or p in self._more:
                raise CacheError(f"page {p} is free and owned")
            seen.add(p)
        owned = sum(1 for o in self._owner if o is not None)
        if owned + len(seen) != self.num_pages:
            raise CacheError("a page is lost: neither free nor owned")


class SlotPool:
    """Fixed-size per-request state slots 0..n-1; the lowest free slot is given first."""

    def __init__(self, num_slots: int):
        self.num_slots = num_slots
        self._free = list(range(num_slots - 1, -1, -1))
        self._owner: List[Optional[Hashable]] = [None] * num_slots

    @property
    def free_slots(self) -> int:
        return len(self._free)

    def acquire(self, owner: Hashable) -> int:
        if not self._free:
            raise CacheError("no free request slot")
        s = self._free.pop()
        self._owner[s] = owner
        return s

    def release(self, slot: int, owner: Hashable) -> None:
        if self._owner[slot] != owner or owner is None:
            raise CacheError(f"slot {slot} is not held by {owner!r}")
        self._owner[slot] = None
        self._free.append(slot)
        self._free.sort(reverse=True)


@dataclass
class GroupTable:
    """One request's pages in one layer group."""
    blocks: List[int] = field(default_factory=list)   # block number -> page id or UNMAPPED
    first_held: int = 0                               # blocks below this were given back (window)


@dataclass
class RequestCache:
    request_id: Hashable
    slot: int
    length: int = 0                # positions whose keys and values are in the cache (committed)
    reserved: int = 0              # positions reserved beyond `length` for the step in flight
    family: int = 0                # a number of its own, or that of the request it goes on from (ids may be used again, families are not)
    common: int = 1 << 30          # at least so many leading blocks it has in common with all of its family (no limit while it is alone)
    tables: Dict[int, GroupTable] = field(default_factory=dict)   # group index -> table


@dataclass(frozen=True)
class PageGroup:
    """Layers with the same needs share page ids: `window` = 0 keeps every key, else the last `window`."""
    cache_ids: tuple          # the cache layers of this group, in pool order
    num_kv_heads: int
    head_dim: int
    window: int = 0


class PageTables:
    """Requests, their block tables in every group, and the pools behind them."""

    def __init__(self, groups: List[PageGroup], page_size: int, pages_per_group: List[int], max_requests: int):
        if page_size < 1:
            raise CacheError("page_size must be at least 1")
        if len(groups) != len(pages_per_group):
            raise CacheError("one page count is needed for each group")
        self.groups = list(groups)
        self.page_size = page_size
        self.pools = [PagePool(n) for n in pages_per_group]
        self.slots = SlotPool(max_requests)
        self.requests: Dict[Hashable, RequestCache] = {}
        self._families = itertools.count()

    # -- requests ---------------------------------------------------------------------------
    def open(self, request_id: Hashable) -> RequestCache:
        if request_id in self.requests:
            raise CacheError(f"request {request_id!r} is already open")
        rc = RequestCache(request_id, self.slots.acquire(request_id))
        rc.tables = {g: GroupTable() for g in range(len(self.groups))}
        rc.family = next(self._families)
        self.requests[request_id] = rc
        return rc

    # -- requests that hold pages in common ---------------------------------------------------
    def _tail_copies(self, rc: RequestCache) -> List[int]:
        """The groups in which a request that goes on from rc needs a page of its own for the page rc is in the middle of."""
        if rc.length % self.page_size == 0:
            return []
        return [g for g, t in rc.tables.items() if t.blocks[rc.length // self.page_size] != UNMAPPED]

    def _continue(self, rc: RequestCache, source: RequestCache, kept: Sequence[int]) -> List[tuple]:
        """rc, which holds source's first kept[g] blocks of every group and no others, holds what source has; returns (group, source's page, rc's
        page) for each page to copy."""
        copies = []
        tails = self._tail_copies(source)
        full = source.length // self.page_size
        for g, table in source.tables.items():
            mine = rc.tables[g]
            mine.blocks += table.blocks[kept[g]:full]
            mine.first_held = table.first_held
            for page in mine.blocks[kept[g]:]:
                if page != UNMAPPED:
                    self.pools[g].share(page, rc.request_id)
            if source.length % self.page_size:
                if g in tails:
                    mine.blocks.append(self.pools[g].alloc(rc.request_id))
                    copies.append((g, table.blocks[full], mine.blocks[full]))
                else:
                    mine.blocks.append(UNMAPPED)
        rc.length, rc.reserved, rc.family = source.length, 0, source.family
        source.common = min(source.common, full)
        rc.common = source.common
        return copies

    def fork(self, source_id: Hashable, request_id: Hashable) -> List[tuple]:
        """Open request_id as a request that goes on from where source_id stands.  Returns (group, from page, to page) for the
        pages whose content has to be copied.  Pages and a slot are there, or nothing is changed."""
        return self.fork_many([(request_id, source_id)])

    def fork_many(self, pairs: Sequence[tuple]) -> List[tuple]:
        """fork() for every (request, source): all of them, or nothing is changed."""
        requests = [r for r, _ in pairs]
        if len(set(requests)) != len(requests):
            raise CacheError("a request is opened twice")
        for request_id in requests:
            if request_id in self.requests:
                raise CacheError(f"request {request_id!r} is already open")
        sources = [self.get(s) for _, s in pairs]
        if any(source.reserved for source in sources):
            raise CacheError("fork during a step")
        tails = [self._tail_copies(source) for source in sources]
        for g, pool in enumerate(self.pools):
            need = sum(1 for t in tails if g in t)
            if need > pool.free_pages:
                raise OutOfPages(f"group {g} needs {need} pages for the ends of requests {requests!r} and has {pool.free_pages}")
        if len(requests) > self.slots.free_slots:
            raise CacheError("no free request slot")
        copies = []
        for request_id, source in zip(requests, sources):
            copies += self._continue(self.open(request_id), source, [0] * len(self.groups))
        return copies

    def adopt(self, pairs: List[tuple]) -> List[tuple]:
        """For every (request, source): the request forgets what it holds and goes on from where the source stands.  No request is named
        twice, or as a source too.  Returns the pages to copy, as fork() does.  Enough pages, or nothing is changed."""
        requests = [r for r, _ in pairs]
        if len(set(requests)) != len(requests) or set(requests) & {s for _, s in pairs}:
            raise CacheError("a request is adopted into twice, or is a source too")
        rcs = [(self.get(r), self.get(s)) for r, s in pairs]
        if any(rc.reserved or source.reserved for rc, source in rcs):
            raise CacheError("adopt during a step")
        # what a request and its source hold in common already stays where it is
        kept = [[self._common(rc.tables[g], source.tables[g], source.length // self.page_size) for g in range(len(self.groups))] for rc, source in rcs]
        for g, pool in enumerate(self.pools):
            need = sum(1 for _, source in rcs if g in self._tail_copies(source))
            if need > pool.free_pages:
                # a page comes back when everybody who holds it is among the requests that let go of it
                leaving = {}
                for (rc, _), k in zip(rcs, kept):
                    for page in rc.tables[g].blocks[k[g]:]:
                        if page != UNMAPPED:
                            leaving.setdefault(page, set()).add(rc.request_id)
                back = sum(1 for page, who in leaving.items() if who.issuperset(pool.holders(page)))
                if need > pool.free_pages + back:
                    raise OutOfPages(f"group {g} needs {need} pages and has {pool.free_pages + back}")
        for (rc, _), k in zip(rcs, kept):
            for g, table in rc.tables.items():
                for page in table.blocks[k[g]:]:
                    if page != UNMAPPED:
                        self.pools[g].free(page, rc.request_id)
                del table.blocks[k[g]:]
        copies = []
        for (rc, source), k in zip(rcs, kept):
            copies += self._continue(rc, source, k)
        return copies

    @staticmethod
    def _common(a: GroupTable, b: GroupTable, limit: int) -> int:
        """How many leading blocks two tables have alike, at most `limit`."""
        n = min(len(a.blocks), len(b.blocks), limit)
        return next((i for i, (x, y) in enumerate(zip(a.blocks[:n], b.blocks)) if x != y), n)

    def get(self, request_id: Hashable) -> RequestCache:
        try:
            return self.requests[request_id]
        except KeyError:
            raise CacheError(f"request {request_id!r} is not open") from None

    def close(self, request_id: Hashable) -> None:
        """Give back every page and the slot."""
        rc = self.get(request_id)
        for g, table in rc.tables.items():
            for page in table.blocks:
                if page != UNMAPPED:
                    self.pools[g].free(page, request_id)
        self.slots.release(rc.slot, request_id)
        del self.requests[request_id]

    # -- pages ------------------------------------------------------------------------------
    def _first_needed_block(self, g: int, first_query_pos: int) -> int:
        w = self.groups[g].window
        if w <= 0:
            return 0
        return max(0, first_query_pos - w + 1) // self.page_size

    def pages_needed(self, request_id: Hashable, n_tokens: int) -> List[int]:
        """New pages each group must give for the request's next n_tokens positions."""
        rc = self.get(request_id)
        end = rc.length + rc.reserved + n_tokens
        need = []
        for g in range(len(self.groups)):
            have = len(rc.tables[g].blocks)
            need.append(max(0, -(-end // self.page_size) - have))
        return need

    def can_reserve(self, plan: List[tuple]) -> bool:
        """Whether the pools hold enough for every (request_id, n_tokens) of a step together."""
        total = [0] * len(self.groups)
        for request_id, n in plan:
            for g, k in enumerate(self.pages_needed(request_id, n)):
                total[g] += k
        return all(total[g] <= self.pools[g].free_pages for g in range(len(self.groups)))

    def reserve(self, request_id: Hashable, n_tokens: int) -> None:
        """Hold pages for positions [length, length + n_tokens).  All groups or nothing."""
        rc = self.get(request_id)
        if n_tokens < 1:
            raise CacheError("a step needs at least one token of a request")
        need = self.pages_needed(request_id, n_tokens)
        for g, k in enumerate(need):
            if k > self.pools[g].free_pages:
                raise OutOfPages(f"group {g} needs {k} pages for request {request_id!r} and has {self.pools[g].free_pages} free")
        for g, k in enumerate(need):
            for _ in range(k):
                rc.tables[g].blocks.append(self.pools[g].alloc(request_id))
        rc.reserved += n_tokens

    def commit(self, request_id: Hashable) -> None:
        """The step ran: the reserved positions are now cached.  Pages a window has passed go back."""
        rc = self.get(request_id)
        rc.length += rc.reserved
        rc.reserved = 0
        for g in range(len(self.groups)):
            table = rc.tables[g]
            first = min(self._first_needed_block(g, rc.length), len(table.blocks))
            for b in range(table.first_held, first):
                if table.blocks[b] != UNMAPPED:
                    self.pools[g].free(table.blocks[b], request_id)
                    table.blocks[b] = UNMAPPED
            table.first_held = max(table.first_held, first)

    def rollback(self, request_id: Hashable) -> None:
        """The step did not run: give back the pages that only the reserved positions needed."""
        rc = self.get(request_id)
        rc.reserved = 0
        self._trim(rc, rc.length)

    def truncate(self, request_id: Hashable, length: int) -> None:
        """Forget positions >= length (cf. vitna_llama_truncate, engine/src/model.c:467-469).  A group
        with a window cannot go back behind what it has already given away."""
        rc = self.get(request_id)
        if rc.reserved:
            raise CacheError("truncate during a step")
        if length < 0 or length > rc.length:
            raise CacheError(f"cannot truncate request {request_id!r} of length {rc.length} to {length}")
        for g in range(len(self.groups)):
            if self._first_needed_block(g, length) < rc.tables[g].first_held:
                raise CacheError(f"group {g} has already given back pages that position {length} needs")
            if length % self.page_size and length < rc.length:
                page = rc.tables[g].blocks[length // self.page_size]
                if page != UNMAPPED and self.pools[g].is_shared(page):
                    raise CacheError(f"position {length} of request {request_id!r} lies inside a page that others hold too")
        rc.length = length
        rc.common = min(rc.common, length // self.page_size)
        self._trim(rc, length)

    def families(self, request_ids: Sequence[Hashable]) -> List[List[int]]:
        """The requests' places in the sequence, family by family (requests that were forked from one another)."""
        found: Dict[int, List[int]] = {}
        for i, rid in enumerate(request_ids):
            found.setdefault(self.get(rid).family, []).append(i)
        return list(found.values())

    def common_blocks(self, request_ids: Sequence[Hashable], g: int) -> int:
        """How many leading blocks requests of one family have alike in group g."""
        rcs = [self.get(r) for r in request_ids]
        blocks = [rc.tables[g].blocks for rc in rcs]
        n, most = min(rc.common for rc in rcs), min(len(b) for b in blocks)
        n = min(n, most)
        while n < most and all(b[n] == blocks[0][n] for b in blocks[1:]):
            n += 1
        return n

    def _trim(self, rc: RequestCache, length: int) -> None:
        keep = -(-length // self.page_size)
        for g, table in rc.tables.items():
            while len(table.blocks) > keep:
                page = table.blocks.pop()
                if page != UNMAPPED:
                    self.pools[g].free(page, rc.request_id)
            table.first_held = min(table.first_held, len(table.blocks))

    # -- what a step needs --------------------------------------------------------------------
    def slot_of_position(self, request_id: Hashable, g: int, pos: int) -> int:
        page = self.get(request_id).tables[g].blocks[pos // self.page_size]
        if page == UNMAPPED:
            raise CacheError(f"position {pos} of request {request_id!r} has no page in group {g}")
        return page * self.page_size + pos % self.page_size

    def check(self) -> None:
        """Pool consistency, and every held page is in exactly the tables of those who hold it."""
        for g, pool in enumerate(self.pools):
            pool.check()
            held = {}
            for rc in self.requests.values():
                for page in rc.tables[g].blocks:
                    if page == UNMAPPED:
                        continue
                    if rc.request_id not in pool.holders(page):
                        if page in held:
                            raise CacheError(f"page {page} of group {g} is held by {held[page]!r} and {rc.request_id!r}")
                        raise CacheError(f"page {page} of group {g} is in a table but owned by {pool.owner(page)!r}")
                    held.setdefault(page, []).append(rc.request_id)
            for page, requests in held.items():
                if len(requests) != len(pool.holders(page)) or len(set(requests)) != len(requests):
                    raise CacheError(f"page {page} of group {g} is in the tables of {requests!r} and held by {pool.holders(page)!r}")
            if len(held) + pool.free_pages != pool.num_pages:
                raise CacheError(f"group {g}: {pool.num_pages - pool.free_pages - len(held)} pages are owned but in no table")
