"""The cache manager: page tables on the host, pools and state arenas on the device.

A model hands over, for each of its cache layers, what that layer's mixer
needs: `KVSpec` (keys and values in pages; all of them, or a window) or
`StateSpec` (a fixed-size state per request).  Cache layers with the same
KVSpec form a group that shares page ids and has a pool of its own:

    pool[group]   [layers of the group, pages, 2 (k, v), kv heads, page_size, head_dim]
                  (values of another size than the keys: [layers, pages, kv heads * page_size * (head_dim + v_dim)],
                  a page's keys [kv heads, page_size, head_dim] followed by its values [kv heads, page_size, v_dim];
                  values inside the keys: [layers, pages, kv heads * page_size * head_dim];
                  v_share key heads to a value head: the values are [kv heads / v_share, page_size, v_dim])
    state[cache]  [max_requests, *shape]     one row per request slot (cache layers of one shape lie at equal distances in one allocation)

A request holds one slot from open() to close(); its state rows are zeroed
when the slot is taken.  fork() and adopt() let requests go on from where others
stand: full pages are held in common, the page in the middle and the state rows are
copied, one launch for each group of pages and each shape of states.  (They read what is
there: ModelRunner's forms see to it that the steps which wrote it have worked.)
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Dict, Hashable, List, Optional, Sequence, Tuple, Union

import torch

from .pages import CacheError, OutOfPages, PageGroup, PageTables, UNMAPPED  # noqa: F401


@dataclass(frozen=True)
class KVSpec:
    """Keys and values of `num_kv_heads` heads of `head_dim`; window = 0 keeps every position; v_dim = 0: values of
    the keys' size, else their own size (a page then holds the keys of its slots followed by the values).
    value_in_key: a key's first v_dim values ARE its value; the cache then holds the keys alone (a latent that is
    read both as part of the key and as the value is stored once).
    v_share > 1: that many neighbouring key heads read one value head (several score maps over the same values); a page
    then holds num_kv_heads heads of keys followed by num_kv_heads / v_share heads of values."""
    num_kv_heads: int
    head_dim: int
    window: int = 0
    v_dim: int = 0
    value_in_key: bool = False
    v_share: int = 1


@dataclass(frozen=True)
class StateSpec:
    """A per-request state of fixed shape, kept in the request's slot."""
    shape: Tuple[int, ...]
    dtype: torch.dtype = torch.float32


CacheSpec = Union[KVSpec, StateSpec, None]


@dataclass
class LayerCacheView:
    """What one cache layer looks like to its mixer during a step."""
    spec: CacheSpec
    group: int = -1                              # page group (KVSpec)
    pages: Optional[torch.Tensor] = None         # [pages, 2, nkv, page_size, hd] of this layer
    state: Optional[torch.Tensor] = None         # [max_requests, *shape] (StateSpec)


class CacheManager:
    def __init__(self, specs: Sequence[CacheSpec], *, page_size: int, num_pages: Union[int, Sequence[int]],
                 max_requests: int, dtype: torch.dtype, device: Union[str, torch.device], allocate: bool = True):
        self.specs = list(specs)
        self.page_size = page_size
        self.max_requests = max_requests
        self.dtype = dtype
        self.device = torch.device(device)
        by_spec: Dict[KVSpec, List[int]] = {}
        for cid, spec in enumerate(self.specs):
            if isinstance(spec, KVSpec):
                by_spec.setdefault(spec, []).append(cid)
        self.groups = [PageGroup(tuple(ids), s.num_kv_heads, s.head_dim, s.window) for s, ids in by_spec.items()]
        self._v_dims = [0 if s.value_in_key else (s.v_dim or s.head_dim) for s in by_spec]      # values stored beside the keys
        self._v_heads = [s.num_kv_heads // max(1, s.v_share) for s in by_spec]
        for s in by_spec:
            if s.v_share < 1 or s.num_kv_heads % s.v_share or (s.value_in_key and s.v_share != 1):
                raise ValueError("key heads do not divide into the value heads they share")
        if isinstance(num_pages, int):
            num_pages = [num_pages] * len(self.groups)
        self.tables = PageTables(self.groups, page_size, list(num_pages), max_requests)
        self.views: List[LayerCacheView] = [LayerCacheView(spec) for spec in self.specs]
        self.pools: List[Optional[torch.Tensor]] = []
        for g, grp in enumerate(self.groups):
            pool = None
            if allocate:
                spec = list(by_spec)[g]
                shape = ((2, grp.num_kv_heads, page_size, grp.head_dim)
                         if self._v_dims[g] == grp.head_dim and not spec.value_in_key and spec.v_share == 1
                         else (page_size * (grp.num_kv_heads * grp.head_dim + self._v_heads[g] * self._v_dims[g]),))
                pool = torch.zeros((len(grp.cache_ids), self.tables.pools[g].num_pages, *shape), dtype=dtype, device=self.device)
            self.pools.append(pool)
            for i, cid in enumerate(grp.cache_ids):
                self.views[cid].group = g
                self.views[cid].pages = pool[i] if pool is not None else None
        self._arenas: List[torch.Tensor] = []            # [cache layers of the shape, max_requests, numbers]
        by_state: Dict[StateSpec, List[int]] = {}
        for cid, spec in enumerate(self.specs):
            if isinstance(spec, StateSpec) and allocate:
                by_state.setdefault(spec, []).append(cid)
        for spec, ids in by_state.items():
            numbers = math.prod(spec.shape)
            size = torch.empty((), dtype=spec.dtype).element_size()
            apart = -(-max_requests * numbers * size // 512) * 512 // size      # every layer begins as an allocation of its own would
            whole = torch.zeros((len(ids) * apart,), dtype=spec.dtype, device=self.device)
            self._arenas.append(whole.as_strided((len(ids), max_requests, numbers), (apart, numbers, 1)))
            for i, cid in enumerate(ids):
                self.views[cid].state = whole[i * apart:i * apart + max_requests * numbers].view(max_requests, *spec.shape)

    # -- sizes --------------------------------------------------------------------------------
    def bytes_per_token(self) -> int:
        """Cache bytes one position takes over all groups (every layer, keys and values)."""
        size = torch.empty((), dtype=self.dtype).element_size()
        return sum(len(g.cache_ids) * (g.num_kv_heads * g.head_dim + vh * vd) * size
                   for g, vd, vh in zip(self.groups, self._v_dims, self._v_heads))

    def token_capacity(self) -> int:
        """Positions the smallest pool can hold."""
        if not self.groups:
            return 1 << 62
        return min(p.num_pages for p in self.tables.pools) * self.page_size

    # -- requests -----------------------------------------------------------------------------
    def open(self, request_id: Hashable) -> int:
        rc = self.tables.open(request_id)
        for view in self.views:
            if view.state is not None:
                view.state[rc.slot].zero_()
        return rc.slot

    def close(self, request_id: Hashable) -> None:
        self.tables.close(request_id)

    def fork(self, source_id: Hashable, request_id: Hashable) -> int:
        """Open request_id as one that goes on from where source_id stands (its keys, values and states); returns its slot."""
        self.fork_many([(request_id, source_id)])
        return self.tables.get(request_id).slot

    def fork_many(self, pairs: Sequence[Tuple[Hashable, Hashable]]) -> None:
        """fork() for every (request, source), all of them or nothing; the moves of all in one launch for each group of pages and each shape of states."""
        pairs = list(pairs)
        if pairs:
            self._copy(self.tables.fork_many(pairs), pairs)

    def adopt(self, pairs: Sequence[Tuple[Hashable, Hashable]]) -> None:
        """For every (request, source): the request forgets what it has and goes on from where the source stands.  No request is named
        twice, or as a source too."""
        pairs = list(pairs)
        if pairs:
            self._copy(self.tables.adopt(pairs), pairs)

    def _copy(self, pages: Sequence[tuple], pairs: Sequence[Tuple[Hashable, Hashable]]) -> None:
        from .. import ops
        for g, pool in enumerate(self.pools):
            moves = [(a, b) for group, a, b in pages if group == g]
            if moves and pool is not None:
                ops.copy_rows(pool, [a for a, _ in moves], [b for _, b in moves])
        for arena in self._arenas:
            ops.copy_rows(arena, [self.tables.get(s).slot for _, s in pairs], [self.tables.get(r).slot for r, _ in pairs])

    def length(self, request_id: Hashable) -> int:
        return self.tables.get(request_id).length

    def slot(self, request_id: Hashable) -> int:
        return self.tables.get(request_id).slot

    def is_open(self, request_id: Hashable) -> bool:
        return request_id in self.tables.requests

    def reserve_step(self, plan: Sequence[Tuple[Hashable, int]]) -> None:
        """Pages for every (request, n_tokens) of a step, or OutOfPages with nothing changed."""
        if not self.tables.can_reserve(list(plan)):
            raise OutOfPages("the step needs more pages than are free")
        done = []
        try:
            for rid, n in plan:
                self.tables.reserve(rid, n)
                done.append(rid)
        except CacheError:
            for rid in done:
                self.tables.rollback(rid)
            raise

    def commit_step(self, plan: Sequence[Tuple[Hashable, int]]) -> None:
        for rid, _ in plan:
            self.tables.commit(rid)

    def rollback_step(self, plan: Sequence[Tuple[Hashable, int]]) -> None:
        for rid, _ in plan:
            self.tables.rollback(rid)

    def truncate(self, request_id: Hashable, length: int) -> None:
        """Forget positions >= length.  A fixed-size state cannot be taken back to an earlier position (it has to
        be computed again from the start), so a model with such a state refuses anything but the current length."""
        if self.has_state and length != self.length(request_id):
            raise CacheError("a request with a fixed-size state cannot be truncated; close it and run it again")
        self.tables.truncate(request_id, length)

    def rewind(self, request_id: Hashable, length: int) -> None:
        """truncate() for the step function's own undoing of steps, which restores the states itself."""
        self.tables.truncate(request_id, length)

    # -- fixed-size states across a step --------------------------------------------------------
    @property
    def has_state(self) -> bool:
        return any(v.state is not None for v in self.views)

    def save_states(self, request_ids: Sequence[Hashable]):
        """Copies of the state rows of these requests (None when no cache layer has a state): what restore_states
        needs to undo a step that wrote them."""
        if not self.has_state:
            return None
        slots = torch.tensor([self.tables.get(r).slot for r in request_ids], dtype=torch.long, device=self.device)
        return slots, [(cid, v.state.index_select(0, slots)) for cid, v in enumerate(self.views) if v.state is not None]

    def restore_states(self, saved) -> None:
        if saved is None:
            return
        slots, rows = saved
        for cid, copy in rows:
            self.views[cid].state.index_copy_(0, slots, copy)

    def free_pages(self) -> List[int]:
        return [p.free_pages for p in self.tables.pools]

    def check(self) -> None:
        self.tables.check()
