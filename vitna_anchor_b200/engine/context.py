"""A batch's arrays: from (request, its next tokens) to what the parts and kernels read on the device.

Everything a step's kernels need besides weights and the cache is laid out in ONE pinned host buffer and copied to
the device in one piece.  Where each array lies depends only on the step's counts (tokens, segments, wanted rows,
single-token segments, prompt tiles, width of the block tables), so a CUDA graph captured for one batch finds the
arrays of any other batch with the same counts in the same places.

The step function owns one builder; tests of single parts make their own over a cache manager of theirs, so that
they see the same layout the step function produces.
"""
from __future__ import annotations

from typing import Dict, Hashable, List, Optional, Sequence, Tuple

import numpy as np
import torch

from .. import ops
from ..cache.manager import CacheManager
from ..cache.pages import UNMAPPED
from ..parts.base import GroupMeta, StepContext, Workspace


class MetaOverflow(RuntimeError):
    """The step's arrays do not fit the metadata buffer."""


class _Staging:
    """A pinned host buffer and the event that tells when its last copy to the device is done."""

    def __init__(self, n: int, pinned: bool):
        self.host = torch.empty(n, dtype=torch.int32, pin_memory=pinned)
        self.np = self.host.numpy()
        self.event: Optional[torch.cuda.Event] = None


def meta_words(max_tokens: int, max_segments: int, max_blocks: int, n_groups: int) -> int:
    """The most 32-bit words a step's arrays can take, from the same terms build() puts:
    tokens, positions, token_seg (3T); seg_starts (S+1); seg_context, seg_slots (2S); wanted rows (<= T);
    single-token list (<= S) and the list of the other tokens (<= T); alignment (3); tiles of 64 and of 128
    tokens, four words each (a segment of n tokens makes ceil(n/64) <= n/64 + 1 tiles); and per page group
    the slot mapping (T) and the block tables (S * max_blocks)."""
    T, S = max_tokens, min(max_segments, max_tokens)
    tiles64, tiles128 = T // 64 + S, T // 128 + S
    return 3 * T + (S + 1) + 2 * S + T + S + T + 3 + 4 * tiles64 + 4 * tiles128 + n_groups * (T + S * max_blocks)


def words_used(lens: Sequence[int], wanted: int, max_blocks: int, n_groups: int) -> int:
    """The words build() puts for segments of these lengths with `wanted` rows in all and block tables `max_blocks` wide
    (the same terms in the same order; tests hold it against meta_words)."""
    T, S = sum(lens), len(lens)
    dec = sum(1 for n in lens if n == 1)
    pre = sum(n for n in lens if n > 1)
    off = 3 * T + (S + 1) + 2 * S + wanted + dec + (pre if dec else 0)
    off = (off + 3) & ~3
    off += 4 * sum(-(-n // 64) for n in lens if n > 1) + 4 * sum(-(-n // 128) for n in lens if n > 1)
    return off + n_groups * (T + S * max_blocks)


class ContextBuilder:
    def __init__(self, cache: CacheManager, dtype: torch.dtype, workspace: Workspace, *, max_batch_tokens: int,
                 max_segments: int, max_model_len: int, device, common_heads: Optional[Dict[int, Tuple[int, int, int]]] = None):
        # common_heads: by cache layer, of the attentions that can read common pages once (DecoderModel.common_heads)
        self.cache, self.dtype, self.workspace = cache, dtype, workspace
        self.device = torch.device(device)
        self.page_size = cache.page_size
        self.max_model_len = max_model_len
        self.max_blocks = -(-max_model_len // self.page_size)
        self.max_segments = max_segments
        heads = common_heads or {}
        self._common_heads = [sorted({heads[c] for c in group.cache_ids if c in heads}) for group in cache.groups]
        n_groups = len(cache.groups)
        # batches of single tokens with their families (build: 8 S + 1 and up to 3 of alignment; build_decode: 7 S + 1)
        decode_words = 8 * max_segments + 4 + n_groups * (max_segments + max_segments * self.max_blocks + 3 * max_segments + 1)
        self.meta_len = max(meta_words(max_batch_tokens, max_segments, self.max_blocks, n_groups), decode_words) + 8
        self._staging = [_Staging(self.meta_len, True) for _ in range(4)]
        self._turn = 0
        self.meta_dev = torch.zeros(self.meta_len, dtype=torch.int32, device=self.device)

    @property
    def turn(self) -> int:
        """Which of the staging buffers the latest build used (callers keep side buffers in step with it)."""
        return self._turn

    def _next_staging(self) -> _Staging:
        st = self._staging[self._turn]
        self._turn = (self._turn + 1) % len(self._staging)
        if st.event is not None:
            st.event.synchronize()
        return st

    def _send(self, st: _Staging, words: int) -> None:
        self.meta_dev[:words].copy_(st.host[:words], non_blocking=True)
        if st.event is None:
            st.event = torch.cuda.Event()
        st.event.record()

    # -- any mixture of segments ---------------------------------------------------------------------
    def build(self, segments: Sequence[Tuple[Hashable, Sequence[int], Sequence[int]]], fixed_blocks: Optional[int] = None,
              for_graph: bool = False) -> Tuple[StepContext, Optional[torch.Tensor]]:
        """segments: (request id, its next tokens, wanted places among them).  The requests' pages for the new
        positions must be reserved already.  Returns the context and the flat indices of the wanted rows."""
        S = len(segments)
        ps = self.page_size
        tables = self.cache.tables
        lens = [len(t) for _, t, _ in segments]
        T = sum(lens)
        R = sum(len(w) for _, _, w in segments)
        first = [tables.get(rid).length for rid, _, _ in segments]
        slots = [tables.get(rid).slot for rid, _, _ in segments]
        context = [f + n for f, n in zip(first, lens)]
        maxb = fixed_blocks or max(1, max(-(-c // ps) for c in context))

        st = self._next_staging()
        buf = st.np
        off = 0

        def put(values, count) -> slice:
            nonlocal off
            if off + count > self.meta_len:
                raise MetaOverflow(f"the step's arrays need more than the {self.meta_len} words of the metadata buffer")
            sl = slice(off, off + count)
            buf[sl] = values
            off += count
            return sl

        seg_starts = np.zeros(S + 1, dtype=np.int32)
        np.cumsum(lens, out=seg_starts[1:])
        s_tokens = put(np.concatenate([np.asarray(t, dtype=np.int32) for _, t, _ in segments]), T)
        s_pos = put(np.concatenate([np.arange(f, f + n, dtype=np.int32) for f, n in zip(first, lens)]), T)
        s_seg = put(np.repeat(np.arange(S, dtype=np.int32), lens), T)
        s_starts = put(seg_starts, S + 1)
        s_ctx = put(np.asarray(context, dtype=np.int32), S)
        s_slots = put(np.asarray(slots, dtype=np.int32), S)
        rows = [int(seg_starts[i]) + int(w) for i, (_, _, want) in enumerate(segments) for w in want]
        s_rows = put(np.asarray(rows, dtype=np.int32), R) if R else slice(off, off)
        dec = [int(seg_starts[i]) for i in range(S) if lens[i] == 1]
        pre = [t for i in range(S) if lens[i] > 1 for t in range(int(seg_starts[i]), int(seg_starts[i + 1]))]
        s_dec = put(np.asarray(dec, dtype=np.int32), len(dec)) if dec else None
        s_pre = put(np.asarray(pre, dtype=np.int32), len(pre)) if pre and dec else None
        # tiles in the order of the keys they walk over, longest walk LAST (the kernels start from the end of the list):
        # a launch ends sooner when its longest blocks start first, and in a batch of several prompts the longest walks
        # are not those of the last prompt
        tiles = [(int(seg_starts[i]) + o, min(64, lens[i] - o), first[i] + o, i)
                 for i in range(S) if lens[i] > 1 for o in range(0, lens[i], 64)]
        tiles.sort(key=lambda t: t[2] + t[1])
        off = (off + 3) & ~3                                   # 16-byte alignment for what follows
        s_tiles = put(np.asarray(tiles, dtype=np.int32).reshape(-1), 4 * len(tiles)) if tiles else None
        big = [(int(seg_starts[i]) + o, min(128, lens[i] - o), first[i] + o, i)
               for i in range(S) if lens[i] > 1 for o in range(0, lens[i], 128)]
        big.sort(key=lambda t: t[2] + t[1])
        s_big = put(np.asarray(big, dtype=np.int32).reshape(-1), 4 * len(big)) if big else None
        group_slices = []
        for g in range(len(self.cache.groups)):
            bt = np.zeros((S, maxb), dtype=np.int32)
            sm = np.empty(T, dtype=np.int32)
            for i, (rid, _, _) in enumerate(segments):
                blocks = tables.get(rid).tables[g].blocks
                row = np.asarray(blocks[:maxb], dtype=np.int32)
                pos = np.arange(first[i], first[i] + lens[i])
                sm[seg_starts[i]:seg_starts[i + 1]] = row[pos // ps] * ps + pos % ps
                row = np.where(row == UNMAPPED, 0, row)      # pages behind a window are never read
                bt[i, :len(row)] = row
            group_slices.append((put(sm, T), put(bt.reshape(-1), S * maxb)))
        # (a captured batch of these counts has none: what requests share is not among the counts)
        families = self.families([rid for rid, _, _ in segments]) if not for_graph and T == S else None
        family_slices = [put(self._family_words(families, S, S, g), 3 * S + 1) for g in range(len(self.cache.groups))] if families else []
        self._send(st, off)

        dev = self.meta_dev
        groups = [GroupMeta(dev[a], dev[b].view(S, maxb), maxb) for a, b in group_slices]
        for g, sl in enumerate(family_slices):
            self._set_families(groups[g], g, dev[sl], S)
        ctx = StepContext(
            num_tokens=T, num_segments=S, dtype=self.dtype, tokens=dev[s_tokens], positions=dev[s_pos],
            token_seg=dev[s_seg], seg_starts=dev[s_starts], seg_context=dev[s_ctx], seg_slots=dev[s_slots], groups=groups,
            caches=self.cache.views, workspace=self.workspace, host_seg_lens=lens, host_seg_first_pos=first,
            host_seg_slots=slots, max_seg_len=max(lens), max_context=self.max_model_len if for_graph else max(context),
            decode_only=all(n == 1 for n in lens),
            num_dec=len(dec), dec_tokens=None if (s_dec is None or not pre) else dev[s_dec],
            num_pre=len(pre), pre_tokens=None if s_pre is None else dev[s_pre],
            pre_tiles=None if s_tiles is None else dev[s_tiles].view(-1, 4),
            pre_tiles_big=None if s_big is None else dev[s_big].view(-1, 4))
        return ctx, (dev[s_rows] if R else None)

    # -- single tokens, padded to a fixed number of segments -----------------------------------------------
    def families(self, requests: Sequence[Hashable]) -> Optional[List[Tuple[List[int], List[int]]]]:
        """What requests of a batch of single tokens hold in common: for every family its places in the batch and the positions it shares in each page
        group (0 in groups with a window).  None where no attention would read those once, or it is not worth it (ops.attention_shared_serves, ops.attention_shared_pays)."""
        tables, ps = self.cache.tables, self.page_size
        if not any(pool.has_shared for pool in tables.pools):
            return None
        by_family = tables.families(requests)
        if len(by_family) == len(requests):
            return None
        out = [(f, [tables.common_blocks([requests[i] for i in f], g) * ps if len(f) > 1 and group.window == 0 else 0 for g, group in enumerate(self.cache.groups)])
               for f in by_family]
        for g, group in enumerate(self.cache.groups):
            saved = sum((len(f) - 1) * shared[g] for f, shared in out)
            read = any(ops.attention_shared_serves(self.dtype, *heads, len(requests), self.max_blocks * ps) for heads in self._common_heads[g])
            if ops.attention_shared_pays(saved, group.num_kv_heads, group.head_dim, self.dtype, read, self.max_model_len):
                return out
        return None

    @staticmethod
    def _family_words(families: List[Tuple[List[int], List[int]]], S: int, B: int, g: int) -> np.ndarray:
        """A page group's members [B], starts [B + 1] and shared [B] of a batch of S single tokens padded to B: a padding token is a family of its own."""
        words = np.zeros(3 * B + 1, dtype=np.int32)
        sizes = [len(f) for f, _ in families] + [1] * (B - S)
        words[:B] = [i for f, _ in families for i in f] + list(range(S, B))
        words[B + 1:B + 1 + len(sizes)] = np.cumsum(sizes)
        words[B + 1 + len(sizes):2 * B + 1] = B
        words[2 * B + 1:2 * B + 1 + len(families)] = [shared[g] for _, shared in families]
        return words

    def _set_families(self, meta: GroupMeta, g: int, words: torch.Tensor, B: int) -> None:
        if self.cache.groups[g].window == 0:
            meta.members, meta.starts, meta.shared = words[:B], words[B:2 * B + 1], words[2 * B + 1:]

    def build_decode(self, requests: Sequence[Hashable], tokens: Sequence[int], B: int, views: bool = True, reach: int = 0,
                     families: Optional[List[Tuple[List[int], List[int]]]] = None):
        """The context of a batch of single tokens, padded to B segments, at offsets that depend on B alone, so
        that a captured graph finds every array where it was at capture.  A padding segment has one token at
        position 0 that writes nothing (slot mapping -1, state slot -1) and reads page 0.  views=False: only fill the buffer.
        families: as families() has them; the page groups without a window then carry what their members share."""
        S, ps, maxb = len(requests), self.page_size, self.max_blocks
        tables = self.cache.tables
        st = self._next_staging()
        buf = st.np
        n_groups = len(self.cache.groups)
        o_families = 7 * B + 1 + n_groups * (B + B * maxb)
        total = o_families + (n_groups * (3 * B + 1) if families else 0)
        if total > self.meta_len:
            raise MetaOverflow(f"a decode batch of {B} needs more than the {self.meta_len} words of the metadata buffer")
        buf[:total] = 0
        o_tok, o_pos, o_seg, o_starts = 0, B, 2 * B, 3 * B
        o_ctx, o_slots, o_rows = 4 * B + 1, 5 * B + 1, 6 * B + 1
        o_groups = 7 * B + 1
        ar = np.arange(B + 1, dtype=np.int32)
        buf[o_seg:o_seg + B] = ar[:B]
        buf[o_starts:o_starts + B + 1] = ar
        buf[o_rows:o_rows + B] = ar[:B]
        buf[o_ctx:o_ctx + B] = 1
        buf[o_slots:o_slots + B] = -1                      # a padding segment has no state slot
        rcs = [tables.get(rid) for rid in requests]
        first = [rc.length for rc in rcs]
        buf[o_tok:o_tok + S] = [int(t) for t in tokens]
        buf[o_pos:o_pos + S] = first
        buf[o_ctx:o_ctx + S] = [f + 1 for f in first]
        buf[o_slots:o_slots + S] = [rc.slot for rc in rcs]
        for g in range(n_groups):
            o_sm = o_groups + g * (B + B * maxb)
            o_bt = o_sm + B
            buf[o_sm:o_sm + B] = -1
            bt = buf[o_bt:o_bt + B * maxb].reshape(B, maxb)
            for i, rc in enumerate(rcs):
                blocks = rc.tables[g].blocks
                row = np.asarray(blocks, dtype=np.int32)
                buf[o_sm + i] = row[first[i] // ps] * ps + first[i] % ps
                np.maximum(row, 0, out=row)
                bt[i, :len(row)] = row
            if families:
                o = o_families + g * (3 * B + 1)
                buf[o:o + 3 * B + 1] = self._family_words(families, S, B, g)
        self._send(st, total)
        if not views:               # a replay needs the arrays in place, not their description
            return None, None
        dev = self.meta_dev
        groups = []
        for g in range(n_groups):
            o_sm = o_groups + g * (B + B * maxb)
            meta = GroupMeta(dev[o_sm:o_sm + B], dev[o_sm + B:o_sm + B + B * maxb].view(B, maxb), maxb)
            if families:
                o = o_families + g * (3 * B + 1)
                self._set_families(meta, g, dev[o:o + 3 * B + 1], B)
            groups.append(meta)
        ctx = StepContext(
            num_tokens=B, num_segments=B, dtype=self.dtype, tokens=dev[o_tok:o_tok + B], positions=dev[o_pos:o_pos + B],
            token_seg=dev[o_seg:o_seg + B], seg_starts=dev[o_starts:o_starts + B + 1], seg_context=dev[o_ctx:o_ctx + B],
            seg_slots=dev[o_slots:o_slots + B], groups=groups, caches=self.cache.views, workspace=self.workspace,
            host_seg_lens=[1] * B, host_seg_first_pos=first + [0] * (B - S), host_seg_slots=[rc.slot for rc in rcs] + [-1] * (B - S),
            max_seg_len=1, max_context=reach or self.max_model_len, decode_only=True, num_dec=B)
        return ctx, dev[o_rows:o_rows + B]
