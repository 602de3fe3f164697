"""The host side of beam search: requests that hold pages in common, who takes over whom, and what is refused; no GPU is needed."""
import ctypes
import random

import pytest
import torch

from vitna_anchor_b200 import ops
from vitna_anchor_b200.cache import CacheError, CacheManager, KVSpec, OutOfPages, PageGroup, PagePool, PageTables, StateSpec, UNMAPPED
from vitna_anchor_b200.engine.beam import attainable, normalised, plan_moves


def test_a_page_goes_back_with_its_last_holder():
    pool = PagePool(2)
    a = pool.alloc("x")
    pool.share(a, "y")
    pool.share(a, "z")
    assert pool.holders(a) == ["x", "y", "z"] and pool.is_shared(a) and pool.free_pages == 1
    with pytest.raises(CacheError):
        pool.share(a, "y")
    with pytest.raises(CacheError):
        pool.free(a, "w")
    pool.free(a, "x")
    with pytest.raises(CacheError):
        pool.free(a, "x")
    pool.check()
    pool.free(a, "z")
    assert pool.holders(a) == ["y"] and not pool.is_shared(a) and pool.free_pages == 1
    pool.free(a, "y")
    assert pool.free_pages == 2 and pool.holders(a) == []
    for page in (a, 1 - a, 5):
        with pytest.raises(CacheError):
            pool.share(page, "q")
    pool.check()


class Model:
    """What the pages hold: every position a request wrote, by (group, page, offset)."""

    def __init__(self, tables):
        self.t, self.cells, self.history, self.next = tables, {}, {}, 0

    def write(self, rid, n):
        rc = self.t.get(rid)
        first = rc.length
        self.t.reserve(rid, n)
        for pos in range(first, first + n):
            self.next += 1
            self.history[rid].append(self.next)
            for g in range(len(self.t.groups)):
                slot = self.t.slot_of_position(rid, g, pos)
                assert len(self.t.pools[g].holders(slot // self.t.page_size)) == 1       # nobody else's page is written
                self.cells[g, slot] = self.next
        self.t.commit(rid)

    def copy(self, moves):
        read = [(g, a, b, [self.cells.get((g, a * self.t.page_size + o)) for o in range(self.t.page_size)]) for g, a, b in moves]
        assert len({(g, b) for g, _, b, _ in read}) == len(read) and not {(g, b) for g, _, b, _ in read} & {(g, a) for g, a, _, _ in read}
        for g, _, b, content in read:
            for o, v in enumerate(content):
                self.cells[g, b * self.t.page_size + o] = v

    def check(self):
        self.t.check()
        for rid, history in self.history.items():
            rc = self.t.get(rid)
            assert rc.length == len(history)
            for g, group in enumerate(self.t.groups):
                lo = 0 if group.window == 0 else max(0, rc.length - group.window + 1)
                for pos in range(lo, rc.length):
                    assert self.cells[g, self.t.slot_of_position(rid, g, pos)] == history[pos]


@pytest.mark.parametrize("seed", range(12))
def test_forks_and_adoptions_keep_everybodys_positions(seed):
    rng = random.Random(seed)
    ps = rng.choice([1, 3, 4])
    t = PageTables([PageGroup((0,), 1, 8, 0), PageGroup((1,), 1, 8, rng.choice([0, 5, 9]))], ps, [60, 60], 8)
    m, n = Model(t), 0
    for _ in range(200):
        live = list(m.history)
        what = rng.choice(["open", "write", "write", "fork", "adopt", "adopt", "close", "truncate"])
        before = {r: (list(t.get(r).tables[0].blocks), t.get(r).length) for r in live}
        try:
            if what == "open" and len(live) < 8:
                n += 1
                t.open(n)
                m.history[n] = []
            elif what == "write" and live:
                rid, count = rng.choice(live), rng.randint(1, 6)
                if t.can_reserve([(rid, count)]):
                    m.write(rid, count)
            elif what == "fork" and live and len(live) < 8:
                source = rng.choice(live)
                n += 1
                m.copy(t.fork(source, n))
                m.history[n] = list(m.history[source])
                assert t.get(n).family == t.get(source).family
            elif what == "adopt" and len(live) > 1:
                rng.shuffle(live)
                k = rng.randint(1, len(live) - 1)
                pairs = [(r, rng.choice(live[k:])) for r in live[:k]]
                m.copy(t.adopt(pairs))
                for r, source in pairs:
                    m.history[r] = list(m.history[source])
            elif what == "close" and live and rng.random() < 0.3:
                rid = rng.choice(live)
                t.close(rid)
                del m.history[rid]
            elif what == "truncate" and live:
                rid = rng.choice(live)
                length = rng.randint(0, t.get(rid).length)
                t.truncate(rid, length)
                del m.history[rid][length:]
        except OutOfPages:
            assert {r: (list(t.get(r).tables[0].blocks), t.get(r).length) for r in before} == before and len(t.requests) == len(m.history)
        except CacheError as e:
            assert what == "truncate", e                      # behind a window, or inside a page that others hold
        m.check()
        for f in t.families(list(m.history)):
            rids = [list(m.history)[i] for i in f]
            blocks = [t.get(r).tables[0].blocks for r in rids]
            same = 0
            while all(same < len(b) for b in blocks) and len({b[same] for b in blocks}) == 1:
                same += 1
            assert t.common_blocks(rids, 0) == same
    for rid in list(m.history):
        t.close(rid)
    assert [p.free_pages for p in t.pools] == [60, 60]


def test_a_name_that_is_used_again_begins_a_family_of_its_own():
    t = PageTables([PageGroup((0,), 1, 8, 0)], 2, [20], 4)
    t.open("a")
    t.reserve("a", 6)
    t.commit("a")
    t.fork("a", "b")
    assert t.families(["a", "b"]) == [[0, 1]] and t.common_blocks(["a", "b"], 0) == 3
    t.close("a")
    t.open("a")
    t.reserve("a", 6)
    t.commit("a")
    assert not set(t.get("a").tables[0].blocks) & set(t.get("b").tables[0].blocks)
    assert t.families(["a", "b"]) == [[0], [1]]
    t.check()


def test_what_fork_and_adopt_refuse():
    t = PageTables([PageGroup((0,), 1, 8, 0)], 4, [5], 3)
    t.open("a")
    t.reserve("a", 6)
    with pytest.raises(CacheError):
        t.fork("a", "b")                                      # a step is in flight
    t.commit("a")
    t.fork("a", "b")
    t.open("c")
    for pairs in [[("a", "a")], [("a", "b"), ("a", "c")], [("a", "b"), ("b", "c")], [("q", "a")], [("a", "q")]]:
        with pytest.raises(CacheError):
            t.adopt(pairs)
    with pytest.raises(CacheError):
        t.fork("a", "c")                                      # open already
    t.close("c")
    with pytest.raises(CacheError):
        t.truncate("b", 2)                                    # inside the page both hold
    t.truncate("b", 4)
    assert t.get("b").length == 4
    t.reserve("b", 12); t.commit("b")
    t.open("d")
    with pytest.raises(OutOfPages):
        t.adopt([("d", "a")])                                 # a page for the end is wanted and none is free
    assert t.get("d").length == 0
    t.check()


def test_states_of_one_shape_lie_in_one_arena():
    specs = [StateSpec((3, 5)), KVSpec(2, 8), StateSpec((7,), torch.float64), StateSpec((3, 5))]
    c = CacheManager(specs, page_size=4, num_pages=6, max_requests=5, dtype=torch.float32, device="cpu")
    assert len(c._arenas) == 2 and c._arenas[0].shape == (2, 5, 15) and c._arenas[1].shape == (1, 5, 7)
    for i, cid in enumerate([0, 3]):
        view = c.views[cid].state
        assert view.shape == (5, 3, 5) and view.is_contiguous() and (view.data_ptr() - c._arenas[0].data_ptr()) % 512 == 0
        view[2] = i + 1.0
        assert bool((c._arenas[0][i, 2] == i + 1.0).all())
    assert c.views[2].state.dtype == torch.float64 and bool((c._arenas[1] == 0).all())


def test_who_takes_over_whom():
    assert plan_moves([0, 1, 2], "abc") == (["a", "b", "c"], [], [])
    assert plan_moves([2, 2, 0], "abc") == (["c", "b", "a"], [("b", "c")], [])
    assert plan_moves([1, 1, 1, 1], "abcd") == (["b", "a", "c", "d"], [("a", "b"), ("c", "b"), ("d", "b")], [])
    assert plan_moves([0, 0, 0], "a") == (["a", None, None], [], [])
    assert plan_moves([2], "abc") == (["c"], [], ["a", "b"])
    rng = random.Random(1)
    for _ in range(300):
        live = list(range(100, 100 + rng.randint(1, 9)))
        parents = [rng.randrange(len(live)) for _ in range(rng.randint(1, 9))]
        requests, pairs, left = plan_moves(parents, live)
        named = [r for r in requests if r is not None]
        assert len(set(named)) == len(named) and not set(left) & set(named)
        assert not {r for r, _ in pairs} & {s for _, s in pairs}
        source = dict(pairs)
        for r, p in zip(requests, parents):
            assert r is None or source.get(r, r) == live[p]
        assert (None in requests) <= (not left)


def test_when_common_pages_are_read_once():
    """The rule's two sides (positions of 32 heads of 64: 8 KB; of 3: 0.75 KB), and the switch."""
    pays = ops.attention_shared_pays
    assert not pays(3 * 2000, 32, 64) and pays(7 * 2000, 32, 64) and not pays(63 * 500, 3, 64) and pays(63 * 4000, 3, 64) and not pays(0, 32, 64)
    for mode, taken in [(0, False), (1, True)]:
        assert ops.set_attention_shared(mode) == 2
        assert pays(8, 1, 16) == taken and not pays(0, 1, 16)
        assert ops.set_attention_shared(2) == mode


def test_scores():
    assert normalised(-6.0, 4, 0.5) == -3.0 and normalised(-6.0, 4, 0.0) == -6.0
    assert attainable(-6.0, 4, 16, 0.5) == -1.5 and attainable(-6.0, 4, 16, -0.5) == -12.0 and attainable(-6.0, 4, 16, 0.0) == -6.0


def test_entries_refuse_before_anything_runs():
    """The C entries say no to sizes they do not take; nothing is launched, so no device is needed."""
    lib, null = ops.lib(), ctypes.c_void_p(0)
    some = ctypes.c_void_p(64)
    LL, SIZE = ctypes.c_longlong, ctypes.c_size_t

    def attention(n=4, families=1, nh=4, nkv=2, hd=64, ps=16, maxb=8, dtype=1, scratch=some, room=1 << 40, error=64):
        at = lambda p: p.value or 0      # noqa: E731
        args = ctypes.create_string_buffer(ops._SHARED_ARGS.pack(*[at(some)] * 9, at(scratch), room, 4, 4, n, families, 10, nh, nkv, hd, ps, maxb, 0.1, dtype, error))
        return lib.vk_attention_shared(args, null)

    assert attention(n=0) == 0 and attention(families=0) == 0
    for kw in [dict(n=257), dict(families=257), dict(hd=264), dict(nkv=129, nh=129), dict(hd=12), dict(nh=5), dict(nh=130), dict(ps=0), dict(maxb=0), dict(maxb=1 << 28),
               dict(hd=6, dtype=0), dict(error=0), dict(scratch=ctypes.c_void_p(72)), dict(room=1 << 20)]:
        assert attention(**kw) < 0, kw

    # tiles of 16 keys and rows of outputs are counted in 31 bits; attention_shared_takes says so before, and a decode step then goes the other way
    for n, nh, nkv, hd, reach in [(256, 64, 1, 64, 1 << 21), (256, 64, 64, 64, (1 << 31) - 16), (1, 64, 64, 256, (1 << 31) - 16), (256, 8192, 128, 256, 16)]:
        assert attention(n=n, nh=nh, nkv=nkv, hd=hd, maxb=reach // 16, room=1 << 20) in (-3, -4)
        assert (attention(n=n, nh=nh, nkv=nkv, hd=hd, maxb=reach // 16, room=1 << 20) == -3) == (not ops.attention_shared_takes(torch.bfloat16, nh, nkv, hd, n, reach)), (n, nh, reach)

    def select(rows=8, beams=4, vocab=100, ld=100, keep=8, scratch=some, room=1 << 40):
        return lib.vk_beam_select(some, some, some, some, some, scratch, SIZE(room), rows, beams, vocab, LL(ld), keep, null)

    assert select(rows=0) == 0
    for kw in [dict(beams=3), dict(beams=0), dict(keep=0), dict(keep=129), dict(vocab=0), dict(ld=99), dict(beams=1, keep=101), dict(rows=1028), dict(rows=130, beams=65),
               dict(vocab=64 * 4096 + 1, ld=1 << 20), dict(scratch=null), dict(scratch=ctypes.c_void_p(8)), dict(room=4600)]:
        assert select(**kw) < 0, kw

    def copy(rows=4, src=(0,), dst=(1,), stride=16, size=16, layers=1):
        i = ctypes.c_int32 * len(src)
        return lib.vk_copy_rows(some, layers, rows, LL(0), LL(stride), LL(size), i(*src), i(*dst), len(src), null)

    assert copy(src=(), dst=()) == 0 and copy(layers=0) == 0 and copy(size=0) == 0
    for kw in [dict(src=(4,)), dict(dst=(4,)), dict(src=(-1,)), dict(dst=(-1,)), dict(rows=0), dict(stride=8), dict(layers=70000)]:
        assert copy(**kw) < 0, kw


def test_command_line_of_a_search():
    from vitna_anchor_b200.cli.main import main, parse_args
    a = parse_args(["--beams", "4", "--length-penalty", "0.7", "--ids", "1"])
    assert a["beams"] == 4 and a["length_penalty"] == 0.7
    for argv in [["generate", "--model", "x", "--ids", "1", "--length-penalty", "1"], ["generate", "--model", "x", "--ids", "1", "--beams", "2", "--temperature", "0.5"],
                 ["generate", "--model", "x", "--ids", "1", "--beams", "2", "--logits-out", "f"], ["generate", "--model", "x", "--ids", "1", "--beams", "two"]]:
        assert main(argv) == 1


def test_many_forks_are_one_move(monkeypatch):
    """Every (request, source), the copies of all together: one launch for each group of pages and each shape of states; nothing is changed where one cannot be."""
    specs = [KVSpec(1, 8), KVSpec(2, 8), StateSpec((3,))]
    c = CacheManager(specs, page_size=4, num_pages=[7, 9], max_requests=6, dtype=torch.float32, device="cpu")
    for rid, n in [("a", 6), ("b", 4)]:
        c.open(rid)
        c.reserve_step([(rid, n)])
        c.commit_step([(rid, n)])
    moves = []
    monkeypatch.setattr(ops, "copy_rows", lambda arena, src, dst: moves.append((tuple(arena.shape[:2]), list(src), list(dst))))

    def refused(pairs, error=CacheError):
        before = c.free_pages(), {r: [list(t.blocks) for t in rc.tables.values()] for r, rc in c.tables.requests.items()}, c.tables.slots.free_slots
        with pytest.raises(error):
            c.fork_many(pairs)
        assert before == (c.free_pages(), {r: [list(t.blocks) for t in rc.tables.values()] for r, rc in c.tables.requests.items()}, c.tables.slots.free_slots) and not moves
        c.check()

    refused([("c", "a"), ("c", "b")])
    refused([("c", "a"), ("a", "b")])
    refused([("c", "a"), ("d", "c")])                        # a source that is not open yet
    refused([("c", "a"), ("d", "q")])
    refused([(i, "b") for i in range(5)])                    # four slots
    refused([(i, "a") for i in range(5)], OutOfPages)        # and four pages of the smaller group
    c.fork_many([])
    assert not moves
    c.fork_many([("c", "a"), ("d", "b"), ("e", "a")])
    slot, page = c.slot, lambda r, g: c.tables.get(r).tables[g].blocks[1]      # noqa: E731
    assert moves == [((1, 7), [page("a", 0)] * 2, [page("c", 0), page("e", 0)]), ((1, 9), [page("a", 1)] * 2, [page("c", 1), page("e", 1)]),
                     ((1, 6), [slot("a"), slot("b"), slot("a")], [slot("c"), slot("d"), slot("e")])]
    assert [c.length(r) for r in "cde"] == [6, 4, 6]
    c.check()


def test_pages_of_many_holders_cost_no_more_than_those_of_few():
    """Comparisons of holders' names while a request of 400 pages gets as many holders: as many as there are holders and pages, not their squares."""
    class Name:
        seen = 0

        def __init__(self, i):
            self.i = i

        def __hash__(self):
            return hash(self.i)

        def __eq__(self, other):
            Name.seen += 1
            return isinstance(other, Name) and self.i == other.i

    t = PageTables([PageGroup((0,), 1, 8, 0)], 4, [500], 41)
    names = [Name(i) for i in range(41)]
    t.open(names[0])
    t.reserve(names[0], 1600)
    t.commit(names[0])
    Name.seen = 0
    t.fork_many([(n, names[0]) for n in names[1:]])
    for n in names:
        t.close(n)
    assert Name.seen <= 4 * 41 * 400 and t.pools[0].free_pages == 500


def test_what_the_kernels_count_stays_within_31_bits():
    """Of sizes that are taken: the ends of a walk's keys (a unit's empty tiles counted, and four tiles of 128 asked for ahead), a line's tiles and where the last of its workers
    begins (at most 16 on each of two blocks of 160 multiprocessors).  Tables of nearly 2^31 positions, which passed them, are refused by the entry and by attention_shared_takes alike."""
    lib, null, some = ops.lib(), ctypes.c_void_p(0), 64

    def entry(n, nh, hd, reach):
        args = ctypes.create_string_buffer(ops._SHARED_ARGS.pack(*[some] * 9, some, 0, 4, 4, n, 1, 10, nh, nh, hd, 16, reach // 16, 0.1, 1, some))
        return lib.vk_attention_shared(args, null)

    rng = random.Random(4)
    sizes = [(1, 1, 64, (1 << 31) - 16), (1, 1, 64, 1 << 30), (1, 1, 64, (1 << 30) + 16), (16, 1, 64, (1 << 30) - 1024), (16, 1, 64, (1 << 30) + 16), (256, 8, 128, 1 << 23), (2, 8, 128, 1 << 30), (8, 2, 64, 1 << 30)]
    sizes += [(rng.choice([1, 2, 3, 16, 100, 256]), rng.choice([1, 2, 5, 32, 64]), 64, 16 << rng.randint(0, 26)) for _ in range(300)]
    taken = 0
    for n, nh, hd, reach in sizes:
        assert entry(n, nh, hd, reach) == (-4 if ops.attention_shared_takes(torch.bfloat16, nh, nh, hd, n, reach) else -3), (n, nh, hd, reach)      # -4: no room in the scratch is what stops it
        if ops.attention_shared_takes(torch.bfloat16, nh, nh, hd, n, reach):
            line = n * nh * (-(-reach // 16) + 16)
            assert reach + 16 * 16 + 4 * 128 < 1 << 31 and line + 160 * 2 * 16 * 2 < 1 << 31
            taken += 1
    assert taken > 100 and not ops.attention_shared_takes(torch.bfloat16, 1, 1, 64, 1, (1 << 31) - 16)


def test_a_refused_holder_leaves_a_page_unshared():
    pool = PagePool(2)
    a = pool.alloc("x")
    with pytest.raises(CacheError):
        pool.share(a, "x")
    assert not pool.is_shared(a) and not pool.has_shared
    pool.share(a, "y")
    with pytest.raises(CacheError):
        pool.share(a, "y")
    pool.free(a, "y")
    assert not pool.is_shared(a) and not pool.has_shared and pool.holders(a) == ["x"]
    pool.free(a, "x")
    pool.check()
    assert pool.free_pages == 2


@pytest.mark.parametrize("shape", [(2, 3, 0), (2, 3, 0, 5), (2, 3, 4, 0), (0, 3, 4), (2, 3, 5)])
def test_rows_of_no_numbers_are_not_moved(monkeypatch, shape):
    """An empty row's stride is one number in torch: nothing is launched for it (there is no memory behind it)."""
    calls = []
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0, raising=False)
    monkeypatch.setattr(ops, "_entry", lambda name, types: lambda *a: calls.append(a) or 0)
    arena = torch.zeros(shape)
    assert ops.copy_rows(arena, [0], [2]) is arena
    assert len(calls) == (1 if arena.numel() else 0)
    if arena.numel():
        assert calls[0][1:3] == shape[:2] and calls[0][5] == shape[2] * 4          # layers, rows, bytes a row
    if arena.shape[0]:
        for src, dst in [([0], [3]), ([-1], [1]), ([0, 1], [2])]:
            with pytest.raises(ops.KernelError):
                ops.copy_rows(arena, src, dst)


def test_pairs_may_come_one_by_one(monkeypatch):
    """Any iterable of pairs: the states are moved too."""
    c = CacheManager([StateSpec((3,))], page_size=4, num_pages=4, max_requests=4, dtype=torch.float32, device="cpu")
    moves = []
    monkeypatch.setattr(ops, "copy_rows", lambda arena, src, dst: moves.append((list(src), list(dst))))
    c.open("a")
    c.fork_many((r, "a") for r in "bc")
    c.adopt((r, "a") for r in "cb")
    a, b, d = (c.slot(r) for r in "abc")
    assert moves == [([a, a], [b, d]), ([a, a], [d, b])]
