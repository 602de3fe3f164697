"""The operators of beam search against plain statements in 64 bits: attention over pages held in common, the choice of the best
continuations, moves of cache rows; their edges, and what they refuse."""
import math
import random

import numpy as np
import pytest
import torch

from vitna_anchor_b200 import ops as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    O.lib()
    return O


# -- attention ------------------------------------------------------------------------------------------------------------------------


class Batch:
    """Families of requests over a pool whose unused slots hold NaN: (shared positions, positions of each member's own, its token counted)."""

    def __init__(self, families, nh, nkv, hd, ps, dtype, seed=0, outside=0, pages=None):
        rng = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        self.families, self.nh, self.nkv, self.hd, self.ps, self.dtype = families, nh, nkv, hd, ps, dtype
        tokens = sum(len(own) for _, own in families) + outside
        place = list(range(tokens))
        rng.shuffle(place)
        need = sum(-(-shared // ps) + sum(-(-(shared % ps + n) // ps) + 1 for n in own) for shared, own in families) + 2
        self.pages = pages or need
        free = list(range(self.pages))
        rng.shuffle(free)
        self.tables = [[] for _ in range(tokens)]
        self.pos = [0] * tokens
        self.members, self.starts = [], [0]
        for shared, own in families:
            first = [free.pop() for _ in range(shared // ps)]
            tail = shared % ps
            for n in own:
                t = place[len(self.members)]
                self.members.append(t)
                # a shared end inside a page: the members' pages there are different ones with the same content
                self.tables[t] = first + [free.pop() for _ in range(-(-(tail + n) // ps))]
                self.pos[t] = shared + n - 1
            self.starts.append(len(self.members))
        self.shared = [s for s, _ in families]
        for t in place[len(self.members):]:              # tokens in no family
            self.tables[t] = [free.pop() if free else 0]
        self.cache = torch.full((self.pages, 2, nkv, ps, hd), float("nan"), dtype=dtype)
        self.q = (torch.randn((tokens, nh * hd), generator=g) * 1.5).to(dtype)
        for (shared, own), lo in zip(families, self.starts):
            kv = torch.randn((shared, 2, nkv, hd), generator=g).to(dtype)
            for t in self.members[lo:lo + len(own)]:
                n = self.pos[t] + 1
                mine = torch.cat([kv, torch.randn((n - shared, 2, nkv, hd), generator=g).to(dtype)])
                at = torch.arange(n)
                page = torch.tensor(self.tables[t])[at // ps]
                self.cache[page, :, :, at % ps] = mine
        self.maxb = max(max(len(t) for t in self.tables), 1) + 2

    def device(self, wide=True):
        """wide: block tables so wide that the call does not walk every member by itself (where it can)."""
        i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")      # noqa: E731
        if wide:
            self.maxb = max(self.maxb, (260 << 20) // (max(1, len(self.members)) * self.ps * self.nkv * self.hd * 4) + 1)
        self.d = dict(q=self.q.cuda(), cache=self.cache.cuda(), tables=i([t + [0x7fffffff] * (self.maxb - len(t)) for t in self.tables]), seg=i(list(range(len(self.pos)))),
                      pos=i(self.pos), members=i(self.members).reshape(-1), starts=i(self.starts), shared=i(self.shared))
        self.d["out"] = torch.full_like(self.d["q"], 7.0)
        return self

    def run(self, ops, scratch=None):
        d = self.d
        if scratch is None:
            scratch = torch.zeros(ops.attention_shared_scratch_bytes(max(1, len(self.members)), self.nh, self.nkv, self.hd), dtype=torch.uint8, device="cuda")
        ops.attention_shared(d["q"], d["cache"], d["tables"], d["seg"], d["pos"], d["members"], d["starts"], d["shared"], d["out"], scratch, self.nh, self.nkv,
                             self.hd, self.hd ** -0.5)
        return d["out"]

    def want(self):
        """(the outputs in 64 bits, how far each may be off): half a step of the output's type; the scores' sums of hd products in 32 bits, at most hd steps of 2^-23 of the
        sum of their absolute values, move p by that much relative and the output by twice that times the largest value; p as two bfloat16 parts and as 2^x by the
        special-function unit, 2^-16 together, sums over n keys in blocks of at most 32 and parts, 64 steps of 2^-23."""
        reps, out, tol = self.nh // self.nkv, torch.full(self.q.shape, 7.0, dtype=torch.float64), torch.zeros(self.q.shape, dtype=torch.float64)
        half = torch.finfo(self.dtype).eps / 2
        for t in self.members:
            at = torch.arange(self.pos[t] + 1)
            kv = self.cache[torch.tensor(self.tables[t])[at // self.ps], :, :, at % self.ps].double()
            k, v = (kv[:, i].repeat_interleave(reps, dim=1) for i in (0, 1))
            q = self.q[t].double().view(self.nh, self.hd)
            z = torch.einsum("phd,hd->hp", k, q) * self.hd ** -0.5
            size = (torch.einsum("phd,hd->hp", k.abs(), q.abs()) * self.hd ** -0.5).amax(1)
            o = torch.einsum("hp,phd->hd", torch.softmax(z, 1), v)
            slack = (2 * self.hd * 2.0 ** -23 * size + 2.0 ** -16 + 64 * 2.0 ** -23) * v.abs().amax((0, 2))
            out[t] = o.reshape(-1)
            tol[t] = (half * o.abs() + slack[:, None]).reshape(-1)
        return out, tol

    def check(self, ops, scratch=None):
        got = self.run(ops, scratch).double().cpu()
        want, tol = self.want()
        off = (got - want).abs() - tol
        assert not bool(torch.isnan(got).any()) and float(off.max()) <= 0, f"{float(off.max())} beyond the tolerance"


F32, BF16 = torch.float32, torch.bfloat16
# families, heads, kv heads, dim, page
SHAPES = [
    ([(0, [1])], 1, 1, 8, 16),                                             # one token at position 0
    ([(0, [1]), (0, [33])], 4, 2, 64, 16),                                 # families of one, nothing shared
    ([(32, [1, 1])], 9, 3, 64, 16),                                        # own parts of one key
    ([(512, [24, 1, 7, 19])], 9, 3, 64, 16),
    ([(528, [24, 65, 130, 19, 40, 1, 200, 33])], 32, 32, 64, 16),
    ([(1000, [3, 40]), (0, [77, 5]), (250, [9]), (96, [1, 2, 3, 4, 5])], 15, 5, 64, 16),     # a shared end inside a page; nothing shared; one member
    ([(700, list(range(1, 65)))], 6, 2, 64, 16),                           # 192 rows over three tiles
    ([(130, [5] * 23)], 3, 1, 64, 5),                                      # pages of an odd size, a last tile of two members
    ([(2049, [17, 300])], 16, 2, 128, 16),
    ([(333, [9] * 9)], 64, 1, 128, 32),                                    # all heads read one key-value head
    ([(64, [2, 30, 31])], 40, 2, 64, 16),                                  # 20 heads a key-value head: two tiles of own heads
    ([(100, [20, 3])], 4, 2, 40, 8), ([(100, [20, 3, 8])], 2, 2, 96, 12), ([(77, [20, 3])], 4, 1, 256, 1),
    ([], 4, 2, 64, 16),
    ([(5000, [1, 1, 1])], 2, 1, 64, 64),
    ([(48, [4, 5])] * 40, 4, 4, 64, 16),                                   # many small families
    ([(16, [3])] * 100 + [(160, [7] * 156)], 2, 2, 64, 16),                # 256 tokens
]


@pytest.mark.parametrize("dtype,wide", [(BF16, True), (BF16, False), (F32, True), (F32, False)])
@pytest.mark.parametrize("n", range(len(SHAPES)))
def test_attention_shared(ops, dtype, wide, n):
    families, nh, nkv, hd, ps = SHAPES[n]
    if not families:
        b = Batch([(16, [3])], nh, nkv, hd, ps, dtype, outside=2).device(wide)
        b.d["members"], b.d["starts"], b.d["shared"] = b.d["members"][:0], b.d["starts"][:1], b.d["shared"][:0]
        assert bool((b.run(ops) == 7).all())                               # no family: nothing is written
        return
    Batch(families, nh, nkv, hd, ps, dtype, seed=n).device(wide).check(ops)


@pytest.mark.parametrize("dtype,hd,wide", [(BF16, 64, True), (BF16, 128, True), (BF16, 64, False), (BF16, 128, False), (F32, 64, True), (F32, 64, False)])
def test_attention_shared_random_families(ops, dtype, hd, wide):
    """Many layouts through ONE scratch of exactly the bytes of the largest, with guards around it."""
    rng = random.Random(11)
    most = ops.attention_shared_scratch_bytes(128, 8, 8, hd)
    guarded = torch.full((most + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    scratch = guarded[2048:2048 + most]
    scratch.zero_()
    for n in range(12):
        nkv = rng.choice([1, 2, 8])
        nh = nkv * rng.choice([1, 2, 3, 8] if nkv == 1 else [1])
        fams = [(rng.choice([0, rng.randint(1, 900)]), [rng.randint(1, 90) for _ in range(rng.randint(1, 12))]) for _ in range(rng.randint(1, 9))]
        Batch(fams, nh, nkv, hd, rng.choice([16, 8, 13]), dtype, seed=n, outside=rng.randint(0, 3)).device(wide).check(ops, scratch)
    assert bool((guarded[:2048] == 0x5A).all()) and bool((guarded[2048 + most:] == 0x5A).all())


@pytest.mark.parametrize("wide", [True, False])
def test_attention_shared_claims_that_do_not_fit(ops, wide):
    """shared beyond the smallest position is cut there; an empty family, tokens that are not there, starts that go back and starts beyond
    the list are nothing."""
    b = Batch([(64, [5, 9])], 4, 2, 64, 16, BF16, outside=3).device(wide)
    want, tol = b.want()
    i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")          # noqa: E731
    m = b.members
    # at least one member ends at position 68: its own key is never a common one, and the tables agree up to 64 only when shared says so
    for members, starts, shared in [(m, [0, 2], [64]), (m, [0, 0, 2, 2], [500, 64, 9]), ([-4] + m + [999], [0, 4], [64]), (m, [0, 2, 1], [64, 64]),
                                    (m, [-5, 77], [64]), (m, [0, 2], [-8])]:
        b.d["members"], b.d["starts"], b.d["shared"] = i(members), i(starts), i(shared)
        b.d["out"].fill_(7.0)
        got = b.run(ops, torch.zeros(ops.attention_shared_scratch_bytes(8, 4, 2, 64), dtype=torch.uint8, device="cuda")).double().cpu()
        assert float(((got - want).abs() - tol).max()) <= 0
    same = Batch([(0, [40, 40])], 4, 2, 64, 16, BF16).device(wide)               # two names for one request: all it has is common, but for the token's own key
    t = same.members
    same.d["tables"][t[1]] = same.d["tables"][t[0]]
    same.d["q"][t[1]] = same.d["q"][t[0]]
    same.tables[t[1]], same.q[t[1]] = same.tables[t[0]], same.q[t[0]]
    same.d["shared"] = i([4000])
    same.check(ops)


@pytest.mark.parametrize("wide", [True, False])
def test_attention_shared_bad_blocks_count_as_zeros(ops, wide):
    b = Batch([(64, [20, 9])], 4, 2, 64, 16, BF16)
    b.cache[b.tables[b.members[0]][1]] = 0
    b.cache[b.tables[b.members[1]][4]] = 0
    b.device(wide)
    b.d["tables"][b.members[0], 1] = b.pages
    b.d["tables"][b.members[1], 1] = b.pages
    b.d["tables"][b.members[1], 4] = -7
    b.check(ops)


@pytest.mark.parametrize("wide", [True, False])
def test_attention_shared_of_scores_without_a_number(ops, wide):
    """Scores of -inf weigh nothing; a token all of whose scores are -inf, or one of them NaN, has no number, and the others keep theirs."""
    b = Batch([(128, [40, 9, 30])], 4, 2, 64, 16, BF16)
    b.q.abs_()
    own = b.tables[b.members[0]][8:]
    b.cache[b.tables[b.members[0]][2], 0, :, 3] = -math.inf       # one shared key
    b.cache[own[1], 0, 0, 5] = float("nan")                       # one key of the first member, the first key-value head
    got = b.device(wide).run(ops).double().cpu().view(-1, 4, 64)
    want, tol = (x.view(-1, 4, 64) for x in b.want())
    assert bool(torch.isnan(got[b.members[0], :2]).all()) and bool(torch.isnan(want[b.members[0], :2]).all())
    tol = torch.where(torch.isfinite(tol), tol, torch.tensor(2.0 ** -6).double())      # the bound's sums are over infinite keys
    for t, heads in [(b.members[0], slice(2, 4)), (b.members[1], slice(0, 4)), (b.members[2], slice(0, 4))]:
        assert float(((got[t, heads] - want[t, heads]).abs() - tol[t, heads]).max()) <= 0


MANY = [  # families whose rows fill a tile of 128 or most of it, heads of 128: families, heads, kv heads, page
    ([(64, [3] * 5)], 16, 1, 16),                                          # one tile of keys
    ([(65, [3] * 5)], 16, 1, 16), ([(128, [1] * 8)], 16, 1, 64),
    ([(1000, [2, 70, 9, 1, 33])], 14, 1, 16),                              # 70 rows
    ([(4097, [5] * 16)], 16, 2, 16),                                       # 128 rows
    ([(777, list(range(1, 30)))], 8, 1, 13),                               # 232 rows, a last tile of few, pages of an odd size
    ([(300, [4] * 9), (1200, [8] * 12), (17, [40] * 3), (0, [9])], 16, 2, 8),
    ([(2000, [3] * 80), (500, [7] * 100)], 2, 2, 16),                      # 80 and 100 members of one head
]


@pytest.mark.parametrize("n", range(len(MANY)))
def test_attention_shared_of_many_rows(ops, n):
    families, nh, nkv, ps = MANY[n]
    Batch(families, nh, nkv, 128, ps, BF16, seed=40 + n).device().check(ops)


def test_attention_shared_of_many_rows_far_in_a_large_pool(ops):
    """Element offsets beyond 2^31."""
    b = Batch([(200, [5] * 9)], 32, 4, 128, 16, BF16)
    b.device()
    pages = 140000
    big = torch.empty((pages, 2, 4, 16, 128), dtype=BF16, device="cuda")
    big[pages - b.pages:] = b.d["cache"]
    b.d["cache"] = big
    b.d["tables"] = torch.where(b.d["tables"] < b.pages, b.d["tables"] + (pages - b.pages), b.d["tables"])
    b.check(ops)


def test_attention_shared_of_many_rows_whose_maxima_rise(ops):
    """Every tile's scores are far above the ones before, for some rows, and below for others; one tile weighs nothing at all."""
    b = Batch([(1024, [20] * 8)], 16, 1, 128, 16, BF16, seed=7)
    first = b.tables[b.members[0]][:64]
    along = b.q[b.members[0], :128].float()
    along /= along.norm()
    for i, page in enumerate(first):
        b.cache[page, 0] = (b.cache[page, 0].float() + along * (i - 20)).to(BF16)
    b.cache[first[8:12], 0] = -math.inf
    b.q.abs_()
    got = b.device().run(ops).double().cpu()
    want, tol = b.want()
    tol = torch.where(torch.isfinite(tol), tol, torch.tensor(2.0 ** -6).double())      # the bound's sums are over infinite keys
    assert float(((got - want).abs() - tol).max()) <= 0


def test_attention_shared_of_many_rows_bad_blocks_and_no_number(ops):
    b = Batch([(640, [20, 9, 3, 3, 3, 3])], 16, 1, 128, 16, BF16)
    b.cache[b.tables[b.members[0]][3]] = 0
    b.device()
    for t, bad in zip(b.members, (-1, b.pages, 1 << 30, -(1 << 31), b.pages, -7)):
        b.d["tables"][t, 3] = bad
    b.check(ops)
    b = Batch([(640, [20, 9, 3, 3, 3, 3])], 16, 1, 128, 16, BF16)
    b.cache[b.tables[b.members[0]][3], 0, 0, 2] = float("nan")             # a common key: nobody has a number
    got = b.device().run(ops)
    assert bool(torch.isnan(got[b.members]).all())


def test_attention_shared_of_many_rows_replayed_on_two_streams(ops):
    """Two calls at once on two streams, whose blocks both want tensor memory; a captured one follows other lengths."""
    bs = [Batch([(3000, [5, 60, 17, 9, 30]), (0, [9])], 16, 1, 128, 16, BF16, seed=3 + k).device() for k in (0, 1)]
    streams, graphs = [torch.cuda.Stream() for _ in bs], []
    scratch = [torch.zeros(ops.attention_shared_scratch_bytes(6, 16, 1, 128), dtype=torch.uint8, device="cuda") for _ in bs]
    for b, room in zip(bs, scratch):
        b.run(ops, room)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            for _ in range(8):
                b.run(ops, room)
        b.pos = [max(0, p - 3) if t in b.members else p for t, p in enumerate(b.pos)]
        b.d["pos"].copy_(torch.tensor(b.pos, dtype=torch.int32))
        b.d["shared"].copy_(torch.tensor([2990, 0], dtype=torch.int32))
        b.d["out"].fill_(7.0)
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    ops.check_device_errors()
    for b in bs:
        want, tol = b.want()
        assert float(((b.d["out"].double().cpu() - want).abs() - tol).max()) <= 0


@pytest.mark.parametrize("tile,shared", [(0, 4000), (1, 30000)])      # of 4,000 keys a group of warps has one tile at most, of 30,000 (over at most 148 blocks) three or more
def test_attention_shared_gives_up_a_wait_and_says_so(ops, tile, shared):
    """A tile of keys whose scores are never told of (a hook for this test; nothing faults): the waits run out after the 5 ms set here, the kernel returns by itself with its
    tensor memory freed, the error word is set, and the next launch is right."""
    b = Batch([(shared, [5] * 16)], 16, 2, 128, 16, BF16, seed=2).device()
    ops.set_wait_limit_ms(5.0)
    try:
        ops.skip_stage_once("attention_shared", tile)
        b.run(ops)
        torch.cuda.synchronize()
        assert ops.device_error_code() == 81
        with pytest.raises(ops.KernelGaveUp):
            ops.check_device_errors()
    finally:
        ops.set_wait_limit_ms(0)
    b.check(ops)
    ops.check_device_errors()


@pytest.mark.parametrize("dtype,wide", [(BF16, True), (BF16, False), (F32, True), (F32, False)])
def test_attention_shared_of_a_token_named_twice(ops, dtype, wide):
    """In one family and in two: the token has its one result."""
    for members, starts, shared in [([0, 1, 0], [0, 3], [96]), ([0, 1, 1, 0], [0, 2, 4], [96, 48])]:
        b = Batch([(96, [20, 9])], 6, 2, 64, 16, dtype, seed=4)
        place = b.members
        b.members = [place[m] for m in members]
        b.device(wide)
        b.d["starts"], b.d["shared"] = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (starts, shared))
        b.check(ops)


def test_attention_shared_two_graphs_through_one_scratch(ops):
    """Captured apart, replayed in turns on one stream."""
    a, b = Batch([(400, [5, 60, 17])], 6, 2, 64, 16, BF16, seed=1).device(), Batch([(64, [9, 30]), (128, [70, 3])], 6, 2, 64, 16, BF16, seed=2).device()
    scratch = torch.full((ops.attention_shared_scratch_bytes(4, 6, 2, 64),), 0x7F, dtype=torch.uint8, device="cuda")
    graphs = []
    for x in (a, b):
        x.run(ops, scratch)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            x.run(ops, scratch)
        x.d["out"].fill_(7.0)
    for n in (0, 1, 0, 1, 1, 0):
        graphs[n].replay()
    for x in (a, b):
        want, tol = x.want()
        assert float(((x.d["out"].double().cpu() - want).abs() - tol).max()) <= 0


def test_attention_shared_far_in_a_large_pool(ops):
    """Element offsets beyond 2^31."""
    b = Batch([(96, [5, 40])], 32, 32, 64, 16, BF16)
    b.device()
    small, pages = b.d["cache"], 40000
    big = torch.empty((pages, 2, 32, 16, 64), dtype=BF16, device="cuda")
    big[pages - b.pages:] = small
    b.d["cache"] = big
    b.d["tables"] = torch.where(b.d["tables"] < b.pages, b.d["tables"] + (pages - b.pages), b.d["tables"])
    b.check(ops)


@pytest.mark.parametrize("wide", [True, False])
def test_attention_shared_replayed_and_on_another_stream(ops, wide):
    b = Batch([(200, [5, 60, 17]), (0, [9])], 6, 2, 64, 16, BF16, seed=3).device(wide)
    scratch = torch.zeros(ops.attention_shared_scratch_bytes(4, 6, 2, 64), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = b.run(ops, scratch).clone()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run(ops, scratch)
    b.d["out"].fill_(7.0)
    graph.replay()
    assert torch.equal(b.d["out"], first)                                    # the same parts in the same order: the same bits
    b.pos = [max(0, p - 3) if t in b.members else p for t, p in enumerate(b.pos)]       # other lengths, a shorter common part
    b.d["pos"].copy_(torch.tensor(b.pos, dtype=torch.int32))
    b.d["shared"].copy_(torch.tensor([150, 0], dtype=torch.int32))
    graph.replay()
    want, tol = b.want()
    assert float(((b.d["out"].double().cpu() - want).abs() - tol).max()) <= 0


def test_attention_shared_refuses(ops):
    b = Batch([(64, [5, 9])], 4, 2, 64, 16, BF16).device()
    small = torch.zeros(64, dtype=torch.uint8, device="cuda")
    with pytest.raises(ops.KernelError, match="scratch"):
        b.run(ops, small)
    assert not ops.attention_shared_takes(torch.float16, 4, 2, 64) and not ops.attention_shared_takes(BF16, 5, 2, 64)
    assert not ops.attention_shared_takes(BF16, 4, 2, 260) and not ops.attention_shared_takes(BF16, 4, 2, 12) and not ops.attention_shared_takes(BF16, 130, 2, 64)
    assert not ops.attention_shared_takes(BF16, 4, 2, 64, 257) and ops.attention_shared_takes(F32, 4, 2, 12)
    for name, value in [("starts", b.d["starts"][:1]), ("pos", b.d["pos"][:1]), ("members", b.d["members"].long()), ("out", b.d["out"].float()),
                        ("q", b.d["q"].t()), ("cache", b.d["cache"][:, :1]), ("tables", b.d["tables"].cpu())]:
        kept = b.d[name]
        b.d[name] = value
        with pytest.raises(ops.KernelError):
            b.run(ops)
        b.d[name] = kept
    b.check(ops)


# -- the choice ---------------------------------------------------------------------------------------------------------------------------


def choose(logits, scores, beams, keep):
    x = logits.cpu().numpy().astype(np.float64)
    s = scores.cpu().numpy().astype(np.float64)
    R, V = x.shape
    with np.errstate(all="ignore"):
        top = x.max(1, keepdims=True)
        lse = top + np.log(np.exp(x - top).sum(1, keepdims=True))
        c = s[:, None] + x - lse
    dead = ~np.isfinite(lse[:, 0]) | ~np.isfinite(s)
    c[dead] = -np.inf
    c = c.reshape(R // beams, beams * V)
    at = np.argsort(-c, axis=1, kind="stable")[:, :keep]
    return np.take_along_axis(c, at, 1), at // V, at % V


def select(ops, logits, scores, beams, keep, scratch=None):
    R, V = logits.shape
    out = (torch.full((R // beams, keep), 5.0, device="cuda"), torch.full((R // beams, keep), -9, dtype=torch.int32, device="cuda"),
           torch.full((R // beams, keep), -9, dtype=torch.int32, device="cuda"))
    if scratch is None:
        scratch = torch.zeros(ops.beam_select_scratch_bytes(R, V, keep), dtype=torch.uint8, device="cuda")
    return ops.beam_select(logits, scores, beams, keep, out, scratch)


def check_choice(ops, logits, scores, beams, keep, scratch=None):
    got = select(ops, logits, scores, beams, keep, scratch)
    best, parent, token = choose(logits, scores, beams, keep)
    assert np.array_equal(got[1].cpu().numpy(), parent) and np.array_equal(got[2].cpu().numpy(), token)
    b = got[0].cpu().numpy().astype(np.float64)
    live = np.isfinite(best)
    assert np.array_equal(live, np.isfinite(b)) and np.all(b[~live] == -np.inf)
    # half a step of float32, and the sum of exponentials in 32 bits: V terms in runs of 32 and a tree, 40 steps of 2^-23 of it, so of the logarithm absolutely
    assert np.all(np.abs(b[live] - best[live]) <= 2.0 ** -24 * np.abs(best[live]) + 40 * 2.0 ** -23)


CHOICES = [(1, 1, 1, 1), (1, 1, 1000, 1), (1, 4, 49152, 8), (3, 5, 50257, 10), (8, 8, 49152, 16), (2, 32, 131072, 64), (1, 64, 5003, 128), (7, 3, 2, 6), (2, 2, 64, 128),
           (64, 1, 4097, 2), (1, 2, 262144, 128), (1, 16, 8192, 33), (300, 1, 999, 17), (1, 1, 200, 128), (4, 16, 32000, 100)]


@pytest.mark.parametrize("requests,beams,vocab,keep", CHOICES)
def test_beam_select(ops, requests, beams, vocab, keep):
    g = torch.Generator(device="cuda").manual_seed(vocab + keep)
    logits = torch.randn((requests * beams, vocab), generator=g, device="cuda") * 3
    scores = -20 - 5 * torch.rand(requests * beams, generator=g, device="cuda")
    check_choice(ops, logits, scores, beams, keep)
    # values of few steps: many of a row are equal, and the lowest token is first
    check_choice(ops, (logits * 2).round() / 2, scores, beams, keep)


def test_beam_select_equal_rows_and_first_step(ops):
    row = (torch.randn((1, 5003), device="cuda") * 4).round() / 4
    logits = row.repeat(6, 1)
    check_choice(ops, logits, torch.full((6,), -3.25, device="cuda"), 6, 20)              # equal beams: the lowest is first, wherever a row begins
    scores = torch.full((6,), -math.inf, device="cuda")
    scores[0] = scores[3] = 0.0
    check_choice(ops, logits, scores, 3, 20)                                            # one beam of three lives
    check_choice(ops, torch.zeros((4, 5003), device="cuda"), torch.zeros(4, device="cuda"), 2, 9)
    check_choice(ops, row, torch.zeros(1, device="cuda"), 1, 128)


def test_beam_select_rows_without_a_number(ops):
    g = torch.Generator(device="cuda").manual_seed(5)
    logits = torch.randn((12, 3000), generator=g, device="cuda")
    logits[1] = -math.inf
    logits[2, 77] = float("nan")
    logits[3, 2999] = math.inf
    logits[4, 9:] = -math.inf                                            # fewer live tokens than are kept
    logits[7] = torch.finfo(torch.float32).min
    logits[8, 1:] = torch.finfo(torch.float32).min
    scores = -torch.rand(12, generator=g, device="cuda")
    scores[5], scores[6], scores[9] = float("nan"), math.inf, -math.inf
    for beams, keep in [(12, 128), (12, 24), (1, 20), (3, 60), (2, 128)]:
        check_choice(ops, logits, scores, beams, keep)
    check_choice(ops, torch.full((4, 700), -math.inf, device="cuda"), torch.zeros(4, device="cuda"), 2, 30)


@pytest.mark.parametrize("keep", [3, 16, 17, 50, 100, 128])
def test_beam_select_values_laid_out_against_the_groups(ops, keep):
    """All the largest values where one thread, or one thread's part of every block, has them; values that ascend and descend."""
    V = 40000
    x = torch.randn((2, V), device="cuda")
    i = torch.arange(V, device="cuda")
    one = ((i // 4) % 256 == 37) | ((i // 4) % 256 == 5)
    x[:, one] += 100
    check_choice(ops, x, torch.zeros(2, device="cuda"), 2, keep)
    x[:, (i // 4) % 256 < 8] += 300
    check_choice(ops, x, torch.zeros(2, device="cuda"), 1, keep)
    up = torch.linspace(-5, 5, V, device="cuda").repeat(2, 1)
    check_choice(ops, up, torch.tensor([0.0, -1e-3], device="cuda"), 2, keep)
    check_choice(ops, up.flip(1).contiguous(), torch.tensor([0.0, -1e-3], device="cuda"), 2, keep)


@pytest.mark.parametrize("size", [1e-6, 1e3, 3e4, 1e30])
def test_beam_select_of_small_and_large_logits(ops, size):
    """Beyond what the bounds' 16 bits tell apart.  The scores' gap of 1.5 is far beyond the error of a row's sum, or far below a step of its logits."""
    x = torch.randn((4, 30000), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda") * size
    for beams, keep in [(1, 3), (1, 128), (2, 9)]:
        got = select(ops, x, torch.tensor([0.0, -1.5] * 2, device="cuda"), beams, keep)
        best, parent, token = choose(x, torch.tensor([0.0, -1.5] * 2), beams, keep)
        if beams == 1 or size > 1:
            assert np.array_equal(got[1].cpu().numpy(), parent) and np.array_equal(got[2].cpu().numpy(), token)
        b = got[0].cpu().numpy().astype(np.float64)
        assert np.all(np.abs(b - best) <= 2.0 ** -24 * np.abs(best) + 40 * 2.0 ** -23)


def test_beam_select_scores_in_place(ops):
    """A step's sums over the last step's: the scores are read before any of them is written."""
    g = torch.Generator(device="cuda").manual_seed(21)
    logits = torch.randn((24, 9000), generator=g, device="cuda") * 3
    scores = -torch.rand(24, generator=g, device="cuda")
    best, parent, token = choose(logits, scores, 8, 8)
    out = (scores.view(3, 8), torch.empty((3, 8), dtype=torch.int32, device="cuda"), torch.empty((3, 8), dtype=torch.int32, device="cuda"))
    ops.beam_select(logits, scores, 8, 8, out, torch.zeros(ops.beam_select_scratch_bytes(24, 9000, 8), dtype=torch.uint8, device="cuda"))
    assert np.array_equal(out[1].cpu().numpy(), parent) and np.array_equal(out[2].cpu().numpy(), token)
    assert np.all(np.abs(scores.view(3, 8).cpu().numpy() - best) <= 2.0 ** -24 * np.abs(best) + 40 * 2.0 ** -23)


def test_beam_select_one_strong_row(ops):
    """Everything that is kept comes from the last beam."""
    logits = torch.randn((32, 70000), device="cuda")
    scores = torch.full((32,), -500.0, device="cuda")
    scores[31] = -1.0
    check_choice(ops, logits, scores, 32, 64)
    check_choice(ops, logits, scores, 32, 128)


def test_beam_select_apart_replayed_and_reused(ops):
    g = torch.Generator(device="cuda").manual_seed(9)
    wide = torch.randn((16, 5101), generator=g, device="cuda")
    scores = -torch.rand(16, generator=g, device="cuda")
    scratch = torch.zeros(ops.beam_select_scratch_bytes(64, 50000, 128), dtype=torch.uint8, device="cuda")
    check_choice(ops, wide[:, 1:5001], scores, 4, 8, scratch)                       # rows apart, beginning anywhere
    check_choice(ops, wide[::2, :5000], scores[::2].contiguous(), 4, 8, scratch)
    check_choice(ops, torch.randn((64, 50000), generator=g, device="cuda"), -torch.rand(64, generator=g, device="cuda"), 64, 128, scratch)
    x = torch.randn((8, 6000), generator=g, device="cuda")
    out = select(ops, x, scores[:8], 8, 16, scratch)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.beam_select(x, scores[:8], 8, 16, out, scratch)
    x.copy_(torch.randn((8, 6000), generator=g, device="cuda"))
    graph.replay()
    best, parent, token = choose(x, scores[:8], 8, 16)
    assert np.array_equal(out[1].cpu().numpy(), parent) and np.array_equal(out[2].cpu().numpy(), token)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check_choice(ops, x, scores[:8], 2, 5)


def test_beam_select_refuses(ops):
    x, s = torch.zeros((8, 100), device="cuda"), torch.zeros(8, device="cuda")
    for kw in [dict(beams=3), dict(beams=0), dict(keep=0), dict(keep=129), dict(beams=1, keep=101), dict(scores=s[:7]), dict(logits=x.t()), dict(logits=x.double()),
               dict(scratch=torch.zeros(16, dtype=torch.uint8, device="cuda"))]:
        a = dict(logits=x, scores=s, beams=4, keep=8, scratch=None) | kw
        with pytest.raises(ops.KernelError):
            if a["beams"] < 1 or a["logits"].shape[0] % a["beams"]:
                out = tuple(torch.empty((2, 8), dtype=d, device="cuda") for d in (torch.float32, torch.int32, torch.int32))
                ops.beam_select(a["logits"], a["scores"], a["beams"], a["keep"], out, torch.zeros(100000, dtype=torch.uint8, device="cuda"))
            else:
                select(ops, a["logits"], a["scores"], a["beams"], a["keep"], a["scratch"])
    with pytest.raises(ops.KernelError):
        ops.beam_select(x, s, 4, 8, (torch.empty((2, 8), device="cuda"), torch.empty((2, 7), dtype=torch.int32, device="cuda"), torch.empty((2, 8), dtype=torch.int32, device="cuda")),
                        torch.zeros(1 << 20, dtype=torch.uint8, device="cuda"))


# -- moves of rows ---------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("layers,rows,shape,dtype", [(1, 2, (1,), torch.uint8), (30, 40, (2, 3, 16, 64), BF16), (3, 300, (5, 7), BF16), (4, 9, (10007,), F32), (2, 8, (65537,), torch.uint8),
                                                     (1, 8, (3, 3), torch.float64), (2, 6, (300, 1001), F32)])
@pytest.mark.parametrize("apart", [False, True])
def test_copy_rows(ops, layers, rows, shape, dtype, apart):
    whole = torch.randint(0, 100, (layers, rows + 1, *shape), device="cuda").to(dtype)
    arena = whole[:, 1:] if apart else whole[:, 1:].contiguous()
    rng = random.Random(rows)
    order = list(range(rows))
    rng.shuffle(order)
    for moves in {1, rows // 2, min(3, rows // 2)}:
        dst, src = order[:moves], [rng.choice(order[moves:]) for _ in range(moves)]
        before = whole.clone()
        want = arena.clone()
        want[:, dst] = want[:, src]
        assert ops.copy_rows(arena, src, dst) is arena
        assert torch.equal(arena, want)
        if apart:
            assert torch.equal(whole[:, 0], before[:, 0])


def test_copy_rows_offsets_beyond_32_bits(ops):
    arena = torch.empty((2, 5000, 1 << 19), dtype=torch.uint8, device="cuda")
    arena[:, 3] = 7
    arena[:, 4999] = 1
    ops.copy_rows(arena, [3], [4999])
    assert bool((arena[:, 4999] == 7).all())


def test_copy_rows_replayed(ops):
    arena = torch.arange(24, device="cuda", dtype=torch.int32).reshape(2, 4, 3).contiguous()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_rows(arena, [0, 0], [2, 3])
    arena[:, 0] = 99
    graph.replay()
    assert bool((arena[:, 2:] == 99).all()) and not bool((arena[:, 1] == 99).any())


def test_copy_rows_refuses(ops):
    arena = torch.arange(60, device="cuda").reshape(2, 6, 5).contiguous()
    kept = arena.clone()
    for src, dst in [([0], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [6]), ([6], [0]), ([-1], [0]), ([0], [-1]), ([0, 1], [2])]:
        with pytest.raises(ops.KernelError):
            ops.copy_rows(arena, src, dst)
    for bad in [arena.cpu(), arena.transpose(1, 2), arena[0, 0], arena[:1, :1].expand(2, 6, 5), arena[:, :, ::2]]:
        with pytest.raises(ops.KernelError):
            ops.copy_rows(bad, [0], [1])
    assert ops.copy_rows(arena, [], []) is arena and torch.equal(arena, kept)
