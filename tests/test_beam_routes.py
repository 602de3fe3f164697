"""Where a decode step's attention goes when its requests hold pages in common; no GPU is needed."""
from types import SimpleNamespace

import pytest
import torch

from vitna_anchor_b200 import ops


@pytest.fixture
def went(monkeypatch):
    """Which attention a call reaches: every one is replaced by a note of its name."""
    names = []
    for name in ["attention_shared", "attention_decode", "attention_rows", "attention_prefill"]:
        monkeypatch.setattr(ops, name, lambda *a, _name=name, **k: names.append(_name))
    for name in ["attention_shared_scratch_bytes", "attention_decode_scratch_bytes"]:
        monkeypatch.setattr(ops, name, lambda *a: 16)
    return names


def _step(dtype, hd, context, members=True, window=0, tokens=4, nh=4, nkv=2, page=16):
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32)      # noqa: E731
    meta = SimpleNamespace(block_tables=ints(tokens, 1).expand(tokens, context // page), members=ints(tokens) if members else None, starts=ints(tokens + 1), shared=ints(tokens))
    ws = SimpleNamespace(max_context=context, max_segments=tokens, max_tokens=64, flat=lambda name, n, dtype, zero=False: torch.zeros(n, dtype=dtype))
    ctx = SimpleNamespace(num_dec=tokens, num_pre=0, num_tokens=tokens, pre_tiles=None, pre_tiles_big=None, pre_tokens=None, dec_tokens=None, workspace=ws, token_seg=ints(tokens),
                          positions=ints(tokens), max_context=context)
    q = torch.zeros(tokens, nh * hd, dtype=dtype)
    ops.attention(q, torch.zeros(3, 2, nkv, page, hd, dtype=dtype), meta, ctx, torch.empty_like(q), nh, nkv, hd, 0.1, window)


@pytest.mark.parametrize("context", [256, 32768, 32784, 65536, 131072, 1 << 20])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_common_pages_are_read_once_at_every_context(went, hd, context):
    _step(torch.bfloat16, hd, context)
    assert went == ["attention_shared"]


@pytest.mark.parametrize("kw,name", [
    (dict(context=32768, members=False), "attention_decode"), (dict(context=32784, members=False), "attention_rows"), (dict(context=256, window=64), "attention_decode"),
    (dict(context=65536, window=64), "attention_rows"), (dict(context=256, tokens=257), "attention_decode"), (dict(context=65536, tokens=257), "attention_rows"),
    (dict(context=256, dtype=torch.float32), "attention_rows"), (dict(context=65536, dtype=torch.float32), "attention_rows")])
def test_the_other_steps_go_where_they_went(went, kw, name):
    _step(**{"dtype": torch.bfloat16, "hd": 64, **kw})
    assert went == [name]


@pytest.mark.parametrize("context", [256, 65536])
def test_float32_reads_common_pages_once_in_the_fast_routing_alone(went, context):
    before = ops.set_float32_exact(False)
    try:
        _step(torch.float32, 64, context)
    finally:
        ops.set_float32_exact(before)
    assert went == ["attention_shared"]


class _Builder:
    """A ContextBuilder over tables alone, on the host."""

    def __new__(cls, monkeypatch, groups, page_size=4, requests=6, model_len=64, dtype=torch.bfloat16, **kw):
        from vitna_anchor_b200.cache import CacheManager
        from vitna_anchor_b200.engine import context
        staging = context._Staging
        monkeypatch.setattr(context, "_Staging", lambda n, pinned: staging(n, False))
        monkeypatch.setattr(context.ContextBuilder, "_send", lambda self, st, words: self.meta_dev[:words].copy_(st.host[:words]))
        cache = CacheManager(groups, page_size=page_size, num_pages=200, max_requests=requests, dtype=dtype, device="cpu", allocate=False)
        return context.ContextBuilder(cache, dtype, None, max_batch_tokens=32, max_segments=requests, max_model_len=model_len, device="cpu", **kw)


def _advance(cache, rid, n):
    cache.reserve_step([(rid, n)])
    cache.commit_step([(rid, n)])


@pytest.mark.parametrize("build", ["build", "build_decode"])
def test_a_step_of_single_tokens_names_its_families(monkeypatch, build):
    """With and without graphs: who holds what in common, in groups without a window."""
    from vitna_anchor_b200.cache import KVSpec
    b = _Builder(monkeypatch, [KVSpec(2, 64), KVSpec(2, 64, window=5)])
    c = b.cache
    for rid, n in [("a", 11), ("x", 3), ("p", 8)]:
        c.open(rid)
        _advance(c, rid, n)
    for source, rid in [("a", "b"), ("p", "q"), ("a", "c")]:
        c.tables.fork(source, rid)
    _advance(c, "b", 6)
    order = ["c", "p", "x", "a", "q", "b"]
    before = ops.set_attention_shared(1)
    try:
        c.reserve_step([(rid, 1) for rid in order])
        if build == "build":
            ctx, _ = b.build([(rid, [1], [0]) for rid in order])
            assert b.build([(rid, [1], [0]) for rid in order], for_graph=True)[0].groups[0].members is None
        else:
            ctx, _ = b.build_decode(order, [1] * 6, 6, families=b.families(order))
    finally:
        ops.set_attention_shared(before)
    meta, window = ctx.groups
    assert window.members is None
    assert meta.members.tolist() == [0, 3, 5, 1, 4, 2] and meta.starts.tolist() == [0, 3, 5, 6, 6, 6, 6]
    assert meta.shared.tolist() == [8, 8, 0, 0, 0, 0]           # two whole pages of four of a's eleven positions, both of p's
    for f, shared in zip(([0, 3, 5], [1, 4]), (8, 8)):
        tables = meta.block_tables[f][:, :shared // 4]
        assert bool((tables == tables[0]).all())
    c.rollback_step([(rid, 1) for rid in order])
    c.check()


def _named(monkeypatch, n, dtype=torch.bfloat16, heads=(32, 32, 64), requests=2, model_len=32768):
    """Whether a step of requests that hold `n` positions of 32 heads of 64 in common names its families."""
    from vitna_anchor_b200.cache import KVSpec
    b = _Builder(monkeypatch, [KVSpec(32, 64)], page_size=512, requests=requests, model_len=model_len, dtype=dtype, common_heads=heads and {0: heads})
    b.cache.open(0)
    _advance(b.cache, 0, n)
    for i in range(1, requests):
        b.cache.tables.fork(0, i)
    return b.families(list(range(requests))) is not None


def test_families_are_named_only_where_an_attention_reads_them(monkeypatch):
    """A model none of whose attentions can, a type whose routing has another kernel, more tokens than the kernel takes: no second graph, and no words that nobody reads."""
    assert _named(monkeypatch, 8192) and not _named(monkeypatch, 8192 - 512)                   # 64 MB from 8,192 positions on in bfloat16
    assert not _named(monkeypatch, 32768, heads=None)
    assert not _named(monkeypatch, 32768, dtype=torch.float32)
    before = ops.set_float32_exact(False)
    try:
        assert _named(monkeypatch, 4096, dtype=torch.float32) and not _named(monkeypatch, 4096 - 512, dtype=torch.float32)      # and from 4,096 in float32
    finally:
        ops.set_float32_exact(before)
    assert _named(monkeypatch, 512, model_len=65536) and not _named(monkeypatch, 512, heads=None, model_len=65536)              # 4 MB of what the general attention would read again
    assert _named(monkeypatch, 8192, requests=256) and not _named(monkeypatch, 8192, requests=257)
    ops.set_attention_shared(1)
    try:
        assert _named(monkeypatch, 512, heads=None)                                             # every step that shares, whatever reads it
    finally:
        ops.set_attention_shared(2)


def test_which_attentions_can_read_common_pages_once():
    from vitna_anchor_b200.parts.attention import PagedAttention
    from vitna_anchor_b200.parts.base import Mixer
    w, wo = torch.zeros(4 * 16 + 2 * 2 * 16, 8), torch.zeros(8, 4 * 16)
    assert PagedAttention(8, 4, 2, 16, w, wo, None).common_heads() == (4, 2, 16)
    assert PagedAttention(8, 4, 2, 16, w, wo, None, window=9).common_heads() is None
    assert PagedAttention(8, 4, 2, 16, w, wo, None, qk_norm_eps=1e-6).common_heads() is None
    assert Mixer().common_heads() is None


# (positions that would be read again, key-value heads, their size, type, context): both sides of every line, from the measured ones
@pytest.mark.parametrize("sizes,once", [
    ((7 * 2000, 32, 64, torch.bfloat16, 4096), True), ((3 * 2000, 32, 64, torch.bfloat16, 4096), False), ((15 * 4000, 5, 64, torch.bfloat16, 8192), True), ((31 * 500, 3, 64, torch.bfloat16, 8192), False),
    ((15 * 2000, 8, 128, torch.bfloat16, 4096), True), ((3 * 2000, 8, 128, torch.bfloat16, 16384), False),
    ((7 * 2000, 32, 96, torch.bfloat16, 4608), False), ((63 * 8000, 4, 96, torch.bfloat16, 8192), False), ((63 * 8000, 4, 32, torch.bfloat16, 8192), False), ((63 * 8000, 4, 16, torch.bfloat16, 8192), False),
    ((3 * 4000, 32, 256, torch.bfloat16, 4096), False), ((15 * 4000, 4, 80, torch.bfloat16, 4096), True), ((63 * 4000, 4, 24, torch.bfloat16, 4096), True), ((3 * 4000, 4, 80, torch.bfloat16, 4096), False),
    ((31 * 2000, 3, 64, torch.float32, 4096), True), ((7 * 2000, 3, 64, torch.float32, 4096), False), ((3 * 2000, 32, 64, torch.float32, 4096), True), ((15 * 2000, 4, 128, torch.float32, 4096), True),
    ((3 * 2000, 5, 64, torch.bfloat16, 65536), True), ((3 * 8000, 32, 32, torch.bfloat16, 65536), True), ((500, 32, 256, torch.bfloat16, 65536), True), ((96, 32, 256, torch.bfloat16, 65536), False),
    ((6000, 4, 256, torch.float32, 4096), True), ((100, 4, 256, torch.float32, 4096), False), ((48, 2, 64, torch.bfloat16, 65536), False), ((3 * 2000, 5, 64, torch.bfloat16, 32768), False)])
def test_where_reading_common_pages_once_was_measured_to_be_faster(sizes, once):
    saved, nkv, hd, dtype, context = sizes
    assert ops.attention_shared_pays(saved, nkv, hd, dtype, True, context) == once
    assert not ops.attention_shared_pays(saved, nkv, hd, dtype, False, context)


def test_a_model_says_which_of_its_cache_layers_are_read_so():
    """By cache layer; a mixer that knows nothing of it (a class of its own) reads every request by itself."""
    from vitna_anchor_b200.models.decoder import DecoderModel, LayerRun
    can, cannot, own = SimpleNamespace(common_heads=lambda: (4, 2, 16)), SimpleNamespace(common_heads=lambda: None), SimpleNamespace()
    m = DecoderModel.__new__(DecoderModel)
    m.blocks = [SimpleNamespace(mixer=x) for x in (can, cannot, own)]
    m.schedule = [LayerRun(0, 0), LayerRun(1, 1), LayerRun(2, 2), LayerRun(0, 3), LayerRun(1, -1)]
    assert m.common_heads == {0: (4, 2, 16), 3: (4, 2, 16)}
