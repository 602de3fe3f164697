"""Decode steps of requests that hold pages in common, through the step function: that the attention which reads those once is what runs, at every context, and what it gives."""
import numpy as np
import pytest
import torch

from tiny_configs import TINIES, write_tiny

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dirs(tmp_path_factory):
    root = tmp_path_factory.mktemp("steps")
    made = {}
    for nh, kv, hd in [(6, 2, 64), (6, 1, 128), (4, 2, 32)]:
        cfg = dict(TINIES["tinyA"]["config"], hidden_size=256, num_attention_heads=nh, num_key_value_heads=kv, head_dim=hd, vocab_size=500, max_position_embeddings=131072)
        made[hd] = write_tiny(str(root / f"heads{hd}"), dict(TINIES["tinyA"], config=cfg), std=0.1)
    return made


@pytest.fixture
def calls(monkeypatch):
    """How many calls each attention of single tokens got."""
    from vitna_anchor_b200 import ops
    made = {}
    for name in ["attention_shared", "attention_decode", "attention_rows"]:
        def count(*a, _name=name, _of=getattr(ops, name), **k):
            made[_name] = made.get(_name, 0) + 1
            return _of(*a, **k)
        monkeypatch.setattr(ops, name, count)
    return made


def _play(model, context, members, prompt, mode, steps=6, graphs=True):
    """Requests forked from one after its prompt, some steps of single tokens beside a stranger; every step's logits."""
    from vitna_anchor_b200 import ops
    from vitna_anchor_b200.engine.runner import ModelRunner, StepEntry
    before = ops.set_attention_shared(mode)
    try:
        r = ModelRunner(model, page_size=16, max_requests=members + 1, max_batch_tokens=512, max_model_len=context, num_pages=100 + len(prompt) // 16 + members * 3, cuda_graphs=graphs)
        r.open("s")
        r.step([StepEntry("s", prompt[:30], [])])
        r.open(0)
        for at in range(0, len(prompt), 512):
            r.step([StepEntry(0, prompt[at:at + 512], [])])
        for i in range(1, members):
            r.fork(0, i)
        rng = np.random.default_rng(9)
        order = ["s", *range(members)]
        rng.shuffle(order)
        order = [o if o == "s" else int(o) for o in order]
        out = []
        for _ in range(steps):
            out.append(r.step([StepEntry(rid, [int(rng.integers(0, model.vocab_size))], [0]) for rid in order]).clone())
        r.check()
        r.cache.check()
        return torch.stack(out)
    finally:
        ops.set_attention_shared(before)


# tables so wide that the members are not walked one by one (heads of 64: 96 MB, of 128: 240 MB of them); rows of a key-value head's product: 48, 93; 102 (tcgen05 from 65 on)
@pytest.mark.parametrize("hd,members,context", [(64, 16, 32768), (64, 31, 32768), (64, 31, 65536), (128, 17, 32768), (128, 17, 65536), (128, 9, 131072), (32, 5, 65536)])
def test_common_pages_are_read_once_at_every_context(hd, members, context, dirs, calls):
    """bfloat16, against the same steps with every request read by itself: 3e-2 of the logits' scale, as between two ways of cutting one request."""
    from vitna_anchor_b200.engine.loading import load_model
    model = load_model(dirs[hd], "bfloat16", "cuda")
    prompt = [int(t) for t in np.random.default_rng(5).integers(0, model.vocab_size, 1203)]
    a = _play(model, context, members, prompt, 1)
    assert calls["attention_shared"] > 0 and "attention_decode" not in calls
    shared, _ = calls.pop("attention_shared"), calls.pop("attention_rows", 0)
    b = _play(model, context, members, prompt, 0)
    assert "attention_shared" not in calls and calls["attention_decode" if context <= 32768 else "attention_rows"] >= shared
    assert float((a - b).abs().max()) <= 3e-2 * float(b.abs().max())


@pytest.mark.parametrize("hd,context", [(64, 32768), (128, 65536), (32, 256)])
def test_common_pages_are_read_once_without_graphs(hd, context, dirs, calls):
    """Steps that are issued launch by launch, against every request read by itself (the tolerance of the test above)."""
    from vitna_anchor_b200.engine.loading import load_model
    model = load_model(dirs[hd], "bfloat16", "cuda")
    members = 5 if hd == 32 else 17
    prompt = [int(t) for t in np.random.default_rng(6).integers(0, model.vocab_size, 150 if hd == 32 else 1203)]
    a = _play(model, context, members, prompt, 1, graphs=False)
    assert calls["attention_shared"] > 0 and "attention_decode" not in calls
    calls.pop("attention_shared")
    b = _play(model, context, members, prompt, 0, graphs=False)
    assert "attention_shared" not in calls
    assert float((a - b).abs().max()) <= 3e-2 * float(b.abs().max())


def test_logits_that_are_no_numbers_end_a_search_with_an_error(dirs):
    """A final norm's weight that is no number: Engine.beam_search raises and frees everything."""
    from vitna_anchor_b200.engine.engine import Engine
    from vitna_anchor_b200.engine.runner import StepFailed
    eng = Engine(dirs[64], dtype="float32", parallel=4, ctx=128)
    assert len(eng.beam_search([1, 2, 3], beams=3, max_new=4)) == 3
    eng.model.final_norm.tensors()[0].fill_(float("nan"))
    free = eng.runner.cache.free_pages()
    with pytest.raises(StepFailed, match="no numbers"):
        eng.beam_search([1, 2, 3], beams=3, max_new=4)
    assert eng.runner.cache.free_pages() == free and not eng.runner.cache.tables.requests


@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64)])
def test_lists_written_by_the_kernel_just_before(dtype, hd, wide):
    """Positions, or the members, that a kernel of the library writes right before the call: what it wrote is what is read, launched one by one and replayed.
    The kernel is a norm of one long row of ones, which leaves its weights as they are (a mean square of 1, no epsilon): the numbers are their bits.  It lets the kernel
    after it begin at once and takes some hundred microseconds to its end, where the numbers are."""
    from test_beam_ops_gpu import Batch
    from vitna_anchor_b200 import ops
    b = Batch([(500, [20, 3, 41, 9]), (64, [7, 30])], 8, 2, hd, 16, dtype, seed=3).device(wide)
    want, tol = b.want()
    d, n, long = b.d, len(b.pos), 1 << 20
    scratch = torch.zeros(ops.attention_shared_scratch_bytes(n, 8, 2, hd), dtype=torch.uint8, device="cuda")
    ones, weights, row = torch.ones(1, long, device="cuda"), torch.zeros(long, device="cuda"), torch.zeros(1, long, device="cuda")
    for name in ("pos", "members"):
        right, kept = d[name].clone(), d[name]
        weights.view(torch.int32)[-n:] = right
        d[name] = row.view(torch.int32)[0, -n:]

        def call():
            d[name].zero_()
            d["out"].fill_(7.0)
            ops.rmsnorm_rows(ones, weights, 0.0, row)
            return b.run(ops, scratch)
        outs = [call().clone() for _ in range(10)]
        torch.cuda.synchronize()                                  # (one scratch: one stream at a time)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            call()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                call()
            for _ in range(10):
                graph.replay()
                outs.append(d["out"].clone())
        torch.cuda.synchronize()
        assert torch.equal(d[name], right)
        for out in outs:
            assert float(((out.double().cpu() - want).abs() - tol).max()) <= 0
        d[name] = kept


def test_launches_are_counted_as_they_are(dirs):
    """One for members walked by themselves, two for the walk and its join, none where nobody asks for anything; a move a 128; and so for a step that is replayed."""
    from test_beam_ops_gpu import Batch
    from vitna_anchor_b200 import ops

    def count(fn):
        before = ops.launch_count()
        fn()
        return ops.launch_count() - before

    for dtype in (torch.bfloat16, torch.float32):
        for wide, kernels in ((True, 2), (False, 1)):
            b = Batch([(500, [20, 3])], 8, 2, 64, 16, dtype, seed=1).device(wide)
            assert count(lambda: b.run(ops)) == kernels
            b.d.update(members=b.d["members"][:0], starts=b.d["starts"][:1], shared=b.d["shared"][:0])
            assert count(lambda: b.run(ops)) == 0
    arena = torch.zeros(2, 400, 16, device="cuda")
    for moves, kernels in [(0, 0), (1, 1), (128, 1), (129, 2), (200, 2)]:
        assert count(lambda: ops.copy_rows(arena, list(range(moves)), list(range(200, 200 + moves)))) == kernels
    assert count(lambda: ops.copy_rows(torch.empty(2, 3, 0, device="cuda"), [0], [2])) == 0
    none = lambda t: torch.empty((0, 3), dtype=t, device="cuda")      # noqa: E731
    assert count(lambda: ops.beam_select(torch.empty(0, 50, device="cuda"), torch.empty(0, device="cuda"), 2, 3, (none(torch.float32), none(torch.int32), none(torch.int32)),
                                         torch.zeros(4096, dtype=torch.uint8, device="cuda"))) == 0
    # whole steps: with the walk and its join a layer has one launch more than with attention_decode's one
    from vitna_anchor_b200.engine.loading import load_model
    from vitna_anchor_b200.engine.runner import ModelRunner, StepEntry
    model = load_model(dirs[64], "bfloat16", "cuda")
    layers = len(model.schedule)
    r = ModelRunner(model, page_size=16, max_requests=16, max_batch_tokens=256, max_model_len=32768, num_pages=100)
    r.open(0)
    r.step([StepEntry(0, [int(t) for t in np.random.default_rng(1).integers(0, model.vocab_size, 200)], [])])
    r.fork_many([(i, 0) for i in range(1, 16)])
    per_step = {}
    for mode in (0, 1):
        before = ops.set_attention_shared(mode)
        try:
            counts = [count(lambda: r.step([StepEntry(i, [3], [0]) for i in range(16)])) for _ in range(3)]
        finally:
            ops.set_attention_shared(before)
        assert len(set(counts)) == 1                                  # eager and captured, replayed, replayed
        per_step[mode] = counts[0]
    assert per_step[1] - per_step[0] == layers


@pytest.mark.parametrize("vocab", [512, 49152, 262144])
@pytest.mark.parametrize("kind", ["flat", "normal", "wide", "likely", "rising", "high"])
def test_a_rows_log_sum(kind, vocab):
    """What the order across beams hangs on: the best token's continuation at a sum that makes it nearly 0, where float32 holds it to 2^-40, is off by the row's log sum alone.  A thread adds
    up to 128 terms of relative error 2^-22 + 2^-24 of their arguments (weighted by the terms at most 13, the logarithm of their number), 127 steps of 2^-24, and 8 + 2 x 26 exponentials of 2^-22 of
    new maxima and joins: 2^-15 together."""
    from vitna_anchor_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(64, vocab, generator=g, device="cuda") * {"flat": 1e-3, "wide": 5.0}.get(kind, 2.0)
    if kind == "likely":
        at = torch.randint(0, vocab, (64, 200), generator=g, device="cuda")
        x.scatter_add_(1, at, torch.rand(at.shape, generator=g, device="cuda") * 9)
    elif kind == "rising":
        x = x.sort(dim=1).values
    elif kind == "high":
        x += 200
    top, lse = x.max(1).values.double(), torch.logsumexp(x.double(), 1)
    scores = (lse - top).float()
    out = tuple(torch.empty((64, 1), dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32))
    ops.beam_select(x, scores, 1, 1, out, torch.zeros(ops.beam_select_scratch_bytes(64, vocab, 1), dtype=torch.uint8, device="cuda"))
    assert torch.equal(out[2][:, 0].long(), x.argmax(1))
    assert float((out[0][:, 0].double() - (scores.double() + top - lse)).abs().max()) <= 2.0 ** -15


@pytest.mark.parametrize("scale", [0.0, -0.5, 1e-3, 1.0])
@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64), (torch.bfloat16, 40)])
def test_other_scales(dtype, hd, wide, scale):
    """None (every key alike), one that turns the order round, which the tensor-core kernels do not take, a small and a large one.  The tolerance is that of test_beam_ops_gpu with
    the scores' size at this scale: hd products of 32 bits a score, p as two bfloat16 parts and 2^x by the special-function unit, sums in 32 bits, the output's rounding."""
    from test_beam_ops_gpu import Batch
    from vitna_anchor_b200 import ops
    nh, nkv = 8, 2
    b = Batch([(300, [20, 3, 41, 9]), (64, [7, 30])], nh, nkv, hd, 16, dtype, seed=5).device(wide)
    d, n = b.d, len(b.pos)
    scratch = torch.zeros(ops.attention_shared_scratch_bytes(n, nh, nkv, hd), dtype=torch.uint8, device="cuda")
    got = ops.attention_shared(d["q"], d["cache"], d["tables"], d["seg"], d["pos"], d["members"], d["starts"], d["shared"], d["out"], scratch, nh, nkv, hd, scale).double().cpu()
    for t in b.members:
        at = torch.arange(b.pos[t] + 1)
        kv = b.cache[torch.tensor(b.tables[t])[at // 16], :, :, at % 16].double()
        k, v = (kv[:, i].repeat_interleave(nh // nkv, dim=1) for i in (0, 1))
        q = b.q[t].double().view(nh, hd)
        o = torch.einsum("hp,phd->hd", torch.softmax(torch.einsum("phd,hd->hp", k, q) * scale, 1), v)
        size = (torch.einsum("phd,hd->hp", k.abs(), q.abs()) * abs(scale)).amax(1)
        slack = (2 * hd * 2.0 ** -23 * size + 2.0 ** -16 + 64 * 2.0 ** -23) * v.abs().amax((0, 2))
        off = (got[t].view(nh, hd) - o).abs() - torch.finfo(dtype).eps / 2 * o.abs() - slack[:, None]
        assert float(off.max()) <= 0


@pytest.mark.parametrize("beams,stops", [(2, 6), (4, 40), (1, 3), (3, 200), (5, 1)])
def test_a_search_with_many_ends_of_the_text(dirs, beams, stops):
    """The tokens that the first steps like best end the text: the results of the plain search, which walks every continuation until enough go on (float32, whose logits are the
    same bits however the work is cut)."""
    from types import SimpleNamespace
    from test_beam_search import plain_search
    from vitna_anchor_b200.engine import beam
    from vitna_anchor_b200.engine.engine import Engine
    eng = Engine(dirs[64], dtype="float32", parallel=6, ctx=128, kv_block=4)
    prompt = [int(t) for t in np.random.default_rng(11).integers(0, 500, 17)]
    plain = SimpleNamespace(vocab=500, logits_of=lambda ids: eng.logits(ids)[-1].cpu().numpy())
    stop = {int(t) for t in np.argsort(-plain.logits_of(prompt))[:stops]}
    wide, all_in_order = [], beam.all_in_order
    beam.all_in_order = lambda *a: wide.append(1) or all_in_order(*a)
    try:
        for penalty in (1.0, 0.0):
            got = eng.beam_search(prompt, beams=beams, max_new=6, length_penalty=penalty, stop_ids=stop)
            want = plain_search(plain, prompt, beams, 6, penalty, stop)
            assert [(r.ids, r.finish_reason) for r in got] == [(ids, why) for ids, _, why in want]
    finally:
        beam.all_in_order = all_in_order
    assert bool(wide) == (stops > beams)
    assert not eng.runner.cache.tables.requests
