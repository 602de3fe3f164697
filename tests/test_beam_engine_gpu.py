"""Beam search through the engine: against a search that runs every sequence again from its start, on every architecture (pages, windows, states,
loops); forked requests' logits; failures, refusals, the command line."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from tiny_configs import TINIES, write_tiny

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OTHERS = ["lupanex/looped", "lupanex/streams", "siparax/shared", "manatar/all", "tinevik/all", "lirutar/all", "zolapel/all"]


@pytest.fixture(scope="module")
def dirs(tmp_path_factory):
    root = tmp_path_factory.mktemp("beam")
    made = {name: write_tiny(str(root / name), tiny, std=0.15) for name, tiny in TINIES.items()}
    for kv, hd in [(2, 64), (1, 128)]:
        cfg = dict(TINIES["tinyA"]["config"], hidden_size=256, num_attention_heads=6, num_key_value_heads=kv, head_dim=hd, vocab_size=500, max_position_embeddings=131072)
        made[f"heads{hd}"] = write_tiny(str(root / f"heads{hd}"), dict(TINIES["tinyA"], config=cfg), std=0.1)
    import importlib
    for name in OTHERS:
        arch, which = name.split("/")
        made[name] = str(root / name.replace("/", "_"))
        importlib.import_module(f"{arch}_models").make_model(made[name], which)
    return made


@pytest.fixture(params=[1, 2])
def shared_mode(request):
    """Every step that shares goes through the attention that reads common pages once, or those of the rule (on these small models none)."""
    from vitna_anchor_b200 import ops
    before = ops.set_attention_shared(request.param)
    yield request.param
    ops.set_attention_shared(before)


def _engine(path, dtype, **kw):
    from vitna_anchor_b200.engine.engine import Engine
    return Engine(path, dtype=dtype, **{"parallel": 6, "ctx": 256, "kv_block": 4, **kw})


def _log_probs(eng, ids):
    """log softmax of every position's logits, in 64 bits, of the sequence run from its start."""
    x = eng.logits(ids, piece=min(256, eng.runner.max_batch_tokens)).double().cpu().numpy()
    return x - np.logaddexp.reduce(x, axis=1, keepdims=True)


def plain_search(eng, prompt, beams, max_new, penalty=1.0, stop=()):
    """The search's definition, every sequence run again from its start at every step."""
    live, finished = [([], 0.0)], []
    for length in range(1, max_new + 1):
        c = np.stack([lp + _log_probs(eng, list(prompt) + ids)[-1] for ids, lp in live])
        order = np.argsort(-c.reshape(-1), kind="stable")[:min(2 * beams, c.shape[1])]
        chosen = []
        for rank, at in enumerate(order):
            row, token = divmod(int(at), c.shape[1])
            if len(chosen) == beams:
                break
            if token in stop:
                if rank < beams:
                    finished.append((live[row][0] + [token], c[row, token] / length ** penalty))
            else:
                chosen.append((live[row][0] + [token], c[row, token]))
        finished = sorted(finished, key=lambda r: -r[1])[:beams]
        live = chosen
        if length == max_new:
            finished += [(ids, lp / length ** penalty) for ids, lp in live]
            break
        reach = [max(lp / (length + 1) ** penalty, lp / max_new ** penalty) for _, lp in live]
        if not live or (len(finished) == beams and max(reach) <= finished[-1][1]):
            break
    return sorted(finished, key=lambda r: -r[1])[:beams]


@pytest.mark.parametrize("name", ["tinyA", "tinyB", "heads64", "heads128"] + OTHERS)
def test_search_matches_one_that_starts_over(name, dirs):
    """float32, whose logits are the same bits however the work is cut: the same results."""
    eng = _engine(dirs[name], "float32")
    rng = np.random.default_rng(7)
    V = eng.model.vocab_size
    prompt = [int(t) for t in rng.integers(0, V, 21)]
    free = eng.runner.cache.free_pages()
    for beams, max_new, penalty, stop in [(3, 9, 1.0, ()), (5, 7, 0.0, set(range(0, V, 7))), (1, 6, 1.0, ())]:
        got = eng.beam_search(prompt, beams=beams, max_new=max_new, length_penalty=penalty, stop_ids=stop)
        want = plain_search(eng, prompt, beams, max_new, penalty, stop)
        assert [r.ids for r in got] == [ids for ids, _ in want]
        # sums of at most 9 log probabilities, each rounded to 32 bits from sums of exponentials in 32 bits: 9 (2^-24 |sum| + 40 2^-23)
        for r, (ids, score) in zip(got, want):
            assert abs(r.score - score) <= 9 * (2.0 ** -24 * abs(r.log_prob) + 40 * 2.0 ** -23) and r.finish_reason == ("stop" if ids[-1] in stop else "length")
        assert eng.runner.cache.free_pages() == free and not eng.runner.cache.tables.requests
        eng.runner.cache.check()
    assert eng.beam_search(prompt, beams=1, max_new=6)[0].ids == eng.generate(prompt, max_new=6)


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("name", ["tinyB", "heads64", "heads128", "lupanex/looped", "lirutar/all"])
def test_sums_are_those_of_the_sequences(name, graphs, dirs, shared_mode):
    """bfloat16: every result's sum of log probabilities is that of its sequence run from its start, as near as two ways of cutting one request come
    (8e-2 of the logits' scale at a position; the mean over a sequence is held to that)."""
    # heads64 and heads128: tables so wide that the common keys are walked once, not every member by itself (a search of six, heads of 64: 96 MB and more)
    wide = dict(kv_block=16, ctx=65536, num_pages=200) if name.startswith("heads") else {}
    eng = _engine(dirs[name], "bfloat16", cuda_graphs=graphs, **wide)
    rng = np.random.default_rng(3)
    prompt = [int(t) for t in rng.integers(0, eng.model.vocab_size, 150 if name.startswith("heads") else 40)]
    got = eng.beam_search(prompt, beams=6, max_new=40)
    assert len(got) == 6 and len({tuple(r.ids) for r in got}) == 6 and all(len(r.ids) == 40 for r in got)
    assert [r.score for r in got] == sorted((r.score for r in got), reverse=True)
    for r in got:
        logits = eng.logits(prompt + r.ids[:-1])
        scale = max(1.0, float(logits.abs().max()))
        lp = _log_probs(eng, prompt + r.ids[:-1])[len(prompt) - 1:]
        assert abs(lp[np.arange(40), r.ids].sum() - r.log_prob) <= 40 * 8e-2 * scale
    eng.runner.cache.check()
    assert {k[2] for k in eng.runner._decode_graphs} == ({shared_mode == 1} if graphs else set())


@pytest.mark.parametrize("name,tol", [("heads64", 3e-2), ("heads128", 3e-2), ("tinyB", 3e-2)])
def test_forked_requests_give_the_logits_of_separate_ones(name, tol, dirs, shared_mode):
    """Six requests forked from one, decoding beside a stranger through the graph that reads common pages once, against the same tokens in
    requests of their own through the ordinary graph (bfloat16; both see the same keys)."""
    from vitna_anchor_b200.engine.loading import load_model
    from vitna_anchor_b200.engine.runner import ModelRunner, StepEntry
    model = load_model(dirs[name], "bfloat16", "cuda")
    V = model.vocab_size
    rng = np.random.default_rng(5)
    prompt, stranger = ([int(t) for t in rng.integers(0, V, n)] for n in (203, 30))

    def play(fork):
        r = ModelRunner(model, page_size=16, max_requests=8, max_batch_tokens=512, max_model_len=131072, num_pages=200)
        r.open("s")
        r.step([StepEntry("s", stranger, [])])
        for i in range(6):
            if fork and i:
                r.fork(0, i)
            else:
                r.open(i)
                r.step([StepEntry(i, prompt, [])])
        order = [3, 0, "s", 5, 1, 4, 2]
        tokens = np.random.default_rng(9).integers(0, V, (12, 7))
        out = []
        for row in tokens:
            out.append(r.step([StepEntry(rid, [int(t)], [0]) for rid, t in zip(order, row)]).clone())
        r.check()
        assert {k[2] for k in r._decode_graphs} == {fork and shared_mode == 1} and r.graph_replays > 5
        r.cache.check()
        return torch.stack(out)

    a, b = play(True), play(False)
    assert float((a - b).abs().max()) <= tol * float(b.abs().max())


def test_a_failed_step_ends_the_search_and_frees_everything(dirs):
    from vitna_anchor_b200.engine.runner import StepFailed
    eng = _engine(dirs["tinyA"], "float32")
    free = eng.runner.cache.free_pages()
    for at in (0, 12):
        eng.runner.fail_step_once(at)
        with pytest.raises(StepFailed):
            eng.beam_search([1, 2, 3, 4, 5, 6, 7, 8, 9], beams=4, max_new=9)
        assert eng.runner.cache.free_pages() == free and not eng.runner.cache.tables.requests
    assert len(eng.beam_search([1, 2, 3], beams=4, max_new=5)) == 4


def test_pages_run_out(dirs):
    from vitna_anchor_b200.cache import OutOfPages
    eng = _engine(dirs["tinyA"], "float32", num_pages=9)
    with pytest.raises(OutOfPages):
        eng.beam_search(list(range(1, 27)), beams=6, max_new=30)
    assert not eng.runner.cache.tables.requests and eng.runner.cache.free_pages() == [9]


def test_refusals(dirs):
    from vitna_anchor_b200.engine.engine import RequestRefused
    eng = _engine(dirs["tinyA"], "float32", ctx=32)
    for ids, kw in [([], {}), ([256], {}), ([1], dict(beams=0)), ([1], dict(beams=7)), ([1], dict(max_new=0)), (list(range(20)), dict(max_new=13)),
                    ([1], dict(length_penalty=float("nan")))]:
        with pytest.raises(RequestRefused):
            eng.beam_search(ids, **{"beams": 2, "max_new": 4, **kw})
    eng.add_request([1, 2, 3], max_new=3)
    with pytest.raises(RequestRefused):
        eng.beam_search([1], beams=2, max_new=4)
    eng.run()
    assert len(eng.beam_search([1], beams=2, max_new=4)) == 2


def test_a_prompt_that_fills_the_context_and_long_prompts_in_portions(dirs):
    eng = _engine(dirs["tinyB"], "float32", ctx=64, max_batch_tokens=16)
    prompt = [int(t) for t in np.random.default_rng(1).integers(0, 300, 60)]
    got = eng.beam_search(prompt, beams=3, max_new=4)
    assert [r.ids for r in got] == [ids for ids, _ in plain_search(eng, prompt, 3, 4)]


def test_generate_command_with_beams(dirs):
    eng = _engine(dirs["tinyA"], "float32", kv_block=16, parallel=3)
    want = eng.beam_search([5, 17, 3, 9], beams=3, max_new=6, length_penalty=0.5)
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "vitna-anchor"), "generate", "--model", dirs["tinyA"], "--ids", "5,17,3,9", "--max-new", "6", "--beams", "3",
                        "--length-penalty", "0.5", "--dtype", "float32", "--ctx", "256"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    out = json.loads(r.stdout.strip().splitlines()[-1])
    assert out["ids"] == want[0].ids and [b["ids"] for b in out["beams"]] == [w.ids for w in want]
    assert [b["log_prob"] for b in out["beams"]] == [w.log_prob for w in want]
