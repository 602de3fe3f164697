"""The search's rules, on the host: a model that is a table, and requests that are its histories; no GPU is needed."""
from collections import Counter

import numpy as np
import pytest
import torch

from vitna_anchor_b200.engine import beam
from vitna_anchor_b200.engine.beam import beam_search


class Runner:
    """Requests are their tokens; logits are drawn from the history."""
    max_batch_tokens = 7

    def __init__(self, vocab, scale=2.0, favour=(), spoil=None):
        self.vocab, self.scale, self.favour, self.spoil = vocab, scale, list(favour), spoil
        self.requests, self.cache, self.steps, self.widths = {}, self, 0, Counter()

    def logits_of(self, ids):
        x = np.random.default_rng([len(ids), *ids]).standard_normal(self.vocab) * self.scale
        x[self.favour] += 3.0
        if self.spoil is not None and len(ids) >= self.spoil[0]:
            x[:self.spoil[1]] = self.spoil[2]
        return x.astype(np.float32)

    def is_open(self, rid):
        return rid in self.requests

    def open(self, rid):
        assert rid not in self.requests
        self.requests[rid] = []

    def close(self, rid):
        del self.requests[rid]

    def fork_many(self, pairs):
        for r, s in pairs:
            self.open(r)
            self.requests[r] = list(self.requests[s])

    def adopt(self, pairs):
        for r, s in pairs:
            assert r in self.requests
            self.requests[r] = list(self.requests[s])

    def check(self, sync=True):
        pass

    def step(self, entries):
        for e in entries:
            self.requests[e.request_id] += list(e.tokens)
        rows = [self.logits_of(self.requests[e.request_id]) for e in entries if e.want]
        self.widths[len(rows)] += 1
        return torch.from_numpy(np.stack(rows)) if rows else None


class Selector:
    """The choice by its definition."""

    def __init__(self, vocab, beams):
        self.vocab, self.keep = vocab, 2 * beams

    def choose(self, logits, log_probs):
        x = logits.numpy().astype(np.float64)
        with np.errstate(invalid="ignore"):
            lse = np.logaddexp.reduce(x, axis=1, keepdims=True)
            c = np.where(np.isfinite(lse), np.asarray(log_probs)[:, None] + x - lse, -np.inf)
        c = c.reshape(-1)
        at = np.argsort(-c, kind="stable")[:min(self.keep, c.size)]
        return [(float(np.float32(c[i])), int(i) // self.vocab, int(i) % self.vocab) for i in at]


def plain_search(r, prompt, beams, max_new, penalty, stop):
    """Every sequence from its start, every continuation in order until `beams` of them go on."""
    live, finished = [([], 0.0)], []
    for length in range(1, max_new + 1):
        x = np.stack([r.logits_of(list(prompt) + ids) for ids, _ in live]).astype(np.float64)
        c = np.asarray([lp for _, lp in live])[:, None] + x - np.logaddexp.reduce(x, axis=1, keepdims=True)
        chosen = []
        for rank, at in enumerate(np.argsort(-c.reshape(-1), kind="stable")):
            row, token = divmod(int(at), r.vocab)
            if len(chosen) == beams:
                break
            lp = float(np.float32(c[row, token]))
            if token not in stop:
                chosen.append((live[row][0] + [token], lp))
            elif rank < beams:
                finished.append((live[row][0] + [token], lp / length ** penalty, "stop"))
        finished = sorted(finished, key=lambda f: -f[1])[:beams]
        live = chosen
        if length == max_new:
            finished += [(ids, lp / length ** penalty, "length") for ids, lp in live]
            break
        reach = [max(lp / (length + 1) ** penalty, lp / max_new ** penalty) for _, lp in live]
        if not live or (len(finished) == beams and max(reach) <= finished[-1][1]):
            break
    return sorted(finished, key=lambda f: -f[1])[:beams]


def search(r, prompt, beams, max_new, penalty=1.0, stop=()):
    got = beam_search(r, Selector(r.vocab, beams), prompt, beams=beams, max_new=max_new, length_penalty=penalty, stop_ids=stop, name="s")
    assert not r.requests
    return got


@pytest.mark.parametrize("beams", [1, 2, 5])
@pytest.mark.parametrize("stops", [0, 1, 2, 3, 8, 30])
@pytest.mark.parametrize("vocab", [40, 333])
def test_as_many_beams_go_on_as_there_are_whatever_ends_the_text(vocab, stops, beams):
    """The tokens that end the text are the likely ones: more of them than beams stand before those that go on."""
    r = Runner(vocab, favour=range(stops))
    for penalty in (1.0, 0.0, -1.0):
        got = search(r, [3, 1, 4], beams, 6, penalty, range(stops))
        want = plain_search(r, [3, 1, 4], beams, 6, penalty, set(range(stops)))
        assert [(g.ids, g.finish_reason) for g in got] == [(ids, why) for ids, _, why in want]
        assert all(abs(g.score - score) <= 1e-12 * max(1.0, abs(score)) for g, (_, score, _) in zip(got, want))


def test_a_search_does_not_narrow():
    """Of the best four two or more end the text: two beams all the same, at every step."""
    r = Runner(60, favour=(10, 20, 30))
    got = search(r, [1], 2, 5, 3.0, (10, 20, 30))          # a score that grows with the length, so that nothing ends the search early
    assert r.widths[2] == 4 and len(got) == 2               # (the prompt's step has one row; the last step's choice is the end)


@pytest.mark.parametrize("vocab,beams", [(2, 4), (3, 4), (5, 4), (1, 1), (1, 3)])
def test_vocabularies_of_few_tokens(vocab, beams):
    r = Runner(vocab)
    for stop in ((), (0,)):
        got, want = search(r, [0], beams, 4, 1.0, stop), plain_search(r, [0], beams, 4, 1.0, set(stop))
        assert [g.ids for g in got] == [ids for ids, _, _ in want]


def test_all_in_order():
    """Ties to the lowest (row, token); rows without a softmax, or whose sum is not finite, at the end; -inf in place."""
    inf = float("inf")
    x = torch.tensor([[0.0, 1.0, 1.0, -inf], [float("nan"), 9.0, 9.0, 9.0], [1.0, 1.0, 0.0, 0.0], [inf, 0.0, 0.0, 0.0], [-inf] * 4, [5.0, 5.0, 5.0, 5.0]])
    got = beam.all_in_order(x, [0.0, 0.0, 0.0, 0.0, 0.0, -inf], 24)
    assert [(r, t) for _, r, t in got[:8]] == [(0, 1), (0, 2), (2, 0), (2, 1), (0, 0), (2, 2), (2, 3), (0, 3)] and all(v == -inf for v, _, _ in got[7:])
    assert len(got) == 24 and beam.all_in_order(x, [0.0, 0.0, 0.0, 0.0, 0.0, -inf], 3) == got[:3]
    e = np.exp(1.0)
    assert abs(got[0][0] - np.log(e / (1 + 2 * e))) <= 2.0 ** -24 and abs(got[2][0] - np.log(e / (2 + 2 * e))) <= 2.0 ** -23


@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("behind", [3, 5])
def test_logits_that_are_no_numbers_end_the_search_with_an_error(behind, what):
    """From the prompt's step on, or from a later one: no empty list, and nothing is left open."""
    from vitna_anchor_b200.engine.runner import StepFailed
    r = Runner(50, spoil=(behind, 50, what))
    with pytest.raises(StepFailed, match="no numbers"):
        search(r, [3, 1, 4], 3, 6)
    assert not r.requests
    r = Runner(50, spoil=(behind, 49, float("-inf")))         # one token is left: as many beams as there are rows
    assert [g.ids[-1] for g in search(r, [3, 1, 4], 3, 6)] == [49] * (1 if behind == 3 else 3)


def test_beams_whose_logits_are_no_numbers_die():
    r = Runner(50)
    of = r.logits_of
    r.logits_of = lambda ids: np.full(50, np.nan, dtype=np.float32) if ids[3:4] == [top] else of(ids)
    top = int(np.argmax(of([3, 1, 4])))
    got = search(r, [3, 1, 4], 4, 5)
    assert len(got) == 4 and all(g.ids[0] != top for g in got)


def test_penalties_whose_powers_no_float_holds():
    """Lengths to a power beyond a float's range were an OverflowError, or a division by zero, in the middle of a search."""
    for penalty in (400.0, -400.0, 1e300, -1e300, float("inf"), float("nan")):
        assert not beam.penalty_fits(penalty, 10)
    for penalty, max_new in [(1.0, 131072), (-1.0, 131072), (50.0, 131072), (-50.0, 131072), (1e6, 1), (0.0, 1 << 30), (600.0, 2)]:
        assert beam.penalty_fits(penalty, max_new)
        for length in (1, max_new):
            for log_prob in (-1e9, -1e-7, 0.0):
                assert np.isfinite(beam.normalised(log_prob, length, penalty)) and np.isfinite(beam.attainable(log_prob, length, max_new, penalty))


def test_the_engine_refuses_such_a_penalty():
    from types import SimpleNamespace
    from vitna_anchor_b200.engine.engine import Engine, RequestRefused
    eng = Engine.__new__(Engine)
    eng.model, eng.ctx = SimpleNamespace(vocab_size=50), 64
    eng.runner = SimpleNamespace(cache=SimpleNamespace(max_requests=4), max_batch_tokens=64)
    for penalty in (400.0, -400.0, float("nan"), float("-inf")):
        with pytest.raises(RequestRefused, match="length_penalty"):
            eng.beam_search([1], beams=2, max_new=20, length_penalty=penalty)


def test_the_engine_refuses_more_beams_than_a_step_takes_tokens():
    """A step of more single tokens than the step limit was refused in the middle of the search, when it widened."""
    from types import SimpleNamespace
    from vitna_anchor_b200.engine.engine import Engine, RequestRefused
    eng = Engine.__new__(Engine)
    eng.model, eng.ctx = SimpleNamespace(vocab_size=50), 64
    eng.runner = SimpleNamespace(cache=SimpleNamespace(max_requests=16), max_batch_tokens=4)
    for beams in (0, 5, 16, 17):
        with pytest.raises(RequestRefused, match="between 1 and 4"):
            eng.beam_search([1], beams=beams, max_new=20)
