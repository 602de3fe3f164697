"""Beam search over the step function.

A search keeps the `beams` most likely continuations of one prompt.  Its beams are requests of one family: the prompt runs once, the others
are forked from it and hold its pages in common, so that a step's attention reads the prompt once for all of them.  Every step the model
gives the live beams' logits, and the host takes the (beam, token) pairs in order, best first: a token that ends the text finishes a result if
it is among the first `beams`, every other one is a live beam until there are `beams` of them.  The 2 x beams best are chosen on the device.  With
one token that ends the text they are always enough; where several do, and fewer than `beams` of them go on, the host orders all there are.  A beam
that several go on from keeps its request; the others of them take over requests that nothing goes on from.

A result's score is its sum of log probabilities divided by length ** length_penalty (length: its new tokens, the stop token counted).
The search ends when max_new tokens are reached, when no beam lives, or when `beams` results are finished and no live beam can reach the worst of
them any more (log probabilities only add up downwards).  Beams whose logits are no numbers die; where that is all of them the search fails (StepFailed).

The reference has no beam search; its choice of a token (engine/src/sampler.c:31-38) is what one beam does.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Hashable, Iterable, List, Optional, Sequence, Set

import numpy as np
import torch

from .. import ops
from .runner import ModelRunner, StepEntry, StepFailed


@dataclass
class BeamResult:
    ids: List[int]               # new tokens, the stop token included
    score: float                 # sum of log probabilities / len(ids) ** length_penalty
    log_prob: float              # the sum itself
    finish_reason: str           # "stop" or "length"


@dataclass
class _Beam:
    request_id: Hashable
    ids: List[int]
    log_prob: float


class BeamSelector:
    """The choice on the device: buffers for up to `beams` rows, made once."""

    def __init__(self, vocab: int, beams: int, device):
        self.vocab, self.beams = vocab, beams
        self.keep = min(2 * beams, beams * vocab)
        self._scratch = torch.zeros(ops.beam_select_scratch_bytes(beams, vocab, self.keep), dtype=torch.uint8, device=device)
        self._out = torch.empty((3, self.keep), dtype=torch.int32, device=device)
        self._scores = torch.empty(beams, dtype=torch.float32, device=device)
        self._scores_host = torch.empty(beams, dtype=torch.float32).pin_memory()
        self._out_host = torch.empty((3, self.keep), dtype=torch.int32).pin_memory()

    def choose(self, logits: torch.Tensor, log_probs: Sequence[float]) -> List[tuple]:
        """(log probability, row, token) of the best continuations, in descending order; waits for them."""
        n = len(log_probs)
        keep = min(self.keep, n * self.vocab)        # of one row there may be fewer tokens than are kept
        self._scores_host[:n] = torch.tensor(list(log_probs), dtype=torch.float32)
        self._scores[:n].copy_(self._scores_host[:n], non_blocking=True)
        out = (self._out[0:1, :keep].view(torch.float32), self._out[1:2, :keep], self._out[2:3, :keep])
        ops.beam_select(logits, self._scores[:n], n, keep, out, self._scratch)
        self._out_host.copy_(self._out, non_blocking=True)
        torch.cuda.current_stream().synchronize()
        return list(zip(self._out_host[0, :keep].view(torch.float32).tolist(), self._out_host[1, :keep].tolist(), self._out_host[2, :keep].tolist()))


def all_in_order(logits: torch.Tensor, log_probs: Sequence[float], count: int) -> List[tuple]:
    """What BeamSelector.choose gives, for any count of continuations, on the host in 64 bits."""
    x = logits[:len(log_probs)].cpu().numpy().astype(np.float64)
    with np.errstate(invalid="ignore"):
        c = np.asarray(log_probs, dtype=np.float64)[:, None] + x - np.logaddexp.reduce(x, axis=1, keepdims=True)
    c[~np.isfinite(c).any(axis=1) | np.isnan(c).any(axis=1) | (c == np.inf).any(axis=1)] = -np.inf
    c = c.reshape(-1)
    count = min(count, c.size)
    least = np.partition(c, c.size - count)[c.size - count]
    at = np.flatnonzero(c >= least)
    at = at[np.argsort(-c[at], kind="stable")][:count]
    return [(float(np.float32(v)), int(i) // x.shape[1], int(i) % x.shape[1]) for v, i in zip(c[at], at)]


def normalised(log_prob: float, length: int, length_penalty: float) -> float:
    return log_prob / float(length) ** length_penalty


def penalty_fits(length_penalty: float, max_new: int) -> bool:
    """Whether every length's power, and a sum of log probabilities divided by it, is a number that a float holds (a sum is below 2^30: tokens times the largest difference of logits that count)."""
    return math.isfinite(length_penalty) and abs(length_penalty) * math.log(max_new) <= 600.0


def attainable(log_prob: float, length: int, max_new: int, length_penalty: float) -> float:
    """The best score that a live beam of this sum and length can still end with: its sum stays, at the length that divides it most kindly."""
    return max(normalised(log_prob, length, length_penalty), normalised(log_prob, max_new, length_penalty))


def take(best: Sequence[tuple], beams: int, stop: Set[int]) -> tuple:
    """Of continuations (log probability, row, token), best first: the (row, token, log probability) that end among the first `beams`, and the first `beams` that go on."""
    ended, chosen = [], []
    for rank, (log_prob, row, token) in enumerate(best):
        if log_prob == float("-inf") or len(chosen) == beams:
            break
        if token not in stop:
            chosen.append((row, token, log_prob))
        elif rank < beams:
            ended.append((row, token, log_prob))
    return ended, chosen


def plan_moves(parents: Sequence[int], live: Sequence[Hashable]) -> tuple:
    """parents[i]: the place among `live` of the request that new beam i goes on from.  Returns (the new beams' requests, the (request, source)
    pairs to adopt, the requests nobody needs): the first beam that goes on from a request keeps it, the others take over requests that are left;
    None where there is none left and the beam needs a fork."""
    requests: List[Optional[Hashable]] = [None] * len(parents)
    kept: Set[int] = set()
    for i, p in enumerate(parents):
        if p not in kept:
            kept.add(p)
            requests[i] = live[p]
    left = [r for p, r in enumerate(live) if p not in kept]
    pairs = []
    for i, p in enumerate(parents):
        if requests[i] is None and left:
            requests[i] = left.pop(0)
            pairs.append((requests[i], live[p]))
    return requests, pairs, left


def beam_search(runner: ModelRunner, selector: BeamSelector, ids: Sequence[int], *, beams: int, max_new: int, length_penalty: float,
                stop_ids: Iterable[int], name: Hashable) -> List[BeamResult]:
    stop = {t for t in stop_ids if 0 <= t < selector.vocab}
    opened: List[Hashable] = []

    def new_request() -> Hashable:
        rid = (name, len(opened))
        opened.append(rid)
        return rid

    try:
        root = new_request()
        runner.open(root)
        logits = None
        for at in range(0, len(ids), runner.max_batch_tokens):
            piece = list(ids[at:at + runner.max_batch_tokens])
            logits = runner.step([StepEntry(root, piece, [len(piece) - 1] if at + len(piece) == len(ids) else [])])
        live, finished = [_Beam(root, [], 0.0)], []
        for length in range(1, max_new + 1):
            best = selector.choose(logits, [b.log_prob for b in live])
            runner.check(sync=False)                     # the choice has arrived, so every kernel of the step is done
            if best[0][0] == float("-inf"):              # (of a row that has a softmax the largest value is offered, at a finite sum)
                raise StepFailed(f"the logits behind {len(live)} beam(s) of {len(live[0].ids)} new tokens are no numbers that a token can be chosen by (a NaN, an infinity, nothing above -inf)")
            ended, chosen = take(best, beams, stop)
            there = len(live) * selector.vocab
            if len(chosen) < beams and len(best) < there and best[-1][0] != float("-inf"):
                best = all_in_order(logits, [b.log_prob for b in live], beams + len(live) * len(stop))
                ended, chosen = take(best, beams, stop)
            finished += [BeamResult(live[row].ids + [token], normalised(log_prob, length, length_penalty), log_prob, "stop") for row, token, log_prob in ended]
            finished.sort(key=lambda r: -r.score)        # stable: among equals what was finished first
            del finished[beams:]
            if length == max_new:
                finished += [BeamResult(live[row].ids + [token], normalised(lp, length, length_penalty), lp, "length") for row, token, lp in chosen]
                break
            if not chosen or (len(finished) == beams and all(attainable(lp, length + 1, max_new, length_penalty) <= finished[-1].score for _, _, lp in chosen)):
                break
            requests, pairs, left = plan_moves([row for row, _, _ in chosen], [b.request_id for b in live])
            for rid in left:
                runner.close(rid)
            runner.adopt(pairs)
            wider = []
            for i, (row, _, _) in enumerate(chosen):
                if requests[i] is None:                  # more beams than requests: only while the search widens
                    requests[i] = new_request()
                    wider.append((requests[i], live[row].request_id))
            runner.fork_many(wider)
            live = [_Beam(rid, live[row].ids + [token], lp) for rid, (row, token, lp) in zip(requests, chosen)]
            logits = runner.step([StepEntry(b.request_id, [b.ids[-1]], [0]) for b in live])
        finished.sort(key=lambda r: -r.score)
        return finished[:beams]
    finally:
        for rid in opened:
            if runner.cache.is_open(rid):
                runner.close(rid)
