"""Forks between steps that may still be running, on the host's tables; no GPU is needed."""
import pytest
import torch

from vitna_anchor_b200 import ops
from vitna_anchor_b200.cache import CacheManager, KVSpec
from vitna_anchor_b200.engine import runner as runner_module
from vitna_anchor_b200.engine.runner import DeviceStepFailed, ModelRunner, _Issued


class _Event:
    def __init__(self):
        self.done = False

    def query(self):
        return self.done


@pytest.fixture
def runner(monkeypatch):
    """A runner of tables alone, whose steps advance lengths; runner.code is what its kernels left in the error word."""
    r = ModelRunner.__new__(ModelRunner)
    r.device, r._issued, r.code, r.waits = torch.device("cuda"), [], 0, 0
    r.cache = CacheManager([KVSpec(1, 8)], page_size=4, num_pages=30, max_requests=5, dtype=torch.float32, device="cpu", allocate=False)

    class Stream:
        def synchronize(self):
            r.waits += 1
            for item in r._issued:
                item.event.done = True

    def take():
        code, r.code = r.code, 0
        if code:
            raise ops.KernelGaveUp(f"code {code}")

    monkeypatch.setattr(runner_module.torch.cuda, "current_stream", lambda device: Stream())
    monkeypatch.setattr(ops, "device_error_code", lambda: r.code)
    monkeypatch.setattr(ops, "check_device_errors", take)

    def advance(rid, n):
        before = [(rid, r.cache.length(rid))]
        r.cache.reserve_step([(rid, n)])
        r.cache.commit_step([(rid, n)])
        r._issued.append(_Issued(before, None, _Event()))

    r.advance = advance
    return r


@pytest.mark.parametrize("move", ["fork", "adopt"])
def test_nothing_goes_on_from_a_step_that_failed(runner, move):
    """Six positions that are known to be there, two of a step whose wait ran out: the request goes back to six, and nobody has the eight."""
    runner.open("a")
    runner.advance("a", 6)
    runner.check()
    if move == "adopt":
        runner.open("b")
        runner.advance("b", 3)
        runner.check()
    runner.advance("a", 2)
    runner.code = 81
    with pytest.raises(DeviceStepFailed) as e:
        runner.fork("a", "b") if move == "fork" else runner.adopt([("b", "a")])
    assert e.value.request_ids == ["a"] and runner.length("a") == 6 and not runner._issued
    assert runner.length("b") == 3 if move == "adopt" else not runner.cache.is_open("b")
    runner.cache.check()
    runner.fork("a", "c")                                     # and it can go on
    assert runner.length("c") == 6
    runner.cache.check()


def test_moves_wait_only_for_steps_that_are_not_known_to_have_worked(runner):
    runner.open("a")
    runner.advance("a", 5)
    runner.fork("a", "b")
    assert runner.waits == 1 and not runner._issued
    runner.fork("a", "c")
    runner.adopt([("b", "a")])
    assert runner.waits == 1
    runner.advance("a", 1)
    runner._issued[0].event.done = True                       # the caller has waited by itself
    runner.adopt([("b", "a"), ("c", "a")])
    assert runner.waits == 1 and runner.length("c") == 6
    runner.cache.check()
