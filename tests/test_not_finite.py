"""A key or value that an 8-bit cache cannot hold ends its own request and no other: the host's side, with a fake engine."""
import importlib
from types import SimpleNamespace

import pytest

from mlx_lm_b200.engine.scheduler import Scheduler
from mlx_lm_b200.ops import ST_NOT_FINITE, ST_PAGE_RANGE, KernelError

from test_scheduler import FakeEngine, expected, fake_sample, run

G = importlib.import_module("mlx_lm_b200.generate")


class Reporting(FakeEngine):
    """At step ``at`` the requests ``bad`` bring a number that is not finite (and the status word has the bits ``more`` besides)."""

    def __init__(self, at, bad, more=0, **kw):
        super().__init__(**kw)
        self.at, self.bad, self.more, self.host_status, self.failed, self.cleared = at, bad, more, 0, set(), 0

    def step(self, entries):
        out = super().step(entries)
        if len(self.steps) == self.at:
            self.host_status = ST_NOT_FINITE | self.more
        return out

    def find_not_finite(self):
        self.failed.update(r for r in self.bad if r in self.cache.requests)
        self.host_status &= ~ST_NOT_FINITE

    def finish(self, rid):
        super().finish(rid)
        self.failed.discard(rid)

    def clear_status(self):
        self.host_status = 0
        self.cleared += 1


@pytest.mark.parametrize("at", [1, 3, 6])
def test_the_others_go_on(at):
    eng = Reporting(at, bad=[1], n_pages=64)
    s = Scheduler(eng, fake_sample, max_requests=3, max_tokens_per_step=64)
    for _ in range(3):
        s.insert(list(range(10)), max_tokens=12)
    out, reasons = run(s)
    assert reasons == {0: "length", 1: "not_finite", 2: "length"}
    assert out[0] == expected(0, 10, 12) and out[2] == expected(2, 10, 12)
    assert out[1] == expected(1, 10, at - 1) + [-1]
    assert eng.cache.pages_in_use() == [0] and not eng.cache.requests and not eng.failed and eng.cleared == 0


def test_one_that_is_still_in_its_prompt():
    eng = Reporting(2, bad=[1], n_pages=64)
    s = Scheduler(eng, fake_sample, max_requests=2, prefill_step_size=8, max_tokens_per_step=16)
    s.insert(list(range(4)), max_tokens=9)
    s.insert(list(range(60)), max_tokens=9)
    out, reasons = run(s)
    assert reasons == {0: "length", 1: "not_finite"} and out == {0: expected(0, 4, 9), 1: [-1]}
    assert eng.cache.pages_in_use() == [0]


def test_a_fault_of_the_whole_step_still_stops_it():
    eng = Reporting(2, bad=[0], more=ST_PAGE_RANGE, n_pages=64)
    s = Scheduler(eng, fake_sample, max_requests=2)
    s.insert(list(range(4)), max_tokens=9)
    s.next()
    with pytest.raises(KernelError, match="page id outside"):
        s.next()
    assert eng.cleared == 1 and eng.failed == {0}


def test_requests_of_another_scheduler_on_the_same_engine():
    """Whoever reads the status word first: each scheduler ends its own."""
    eng = Reporting(3, bad=[("a", 0), ("b", 0)], n_pages=64)
    names = iter("ab")
    eng.new_namespace = lambda: next(names)
    sample = lambda rows, requests: ([5] * len(rows), [0.0] * len(rows))
    a, b = Scheduler(eng, sample), Scheduler(eng, sample)
    a.insert([1, 2, 3], max_tokens=9)
    b.insert([1, 2, 3], max_tokens=9)
    a.next(), b.next()
    assert [r.finish_reason for r in a.next()[1]] == ["not_finite"]
    assert [r.finish_reason for r in b.next()[1]] == ["not_finite"]
    assert not a.has_work() and not b.has_work() and eng.cache.pages_in_use() == [0]


def test_a_single_request_raises(monkeypatch):
    eng = Reporting(3, bad=[0], n_pages=8)

    class StandIn:
        def __init__(self, device, seed=0, return_logprobs=False, engine=None):
            self.last_logprobs = None

        def __call__(self, rows, requests):
            tokens, logprobs = fake_sample(rows, requests)
            self.last_logprobs = [SimpleNamespace(clone=lambda: None) for _ in tokens]
            return tokens, logprobs

    monkeypatch.setattr(G, "DeviceSampler", StandIn)
    monkeypatch.setattr(G, "get_engine", lambda model: eng)
    got = []
    with pytest.raises(KernelError, match="not finite"):
        for t, _ in G.generate_step(list(range(5)), SimpleNamespace(device="cpu"), max_tokens=9):
            got.append(t)
    assert got == expected(0, 5, 2) and eng.cache.pages_in_use() == [0]
