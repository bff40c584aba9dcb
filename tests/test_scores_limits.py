"""Scores: what is refused, and that it is refused before anything has run (no GPU is needed)."""
from types import SimpleNamespace

import pytest


@pytest.mark.parametrize("top", [21, -1, 1000])
def test_step_logprobs_refuses_alternatives_before_it_looks_at_the_step(top):
    from infer_b200.engine import Engine
    eng = object.__new__(Engine)                     # no cache, no model: whatever the call did with them would be another error
    eng.spec = SimpleNamespace(vocab_size=50)
    with pytest.raises(ValueError, match="alternatives"):
        eng.step_logprobs([("r", [1, 2], [0, 1])], [1, 2], top)


@pytest.mark.parametrize("n", [2.5, 21, -1, float("nan"), float("inf")])
def test_a_scheduler_refuses_alternatives_when_a_request_is_submitted(n):
    """(Later it would be a step that has run: its token would be lost.)"""
    from infer_b200.engine.scheduler import BatchEngine, Request, SampleParams, Scheduler, SchedulerConfig

    class Fake(BatchEngine):
        max_seq_len, max_requests = 64, 4

        def capacity_tokens(self): return 1000
    sch = Scheduler(Fake(), SchedulerConfig())
    with pytest.raises(ValueError, match="alternatives"):
        sch.submit(Request("r", [1, 2], 4, 0, SampleParams(logprobs=n)))
    assert not sch.queue
