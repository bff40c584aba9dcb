"""Scores: what is refused, and that it is refused before anything has run (no GPU is needed)."""
import subprocess
import sys
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


_PLANS = """
import ctypes
from infer_b200.csrc.build import load_module
act, i64 = load_module("act_tc"), ctypes.c_int64
w, s, c = ctypes.c_int(), ctypes.c_int(), ctypes.c_int64()
for M, N, K, sms in ((1 << 29, 1 << 29, 64, 148), ((1 << 30) - 1, (1 << 30) - 1, 8, 148), (100, 100, 64, 1), (100, 100, 64, 0), (1 << 29, 1 << 29, 64, 1)):
    assert act.ib_linear_act_plan(i64(M), i64(N), i64(K), sms, ctypes.byref(w), ctypes.byref(s), ctypes.byref(c)) < 0 and act.ib_last_error()
print("refused")
"""


def test_plans_that_no_width_fits_are_refused():
    """In a process of its own: a division by a width that was never set ends one."""
    proc = subprocess.run([sys.executable, "-c", _PLANS], capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0 and proc.stdout == "refused\n", (proc.returncode, proc.stderr[-300:])


@pytest.mark.parametrize("argv,what", [(["--logprobs", "21"], "0 to 20"), (["--logprobs", "-1"], "0 to 20"), (["cache=off", "--logprobs", "3"], "cache")])
def test_generate_says_what_it_cannot_do(argv, what, capsys):
    from infer_b200.cli import generate
    with pytest.raises(SystemExit) as end:
        generate.main(["--random", "tiny-a", *argv])
    assert end.value.code == 2 and what in capsys.readouterr().err
