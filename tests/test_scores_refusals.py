"""What the scoring operators and products with an activation refuse before anything runs (no GPU is needed), and the scheduler's side of scores."""
import pytest
import torch

from infer_b200 import ops
from infer_b200.ops import KernelError


@pytest.mark.parametrize("kw,what", [({"top": 21}, "alternatives"), ({"top": -1}, "alternatives"), ({"scale": 0.0}, "scale"), ({"scale": -1.0}, "scale"),
                                     ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"), ({"softcap": -1.0}, "cap"),
                                     ({"softcap": float("inf")}, "cap"), ({"softcap": float("nan")}, "cap"),
                                     ({"scale": 1e39}, "scale"), ({"scale": 1e-20}, "scale"), ({"softcap": 1e-20}, "cap"), ({"softcap": 1e20}, "cap")])
def test_distributions_that_are_none(kw, what):
    with pytest.raises(KernelError, match=what):
        ops.token_logprobs(torch.zeros(2, 5), None, **{"top": 0, **kw})
    with pytest.raises(KernelError, match=what):
        ops.head_logprobs(torch.zeros(2, 8), torch.zeros(5, 8), None, **{"top": 0, **kw})


def test_tensors_that_are_not_on_a_gpu():
    with pytest.raises(KernelError, match="CUDA"):
        ops.token_logprobs(torch.zeros(2, 5))
    with pytest.raises(KernelError, match="CUDA"):
        ops.head_logprobs(torch.zeros(2, 8), torch.zeros(5, 8))
    with pytest.raises(KernelError, match="CUDA"):
        ops.linear_act(torch.zeros(2, 8), torch.zeros(5, 8))


def test_activations_without_a_name():
    for name in ("tanh", "GELU", "", None):
        with pytest.raises(KernelError, match="activation"):
            ops.linear_act(torch.zeros(2, 8), torch.zeros(5, 8), None, name)


def test_entry_points_refuse_sizes_they_do_not_take():
    """The C entries answer with an error code and a text, without a launch."""
    import ctypes
    from infer_b200.csrc.build import load_module
    head = load_module("score_head")
    n = ctypes.c_int64()
    i64 = ctypes.c_int64
    for sizes in ((0, 5, 8), (4, 0, 8), (4, 5, 0), (4, 5, 12), (1 << 30, 5, 8), (4, 1 << 30, 8)):
        assert head.ib_head_logprobs_scratch(*map(i64, sizes), 0, 148, ctypes.byref(n)) < 0 and head.ib_last_error()
    assert head.ib_head_logprobs_scratch(i64(4), i64(5), i64(8), 21, 148, ctypes.byref(n)) < 0
    assert head.ib_head_logprobs_scratch(i64(2048), i64(151936), i64(1536), 20, 148, ctypes.byref(n)) == 0 and 0 < n.value < 64 << 20
    act = load_module("act_tc")
    w, s = ctypes.c_int(), ctypes.c_int()
    for sizes in ((0, 5, 8), (4, 0, 8), (4, 5, 12), (1 << 30, 5, 8)):
        assert act.ib_linear_act_plan(*map(i64, sizes), 148, ctypes.byref(w), ctypes.byref(s), None) < 0 and act.ib_last_error()
    null = ctypes.c_void_p()
    for args in ((12, 1, 0, 64, 1), (64, 1, 9, 64, 1), (64, 1, 0, 48, 1), (64, 1, 0, 64, 3), (64, 7, 0, 64, 1), (64, 1, 0, 64, 4)):
        K, dtype, a, width, slices = args
        rc = act.ib_linear_act(null, null, null, null, null, i64(4), i64(5), i64(K), dtype, a, width, slices, 148, null, null)
        assert rc < 0 and act.ib_last_error(), args
    cut = load_module("lin32_cut")
    ns = ctypes.c_int64()
    for sizes in ((0, 5, 8), (4, 0, 8), (4, 5, 0), (4, 5, 16385), (1 << 30, 5, 8), (4, 1 << 30, 8)):
        assert cut.ib_linear_f32_cut_plan(*map(i64, sizes), 148, ctypes.byref(w), ctypes.byref(n), ctypes.byref(ns)) < 0 and cut.ib_last_error()
    assert cut.ib_linear_f32_cut_plan(i64(4), i64(5), i64(8), 1, ctypes.byref(w), ctypes.byref(n), ctypes.byref(ns)) < 0
    for sizes in ((1, 1, 1), (301, 2301, 1001), (5000, 130, 16384)):
        assert cut.ib_linear_f32_cut_plan(*map(i64, sizes), 148, ctypes.byref(w), ctypes.byref(n), ctypes.byref(ns)) == 0
        assert w.value in (32, 64, 96, 128) and n.value == 6 * (sizes[0] + sizes[1]) * -(-sizes[2] // 8) * 8
    some = ctypes.c_void_p(64)
    for K, a, width, scratch, status in ((16385, 0, 64, some, some), (64, 9, 64, some, some), (64, -1, 64, some, some), (64, 0, 48, some, some),
                                         (64, 0, 64, null, some), (64, 0, 64, ctypes.c_void_p(8), some), (64, 0, 64, some, null)):
        assert cut.ib_linear_f32_cut(null, null, null, null, null, i64(4), i64(5), i64(K), a, width, scratch, 148, status, null) < 0 and cut.ib_last_error()


@pytest.mark.parametrize("M,N,K", [(129, 1, 8), (129, 18944, 64), (300, 1000, 1536), (500, 1536, 8960), (2048, 18944, 3584), (4096, 33, 18944), (1 << 20, 7, 8)])
def test_plans_of_products_stay_within_the_kernels_ranges(M, N, K):
    from infer_b200 import fast_ops
    for sms in (2, 132, 148):
        pairs, width, slices = fast_ops._act_plan(M, N, K, sms)
        assert pairs and width % 32 == 0 and 32 <= width <= 256 and slices in (1, 2, 4)
        assert slices == 1 or -(-K // 64) >= 2 * slices


@pytest.mark.parametrize("M", [17, 40, 100, 128])
@pytest.mark.parametrize("N,K", [(33, 64), (300, 520), (1536, 8960), (18944, 3584), (18944, 18944), (40, 18944)])
def test_plans_of_few_rows(M, N, K):
    from infer_b200 import fast_ops
    for float_out in (False, True):
        pairs, width, slices = fast_ops._act_plan(M, N, K, 148, float_out)
        if pairs:
            assert width % 32 == 0 and 32 <= width <= 256 and slices in (1, 2, 4)
        else:
            assert width in (16, 32, 64, 128) and 1 <= slices <= 8
            assert not float_out or -(-(-(-K // 64)) // slices) * 64 <= 768, "a long chain of float sums"


@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 151936), (18, 151936), (19, 151936), (74, 151936), (75, 50257), (149, 151936), (5000, 300)])
def test_clusters_of_a_row(rows, vocab):
    c = ops._logprobs_cluster(rows, vocab, 148)
    assert c in (1, 2, 4, 8) and (c == 1 or rows * c <= 2 * 148)


def test_scores_travel_through_a_scheduler_with_any_engine():
    """An engine whose handles carry scores, and one that knows nothing of them."""
    from infer_b200.engine.scheduler import BatchEngine, Request, SampleParams, Scheduler, SchedulerConfig, TokenScore

    class Fake(BatchEngine):
        max_seq_len, max_requests = 64, 4

        def __init__(self, scored): self.scored = scored
        def capacity_tokens(self): return 1000
        def add_request(self, rid): pass
        def end_request(self, rid): pass
        def tokens_that_fit(self, wanted, rid, n): return n
        def can_run(self, wanted): return True
        def has_room(self, n): return True
        def pages_in_use(self): return 0
        def pages_total(self): return 1
        def run(self, batch): return {b.rid: 7 for b in batch if b.sample is not None}

        def run_async(self, batch):
            handle = super().run_async(batch)
            if self.scored:
                handle.scores = {b.rid: TokenScore(-1.5, 2.0, [(7, -1.5)]) for b in batch if b.sample is not None and b.sample.logprobs is not None}
            return handle
    with pytest.raises(ValueError):
        Scheduler(Fake(True)).submit(Request("c", [1], 2, 0, SampleParams(logprobs=21)))
    for overlap in (False, True):
        for scored in (False, True):
            sch = Scheduler(Fake(scored), SchedulerConfig(overlap=overlap))
            sch.submit(Request("a", [1, 2], 3, 0, SampleParams(logprobs=1)))
            sch.submit(Request("b", [1, 2, 3], 2))
            sch.run_until_idle()
            done = {c.id: c for c in sch.completed}
            assert done["a"].tokens == [7] * 3 and done["b"].tokens == [7] * 2 and done["b"].scores == []
            assert done["a"].scores == ([TokenScore(-1.5, 2.0, [(7, -1.5)])] * 3 if scored else [])
