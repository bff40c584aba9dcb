"""Scores through the public entry points: of given prompts, of generated tokens, and the operators as a run of them."""
import math

import numpy as np
import pytest
import torch

import helpers as H

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SEED = 5


def _llm(name, dtype, **kw):
    from infer_b200.engine.generation import LLM
    kw.setdefault("slots", 4)
    kw.setdefault("max_seq", 256)
    return LLM(None, dtype=dtype, spec=H.spec_of(H.TINY[name]), weights=H.make_weights(name, SEED), **kw)


def _log_softmax(rows):
    return torch.log_softmax(torch.as_tensor(rows, dtype=torch.float64), -1).numpy()


def _check_score(score, ids, rows, top, tol):
    """rows: logits behind each id but the last."""
    lp = _log_softmax(rows)
    n = len(ids) - 1
    assert score.logprobs.shape == score.entropies.shape == (n,) and score.top_ids.shape == score.top_logprobs.shape == (n, top)
    if n == 0:
        return
    assert np.abs(score.logprobs - lp[np.arange(n), ids[1:]]).max() <= tol
    assert np.abs(score.entropies - -(np.exp(lp) * lp).sum(-1)).max() <= 4 * tol
    best = -np.sort(-lp, axis=-1)[:, :top]
    assert np.abs(score.top_logprobs - best).max(initial=0) <= tol
    assert np.abs(np.take_along_axis(lp, score.top_ids.astype(np.int64), -1) - best).max(initial=0) <= 2 * tol


@pytest.mark.parametrize("name", ["a", "b", "c"])
def test_a_prompts_score_in_32_bits(name):
    """Logits of the 32-bit path are at most 2e-5 of their size off (as in its other tests): logprob by twice that."""
    cfg = H.TINY[name]
    prompts = [H.random_ids(cfg, n, 700 + n) for n in (1, 2, 33, 70, 17, 5)]
    llm = _llm(name, torch.float32, max_batch_tokens=24)
    free = llm.engine.cache.pages_free()
    scores = llm.score(prompts, top=7)
    assert llm.engine.cache.pages_free() == free and not llm.engine.cache.requests
    for p, s in zip(prompts, scores):
        ref = H.oracle(cfg, SEED, H.STORED_DTYPE[name], torch.float32, p)
        _check_score(s, p, ref[:-1], 7, 2 * H.F32_ATOL * max(1.0, float(np.abs(ref).max())) + 1e-5)
    assert scores[0].perplexity == 1.0
    assert scores[3].perplexity == pytest.approx(math.exp(-float(scores[3].logprobs.mean())), rel=1e-5)
    again = llm.score([prompts[3]], top=0)[0]
    assert np.array_equal(again.logprobs, scores[3].logprobs) or np.abs(again.logprobs - scores[3].logprobs).max() < 1e-4


@pytest.mark.parametrize("budget", [512, 48])
def test_a_prompts_score_in_bfloat16_is_that_of_its_logits(budget):
    """Against the engine's own logits of the same portions: the head's sums in another order, 2e-6 of their conditioning, well below 1e-4."""
    cfg = H.TINY["b"]
    prompts = [H.random_ids(cfg, n, 800 + n) for n in (150, 40, 3)]
    llm = _llm("b", torch.bfloat16, max_batch_tokens=budget, slots=1)
    scores = llm.score(prompts, top=5)
    eng = llm.engine
    for p, s in zip(prompts, scores):
        eng.add_request("r")
        rows, n = [], 0
        while n < len(p) - 1:
            m = min(budget, len(p) - 1 - n)
            rows.append(eng.step([("r", p[n:n + m], list(range(m)))]).cpu().numpy())
            n += m
        eng.end_request("r")
        _check_score(s, p, np.concatenate(rows), 5, 1e-4)
    eng.check_status()


def test_score_refuses_and_leaves_nothing_behind():
    from infer_b200.engine import OutOfPages
    llm = _llm("a", torch.bfloat16, max_seq=64, slots=2)
    for prompts, kw in (([[]], {}), ([[1, 999]], {}), ([[1, -1]], {}), ([list(range(70))], {}), ([[1, 2]], {"top": 21}), ([[1, 2]], {"top": -1})):
        with pytest.raises(ValueError):
            llm.score(prompts, **kw)
    assert not llm.engine.cache.requests
    assert llm.score([]) == []
    for rid in ("x", "y"):
        llm.engine.add_request(rid)
    with pytest.raises(OutOfPages):
        llm.score([[1, 2, 3]])
    for rid in ("x", "y"):
        llm.engine.end_request(rid)
    assert len(llm.score([[1, 2, 3]])[0].logprobs) == 2
    with pytest.raises(ValueError):
        llm.engine.add_request("z")
        llm.engine.step_logprobs([("z", [1, 2], [0, 1])], [1])
    llm.engine.end_request("z")


def test_step_logprobs_without_wanted_places():
    llm = _llm("a", torch.bfloat16)
    eng = llm.engine
    eng.add_request("r")
    r = eng.step_logprobs([("r", [1, 2, 3], [])], [], 4)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 4)
    assert eng.step_logprobs([], [], 2).top_ids.shape == (0, 2)
    r = eng.step_logprobs([("r", [4], [0])], [-1], 2)                    # what came before is in the cache; no token is asked for
    assert r.logprob.item() == 0.0 and r.top_ids.shape == (1, 2)
    eng.end_request("r")


@pytest.mark.parametrize("overlap", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_generated_tokens_and_their_scores(dtype, overlap):
    """The same tokens as without scores; each score is that of the model's own distribution at its place."""
    cfg = H.TINY["b"]
    prompts = [H.random_ids(cfg, n, 900 + n) for n in (9, 40, 1)]
    for kw in ({}, {"temperature": 0.9, "seed": 4}, {"temperature": 0.7, "seed": 2, "top_k": 30, "top_p": 0.9}):
        llm = _llm("b", dtype, overlap=overlap)
        plain = llm.generate(prompts, max_new=12, **kw)
        got = llm.generate(prompts, max_new=12, logprobs=5, **kw)
        assert [ids for ids, _ in got] == plain
        for p, (ids, scores) in zip(prompts, got):
            assert len(scores) == len(ids)
            want = llm.score([p + ids], top=5)[0]
            tol = 1e-4 if dtype == torch.float32 else 0.15                # (bfloat16: other kernels for other batches; logits O(1))
            for i, s in enumerate(scores):
                k = len(p) - 1 + i
                assert abs(s.logprob - want.logprobs[k]) <= tol and abs(s.entropy - want.entropies[k]) <= tol
                assert len(s.top) == 5 and all(a[1] >= b[1] for a, b in zip(s.top, s.top[1:]))
                assert abs(s.top[0][1] - want.top_logprobs[k][0]) <= tol
                if not kw:
                    assert s.top[0][0] == ids[i] and s.logprob == s.top[0][1]
    assert len(llm.generate([prompts[0]], max_new=3, logprobs=0)[0][1][0].top) == 0
    with pytest.raises(ValueError):
        llm.generate(prompts, logprobs=21)


def test_requests_with_and_without_scores_share_steps_and_survive_preemption():
    from infer_b200.engine import Engine
    from infer_b200.engine.generation import GenerationEngine
    from infer_b200.engine.scheduler import Request, SampleParams, Scheduler, SchedulerConfig
    cfg = H.TINY["a"]
    prompts = [H.random_ids(cfg, 20, 400 + i) for i in range(4)]
    free = _llm("a", torch.float32, max_seq=64).generate(prompts, max_new=30, temperature=0.7, seed=5)
    eng = Engine(H.spec_of(cfg), H.make_weights("a", SEED), dtype=torch.float32, max_tokens=9 * 16, max_requests=4, max_seq_len=64)
    for overlap in (False, True):
        sch = Scheduler(GenerationEngine(eng), SchedulerConfig(max_batch_tokens=64, overlap=overlap))
        for i, p in enumerate(prompts):
            sch.submit(Request(i, list(p), 30, 0, SampleParams(0.7, 5, logprobs=(None, 3, 0, 8)[i])))
        sch.run_until_idle()
        assert sch.preemptions > 0
        done = {c.id: c for c in sch.completed}
        for i in range(4):
            assert done[i].tokens == free[i]
            n = (None, 3, 0, 8)[i]
            assert len(done[i].scores) == (0 if n is None else 30) and all(len(s.top) == n for s in done[i].scores)


def test_heads_with_logits_of_their_own_are_scored_by_those():
    from infer_b200.parts.vocab import LinearHead
    llm = _llm("b", torch.bfloat16)
    ids = H.random_ids(H.TINY["b"], 30, 3)
    head = llm.engine.model.head
    before = llm.score([ids])[0]

    class Shifted(LinearHead):
        def forward(self, x):
            logits = super().forward(x)
            logits[:, ids[1]] += 5.0
            return logits
    head.__class__ = Shifted
    after = llm.score([ids])[0]
    assert after.logprobs[0] > before.logprobs[0] + 1
    head.__class__ = LinearHead
    plain = LinearHead.forward
    head.forward = lambda x: plain(head, x) * 0.0
    assert np.abs(llm.score([ids])[0].logprobs + math.log(H.TINY["b"]["vocab_size"])).max() < 1e-4


def test_capped_head_through_an_engine():
    """A design whose head caps its logits: scores are those of the capped logits."""
    from infer_b200.engine.generation import LLM
    from infer_b200.weights import random_weights
    from infer_b200.config import parse_config
    from infer_b200.models import load_preset
    arch, typed = parse_config(load_preset("tiny-pefazen"))
    spec = arch.to_spec(typed)
    assert spec.head.get("softcap")
    llm = LLM(None, dtype="bfloat16", spec=spec, weights=random_weights(spec, 1, torch.bfloat16), slots=2, max_seq=128)
    ids = np.random.default_rng(0).integers(0, spec.vocab_size, 60).tolist()
    s = llm.score([ids], top=3)[0]
    llm.engine.add_request("r")
    rows = llm.engine.step([("r", ids[:-1], list(range(59)))]).cpu().numpy()
    llm.engine.end_request("r")
    _check_score(s, ids, rows, 3, 2e-3)


def test_one_rounding_feed_forward():
    """A dense feed-forward whose activation takes float sums: nearer to 64 bits than with a rounding before it, through the product's own kernel."""
    from infer_b200 import ops
    from infer_b200.config.specs import PartSpec
    from infer_b200.parts import build_part
    from infer_b200.runtime import Runtime
    rt = Runtime(dtype=torch.bfloat16, device=torch.device(DEV), kernels={}, max_seq_len=64)
    g = torch.Generator().manual_seed(1)
    params = {"up_proj.weight": torch.randn(320, 96, generator=g) * 0.1, "down_proj.weight": torch.randn(96, 320, generator=g) * 0.1}
    for act in ("gelu_tanh", "relu_squared"):
        err = {}
        for one in (False, True):
            part = build_part("feed_forward", PartSpec("dense", dict(hidden_size=96, intermediate_size=320, activation=act, one_rounding=one)), rt)
            part.load(params)
            for T in (3, 40, 200):
                x = torch.randn(T, 96, generator=g).bfloat16().to(DEV)
                res = torch.randn(T, 96, generator=g).to(DEV)
                z = x.double() @ part.up.weight.double().t()
                a = z.clamp(min=0) ** 2 if act == "relu_squared" else z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
                want = res.double() + a @ part.down.weight.double().t()
                before = sum(n for k, n in ops.LAUNCH_KINDS.items() if k in ("ib_linear_skinny_act", "ib_linear_act", "ib_gemm_tc"))
                got = part.forward(x, res.clone())
                err.setdefault(one, []).append((got.double() - want).norm().item())
                if one:
                    assert sum(n for k, n in ops.LAUNCH_KINDS.items() if k in ("ib_linear_skinny_act", "ib_linear_act", "ib_gemm_tc")) > before
        assert all(a < b for a, b in zip(err[True], err[False])) or sum(err[True]) < sum(err[False])
    with pytest.raises(ValueError):
        build_part("feed_forward", PartSpec("dense", dict(hidden_size=96, intermediate_size=320, one_rounding=True, gated=True)), rt)


@pytest.mark.parametrize("T", [1, 7, 40, 129, 500])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_run_of_them(T, dtype):
    """As a last layer uses them: up with activation, down into the residual stream, norm, head; against 64 bits on the roundings that the
    types ask for."""
    from infer_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(T)
    H_, I, V = 256, 1000, 5003
    r = lambda *s: torch.randn(*s, device=DEV, generator=g)
    h, n1, n2 = r(T, H_), 1 + 0.1 * r(H_), 1 + 0.1 * r(H_)
    up, down, head = (r(I, H_) / 16).to(dtype), (r(H_, I) / 32).to(dtype), (r(V, H_) / 8).to(dtype)
    bu, bd = 0.1 * r(I), 0.1 * r(H_)
    t = torch.randint(0, V, (T,), device=DEV, dtype=torch.int32, generator=g)
    x = ops.rmsnorm(h, n1, 1e-6, dtype)
    hidden = ops.linear_act(x, up, bu, "gelu_tanh")
    out = ops.linear_act(hidden, down, bd, "none", h, out=h.clone())
    y = ops.rmsnorm(out, n2, 1e-6, dtype)
    got = ops.head_logprobs(y, head, t, 5)
    z = x.double() @ up.double().t() + bu.double()
    a = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    o = h.double() + a @ down.double().t() + bd.double()
    yy = o * torch.rsqrt((o * o).mean(1, keepdim=True) + 1e-6) * n2.double()
    lp = torch.log_softmax(yy @ head.double().t(), -1)
    want = lp.gather(1, t.long()[:, None])[:, 0]
    # each rounding to the type (hidden rows, normalised rows) moves a logit by half a step of terms that add up at random: a few eps / 2 x the logits' size (2)
    eps = torch.finfo(dtype).eps if dtype == torch.bfloat16 else 2.0 ** -21
    assert (got.logprob.double() - want).abs().max().item() <= 16 * eps
    assert (got.top_logprobs.double() - torch.topk(lp, 5).values).abs().max().item() <= 16 * eps
