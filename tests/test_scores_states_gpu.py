"""Scores of designs that keep a state per request: a refused call leaves pages, lengths and states as they were."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _llm(preset, dtype="bfloat16", **kw):
    from infer_b200.config import parse_config
    from infer_b200.engine.generation import LLM
    from infer_b200.models import load_preset
    from infer_b200.weights import random_weights
    arch, typed = parse_config(load_preset(preset))
    spec = arch.to_spec(typed)
    return LLM(None, dtype=dtype, spec=spec, weights=random_weights(spec, 3, torch.bfloat16), slots=2, max_seq=128, **kw)


@pytest.mark.parametrize("preset", ["tiny-fozerax", "tiny-ruvenex", "tiny-b"])
def test_a_refused_step_changes_nothing(preset):
    eng = _llm(preset).engine
    ids = np.random.default_rng(1).integers(0, eng.spec.vocab_size, 40).tolist()

    def portions(rid, refused):
        got = []
        eng.add_request(rid)
        for lo, hi in ((0, 20), (20, 39)):
            entry = [(rid, ids[lo:hi], list(range(hi - lo)))]
            if refused:
                free, length = eng.cache.pages_free(), eng.cache.length(rid)
                for asked, top in ((ids[lo + 1:hi + 1], 21), (ids[lo + 1:hi + 1], -1), (ids[lo + 1:hi], 3), ([eng.spec.vocab_size] * (hi - lo), 3)):
                    with pytest.raises(ValueError):
                        eng.step_logprobs(entry, asked, top)
                    assert eng.cache.pages_free() == free and eng.cache.length(rid) == length and eng.cache.requests[rid].reserved == length
            got.append(eng.step_logprobs(entry, ids[lo + 1:hi + 1], 3))
        eng.end_request(rid)
        return [torch.cat(t) for t in zip(*got)]
    plain, after = portions("a", False), portions("b", True)
    assert all(torch.equal(x, y) for x, y in zip(plain, after))
    eng.check_status()


@pytest.mark.parametrize("scale,cap", [(-0.5, 0.0), (1e-20, 0.0), (-1.0, 20.0), (2.0, 1e20)])
def test_a_head_whose_scale_the_operator_does_not_take_is_scored_by_its_logits(scale, cap):
    """Against the engine's own logits: the same kernel on the same logits, so the same bits."""
    from infer_b200 import ops
    eng = _llm("tiny-b").engine
    head = eng.model.head
    head.logit_scale, head.softcap = scale, cap
    ids = np.random.default_rng(2).integers(0, eng.spec.vocab_size, 30).tolist()
    eng.add_request("r")
    got = eng.step_logprobs([("r", ids[:-1], list(range(29)))], ids[1:], 4)
    eng.end_request("r")
    eng.add_request("s")
    logits = eng.step([("s", ids[:-1], list(range(29)))])
    eng.end_request("s")
    want = ops.token_logprobs(logits, torch.tensor(ids[1:], dtype=torch.int32, device=logits.device), 4)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got.logprob.isfinite().all()


@pytest.mark.parametrize("preset", ["tiny-a", "tiny-b", "tiny-pefazen"])
@pytest.mark.parametrize("rows", [1, 7, 39])
def test_a_32_bit_heads_logits_are_stored_for_some_rows_at_a_time(preset, rows, monkeypatch):
    """The 32-bit products sum a row in the same order whatever the number of rows: the same bits."""
    from infer_b200.parts import vocab
    llm = _llm(preset, "float32")
    V = llm.engine.spec.vocab_size
    ids = np.random.default_rng(5).integers(0, V, 41).tolist()
    want = llm.score([ids], top=3)[0]
    monkeypatch.setattr(vocab, "LOGPROB_LOGITS", rows * V + V // 2)
    head, seen = llm.engine.model.head, []
    plain = type(head).forward

    class Counted(type(head)):
        def forward(self, x):
            seen.append(len(x))
            return plain(self, x)
    head.__class__ = Counted
    got = llm.score([ids], top=3)[0]
    assert seen == [rows] * (40 // rows) + ([40 % rows] if 40 % rows else [])
    for a, b in zip((want.logprobs, want.entropies, want.top_ids, want.top_logprobs), (got.logprobs, got.entropies, got.top_ids, got.top_logprobs)):
        assert np.array_equal(a, b)
