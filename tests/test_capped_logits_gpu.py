"""Log probabilities under a cap: a value is the same logit wherever the kernels evaluate it, so that a token that is all but certain keeps its digits; and values
whose product with scale / cap is no float32 number.

Tolerances. A logit cap tanh(u): u = z (scale / cap) carries two roundings, 2 x 2^-24 |u|, of which tanh keeps at most |u| / cosh^2 u < 0.45 of its size; tanh itself
5 x 2^-24, the product with the cap one more: off by less than 7 x 2^-24 cap. Where a token's probability is p, the others' share S - 1 of the sum S is at
most (1 - p) / p, and an error of 7 x 2^-24 cap in each difference l - m moves it by twice that times itself; its exponentials' errors (test_logprobs_gpu.py: below
40 x 2^-24 of each) come on top. S itself is near 1 once the token is in it, and each addition from there on rounds by half a step of a number in [1, 2), 2^-24: at
most 10 within the token's group of 16 and 2 groups behind it, 10 in the block and 5 among a row's CTAs from logits, 18 within the token's group of 32 columns, 16 groups
behind it, 19 chunks a lane and 5 lanes from a head's rows: below 60 x 2^-24. The logarithm of a number next to 1 rounds once more.
"""
import math

import pytest
import torch

from test_logprobs_gpu import DEV, STEP, check

pytestmark = pytest.mark.gpu


def _sure(r, l, tokens, cap):
    want = torch.log_softmax(l, 1).gather(1, tokens.long()[:, None])[:, 0]
    got = r.logprob.double()
    rest = -torch.expm1(want) / want.exp()
    assert (got <= 0).all(), "likelier than 1"
    over = (got - want).abs() - (61 * STEP + rest * (2 * 7 * STEP * cap + 40 * STEP))
    assert over.max().item() <= 0, f"{over.max().item():.3e} beyond its bound"
    if r.top_ids.shape[1]:
        assert torch.equal(r.top_ids[:, 0], tokens) and torch.equal(r.top_logprobs[:, 0], r.logprob)


@pytest.mark.parametrize("cap", [10.0, 30.0, 45.5, 60.0])
@pytest.mark.parametrize("scale", [1.0, 0.7, 1.9])
def test_a_sure_token_keeps_its_digits(cap, scale):
    from infer_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(int(cap))
    for B, V, H in ((5, 300, 64), (40, 5003, 64), (300, 50257, 128)):
        # each row's token at another place of tanh (u from 0.2 to 2.2), the others far below
        u = torch.linspace(0.2, 2.2, B, device=DEV)
        z = (torch.randn(B, V, device=DEV, generator=g) * 0.5 + (u - 1.5)[:, None] * cap / scale)
        t = torch.randint(0, V, (B,), device=DEV, generator=g, dtype=torch.int32)
        z[torch.arange(B, device=DEV), t.long()] = u * cap / scale
        for top in (0, 4):
            r = ops.token_logprobs(z, t, top, scale=scale, softcap=cap)
            _sure(r, cap * torch.tanh(z.double() * scale / cap), t, cap)
        # rows with a single one choose a column of the matrix: each logit is a bfloat16 number, exactly
        w = z.t().bfloat16()[:, :min(B, H)].contiguous()
        w = torch.nn.functional.pad(w, (0, H - w.shape[1])).contiguous()
        which = torch.arange(B, device=DEV) % min(B, H)
        x = torch.zeros(B, H, device=DEV, dtype=torch.bfloat16)
        x[torch.arange(B, device=DEV), which] = 1.0
        th = t[which].contiguous()
        zh = w.double().t()[which]
        for top in (0, 4):
            r = ops.head_logprobs(x, w, th, top, scale=scale, softcap=cap)
            _sure(r, cap * torch.tanh(zh * scale / cap), th, cap)


def test_no_token_is_likelier_than_one_without_a_cap():
    from infer_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(9)
    z = torch.randn(2000, 500, device=DEV, generator=g) - 60
    t = torch.randint(0, 500, (2000,), device=DEV, generator=g, dtype=torch.int32)
    z[torch.arange(2000, device=DEV), t.long()] = 40 + 20 * torch.rand(2000, device=DEV, generator=g)
    for scale in (1.0, 0.7, 1.3):
        r = ops.token_logprobs(z, t, 1, scale=scale)
        assert (r.logprob <= 0).all() and (r.logprob >= -4 * STEP).all() and torch.equal(r.logprob, r.top_logprobs[:, 0])


@pytest.mark.parametrize("V", [40, 8200, 50257])
@pytest.mark.parametrize("scale,cap", [(2.0, 0.5), (1.0, 30.0), (4.0, 30.0), (1e18, 1e-18), (1.0, 0.25)])
def test_values_whose_product_is_no_float(V, scale, cap):
    """Masks of the type's lowest value are finite logits: -cap under a cap; +inf is the cap; -inf stays masked, a NaN is one."""
    from infer_b200 import ops
    inf, low = math.inf, torch.finfo(torch.float32).min
    g = torch.Generator(device=DEV).manual_seed(V)
    n = lambda: torch.randn(V, device=DEV, generator=g)
    every = torch.arange(V, device=DEV)
    rows = [torch.full((V,), low, device=DEV), n().masked_fill(every % 3 == 1, low), n().masked_fill(every % 3 == 1, low).masked_fill(every % 3 == 2, -inf),
            n().masked_fill(every % 5 == 1, -low).masked_fill(every % 5 == 2, inf), torch.full((V,), -inf, device=DEV),
            n().masked_fill(every == V // 2, math.nan), torch.full((V,), -inf, device=DEV).masked_fill(every == 3, low), torch.full((V,), inf, device=DEV)]
    z = torch.stack(rows)
    l = cap * torch.tanh(z.double() * scale / cap).masked_fill(z == -inf, -inf)
    t = torch.arange(len(rows), device=DEV, dtype=torch.int32) % V
    for top in (0, 7):
        check(ops.token_logprobs(z, t, top, scale=scale, softcap=cap), l, z, t, top, 7 * STEP * cap)
