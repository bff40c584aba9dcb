"""``token_logprobs`` with alternatives where a CTA's share of a row is more than one segment (98,304 elements): the list that goes from one to the next. Tolerances as
derived in test_logprobs_gpu.py."""
import math

import pytest
import torch

from test_logprobs_gpu import DEV, check

pytestmark = pytest.mark.gpu
SEGMENT = 48 * 512 * 4


@pytest.mark.parametrize("B,V,top", [(160, 151936, 1), (160, 151936, 20), (80, 200001, 1), (80, 200001, 20), (150, 98304, 20), (150, 98311, 20), (150, 300007, 5)])
@pytest.mark.parametrize("shift", [0, 3])
def test_rows_of_several_segments(B, V, top, shift):
    from infer_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(V + top)
    l = torch.empty(B * V + shift, device=DEV)[shift:].view(B, V)
    l.copy_(torch.randn(B, V, device=DEV, generator=g) * 2.5)
    every = torch.arange(V, device=DEV)
    share = -(-V // ops._logprobs_cluster(B, V, ops.sm_count(l.device)))
    edges = sorted({e for lo in range(0, V, share) for e in range(lo, V, SEGMENT)} | {V})
    l[0] = every.float() / 1024                                          # every segment beats the list so far
    l[1] = l[0].flip(0).clone()                                          # none does
    l[2] = 0.0                                                           # the lowest ids stay
    l[3] = (l[3] * 2).round()                                            # many ties
    l[4] = -math.inf
    for e in edges:                                                      # the best around each segment's end, equal ones on both sides
        l[5, max(0, e - 5):e + 5] = 30.0
        l[6, max(0, e - 3):e] = 20.0 + e / V
        l[6, e:e + 3] = 21.0 + e / V
        l[4, max(0, e - 2):e + 1] = 1.0                                  # and nothing else
    l[7] = -math.inf
    l[7, V - 1] = 2.0
    l[8, :min(V, SEGMENT)] = -math.inf                                   # an empty first segment
    l[9, min(V, SEGMENT):] = -math.inf                                   # empty ones behind it
    l[10, (every // 4) % 512 == 77] += 40.0                              # all with one thread
    l[11, V // 2] = math.nan
    t = torch.randint(0, V, (B,), device=DEV, generator=g, dtype=torch.int32)
    check(ops.token_logprobs(l, t, top), l, l, t, top)
