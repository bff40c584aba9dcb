"""32-bit products whose results are computed again because they are not finite, where a pair of SMs has more than one tile: the issuer, the producer and the other
CTA wait meanwhile, and their bounded waits (about a second) must not run out. A tile's results took 137 ms at the longest K."""
import math

import pytest
import torch

from test_linear_act_gpu import DEV
from test_linear_act_f32_gpu import _cut

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K,width", [(260, 128), (1024, 96), (16384, 128)])
def test_tiles_that_wait_for_one_that_is_computed_again(K, width):
    from infer_b200 import fast_ops
    sms = fast_ops.device_state(torch.device(DEV)).sm_count
    M, N = 300, width * (sms // 2 + 2) - 5                       # two tiles of rows: every pair has two tiles at least, some three
    x = torch.full((M, K), math.inf, device=DEV)
    w = torch.rand(N, K, device=DEV) + 0.5
    y = _cut(x, w, None, "none", None, width)                    # (asserts that no wait ran out)
    assert (y == math.inf).all()
    # every other row finite: what is not computed again is the product
    g = torch.Generator(device=DEV).manual_seed(K)
    x[1::2] = torch.randn(M // 2, K, device=DEV, generator=g)
    y = _cut(x, w, None, "relu", None, width)
    assert (y[::2] == math.inf).all()
    z = (x[1::2].double() @ w.double().t()).clamp(min=0)
    c = x[1::2].double().abs() @ w.double().t()
    assert ((y[1::2].double() - z).abs() - (2e-6 * c + 2.0 ** -22 * z)).max().item() <= 0
