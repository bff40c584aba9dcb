"""``Linear`` with an activation: the products that the runtime chooses. Plain ones are the plain kernels, and in 32 bits a row's bits do not depend on how many rows
there are. Tolerances as derived in test_linear_act_gpu.py (its ``check``)."""
import pytest
import torch

from test_linear_act_gpu import DEV, _operands, check

pytestmark = pytest.mark.gpu


def _linear(dtype, w, bias, **kernels):
    from infer_b200.parts.linear import Linear
    from infer_b200.runtime import Runtime
    return Linear(Runtime(dtype=dtype, device=torch.device(DEV), kernels=kernels, max_seq_len=64), w, bias)


@pytest.mark.parametrize("N,K", [(1000, 1000), (130, 500), (1030, 1024), (60, 300)])
@pytest.mark.parametrize("act", ["none", "gelu_tanh", "relu_squared", "silu"])
def test_a_32_bit_rows_bits_do_not_depend_on_the_batch(N, K, act):
    M = 300
    x, w, bias, res = _operands(M, N, K, torch.float32)
    lin = _linear(torch.float32, w, bias)
    whole = lin(x, activation=act)
    check(whole, x, w, bias, act, None)
    added = lin(x, residual=res.clone(), activation=act)
    check(added, x, w, bias, act, res)
    for lo, hi in ((0, 1), (7, 15), (40, 104), (299, 300)):
        assert torch.equal(lin(x[lo:hi].clone(), activation=act), whole[lo:hi])
        assert torch.equal(lin(x[lo:hi].clone(), residual=res[lo:hi].clone(), activation=act), added[lo:hi])


@pytest.mark.parametrize("M", [1, 40, 200])
def test_plain_products_stay_plain(M):
    from infer_b200 import ops
    x, w, bias, res = _operands(M, 520, 256, torch.bfloat16)
    for kernels, fast in (({"linear": "plain"}, False), ({}, True)):
        lin = _linear(torch.bfloat16, w, bias, **kernels)
        before = dict(ops.LAUNCH_KINDS)
        check(lin(x, activation="gelu"), x, w, bias, "gelu", None)
        check(lin(x, residual=res.clone(), activation="silu"), x, w, bias, "silu", res)
        check(lin(x, out_dtype=torch.float32, activation="relu"), x, w, bias, "relu", None)
        ran = {k: n - before.get(k, 0) for k, n in ops.LAUNCH_KINDS.items() if n != before.get(k, 0)}
        assert (ran.get("ib_linear_plain", 0) == ran.get("ib_act_residual", 0) == 3) == (not fast), ran
