"""A product with bias, activation and residual, rounded once, against the formula in 64 bits.

Tolerance. The product is off by at most 2e-6 of its conditioning c = |x| . |w| (as for the other products on the tensor cores; the 32-bit ones stay
below that too), and so is the sum with the bias. An activation passes it on times its slope: at most 1.13 (gelu), for relu
squared 2 |z|. Its own evaluation is off by less than 4 x 2^-24 of the result's size (gelu's own fit 24 x 2^-24) and, where it is z sigmoid(y), by 2^-23 |y| of it, with |y| at
most 16 where the result is above 2^-23 of |z|: 2^-18 of |result| covers both. At the end one rounding: half a step.
"""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ACTS = ("none", "relu", "relu_squared", "gelu_tanh", "gelu", "silu")


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "relu_squared":
        return z.clamp(min=0) ** 2
    if act == "gelu_tanh":
        # 1 + tanh u = 2 sigmoid(2 u); as written, the sum keeps nothing of it below u = -18.7, in 64 bits either
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def check(y, x, w, bias, act, residual):
    z = x.double() @ w.double().t()
    c = x.double().abs() @ w.double().abs().t()
    if bias is not None:
        z, c = z + bias.double(), c + bias.double().abs()
    a = _act(z, act)
    want = a if residual is None else a + residual.double()
    slope = 2 * z.abs() + 1e-3 if act == "relu_squared" else 1.13
    bound = slope * 2e-6 * c + (2e-6 * c) ** 2 + 2.0 ** -18 * a.abs() + torch.finfo(y.dtype).eps / 2 * (want.abs() * 1.001) + 2.0 ** -22 * want.abs() + 1e-12
    over = ((y.double() - want).abs() - bound).max().item()
    assert y.isfinite().all() and over <= 0, f"{over:.3e} beyond the bound"


SIZES = [(1, 1, 64), (1, 300, 8), (2, 320, 96), (8, 8960, 1536), (16, 301, 1000), (17, 300, 520), (33, 1, 72), (64, 1536, 8960), (100, 777, 200), (128, 128, 128), (129, 128, 128),
         (130, 301, 96), (200, 300, 4096), (300, 1000, 1536), (500, 1536, 8960), (1100, 3000, 520), (2048, 2048, 1536), (257, 264, 64), (4000, 72, 136)]


def _operands(M, N, K, dtype):
    g = torch.Generator(device=DEV).manual_seed(M * 7 + N * 3 + K)
    x = torch.randn(M, K, device=DEV, generator=g).to(dtype)
    w = (torch.randn(N, K, device=DEV, generator=g) / math.sqrt(K) * 1.5).to(dtype)
    return x, w, torch.randn(N, device=DEV, generator=g), torch.randn(M, N, device=DEV, generator=g)


@pytest.mark.parametrize("M,N,K", SIZES)
def test_bfloat16(M, N, K):
    from infer_b200 import fast_ops, ops
    x, w, bias, res = _operands(M, N, K, torch.bfloat16)
    st = fast_ops.device_state(DEV)
    st.status.zero_()
    for i, act in enumerate(ACTS):
        b = bias if i % 2 else None
        y = ops.linear_act(x, w, b, act)
        assert y.dtype == torch.bfloat16 and y.shape == (M, N)
        check(y, x, w, b, act, None)
        check(ops.linear_act(x, w, b, act, None, torch.float32), x, w, b, act, None)
        y = ops.linear_act(x, w, b, act, res)
        assert y.dtype == torch.float32
        check(y, x, w, b, act, res)
        check(ops.linear_act(x, w, b, act, res, torch.bfloat16), x, w, b, act, res)
    assert st.status.item() == 0


# tile width, slices of K: every kernel on pairs of SMs, with ragged rows and columns, K of one k-block to several chains, odd numbers of k-blocks
@pytest.mark.parametrize("width,slices", [(32, 1), (64, 1), (96, 2), (128, 4), (160, 1), (192, 4), (224, 4), (256, 1), (256, 2), (32, 4)])
@pytest.mark.parametrize("M,N,K", [(129, 40, 72), (300, 301, 520), (257, 520, 1160), (600, 1000, 2056), (1, 9, 1024)])
def test_pairs_of_sms(width, slices, M, N, K):
    from infer_b200 import fast_ops, ops
    if slices > 1 and -(-K // 64) < 2 * slices:
        slices = 1
    x, w, bias, res = _operands(M, N, K, torch.bfloat16)
    st = fast_ops.device_state(DEV)
    st.status.zero_()
    for dtype, code in ((torch.float32, 0), (torch.bfloat16, 1)):
        for act, b, r in ((0, None, None), (3, bias, None), (5, bias, res), (2, None, res)):
            out = torch.full((M, N), 7.0, dtype=dtype, device=DEV)
            ops._call(fast_ops._act_fn("act_tc"), x.data_ptr(), w.data_ptr(), None if b is None else b.data_ptr(), None if r is None else r.data_ptr(),
                      out.data_ptr(), M, N, K, code, act, width, slices, st.sm_count, st.status.data_ptr(), ops._stream())
            check(out, x, w, b, ACTS[act], r)
    assert st.status.item() == 0


@pytest.mark.parametrize("M,N,K", [(600, 512, 18944), (140, 256, 8960), (2048, 128, 8960)])
def test_long_sums_keep_their_digits(M, N, K):
    """Float results: chains of 512 elements, each off by at most 2^-23 of its running sum at each of 32 steps, below 32 x 2^-23 / 2 of its size on average
    and 1e-6 of the whole in norm (the chains' errors add up as their sizes do); one chain over K would be 1e-5 off."""
    from infer_b200 import ops
    x, w, bias, res = _operands(M, N, K, torch.bfloat16)
    y = ops.linear_act(x, w, None, "none", None, torch.float32).double()
    z = x.double() @ w.double().t()
    assert ((y - z).norm() / z.norm()).item() < 2e-6


@pytest.mark.parametrize("M", [8, 60, 200])
def test_results_and_residuals_that_start_anywhere(M):
    from infer_b200 import ops
    N = 64
    x, w, bias, res = _operands(M, N, 256, torch.bfloat16)
    for shift in (1, 2, 3):
        r = torch.empty(M * N + shift, device=DEV)[shift:].view(M, N).copy_(res)
        for dtype in (torch.float32, torch.bfloat16):
            out = torch.empty(M * N + shift, dtype=dtype, device=DEV)[shift:].view(M, N)
            b = torch.empty(N + shift, device=DEV)[shift:].copy_(bias)
            check(ops.linear_act(x, w, b, "gelu", r, dtype, out), x, w, bias, "gelu", res)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (3, 37, 65), (8, 300, 1000), (17, 1030, 1024), (301, 2301, 1000), (130, 1500, 2048), (64, 100, 7)])
def test_float32(M, N, K):
    from infer_b200 import ops
    x, w, bias, res = _operands(M, N, K, torch.float32)
    for act in ACTS:
        y = ops.linear_act(x, w, bias, act)
        assert y.dtype == torch.float32
        check(y, x, w, bias, act, None)
        check(ops.linear_act(x, w, None, act, res), x, w, None, act, res)
    check(ops.linear_act(x, w, bias, "silu", None, torch.bfloat16), x, w, bias, "silu", None)


@pytest.mark.parametrize("M,N,K", [(5, 64, 99), (40, 301, 7), (200, 130, 1001)])
def test_rows_that_do_not_keep_to_16_bytes(M, N, K):
    from infer_b200 import ops
    x, w, bias, res = _operands(M, N, K, torch.bfloat16)
    check(ops.linear_act(x, w, bias, "gelu"), x, w, bias, "gelu", None)
    x, w, bias, res = _operands(M, N, 96, torch.bfloat16)
    y = torch.empty(M * 96 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(M, 96).copy_(x)
    check(ops.linear_act(y, w, bias, "silu", res), x, w, bias, "silu", res)


@pytest.mark.parametrize("M", [8, 60, 500])
def test_residual_in_place_and_given_results(M):
    from infer_b200 import ops
    x, w, bias, res = _operands(M, 640, 256, torch.bfloat16)
    h = res.clone()
    out = ops.linear_act(x, w, bias, "none", h, out=h)
    assert out.data_ptr() == h.data_ptr()
    check(h, x, w, bias, "none", res)
    y = torch.empty(M, 640, dtype=torch.bfloat16, device=DEV)
    assert ops.linear_act(x, w, bias, "relu", out=y) is y
    check(y, x, w, bias, "relu", None)
    assert ops.linear_act(x[:0], w, bias).shape == (0, 640)


@pytest.mark.parametrize("act", ACTS)
def test_the_ends_of_an_activation(act):
    """Large values of both signs, infinities and NaN (as the formula has them), through each kind of kernel."""
    from infer_b200 import ops
    vals = torch.tensor([-3e38, -1e30, -1e5, -100.0, -20.0, -9.0, -1e-3, -0.0, 0.0, 1e-30, 1e-3, 9.0, 20.0, 100.0, 1e5, 1e18], device=DEV)
    for M in (4, 40, 300):
        x = torch.zeros(M, 64, device=DEV).bfloat16()
        w = torch.zeros(vals.numel(), 64, device=DEV).bfloat16()
        y = ops.linear_act(x, w, vals, act, None, torch.float32)
        want = _act(vals.double(), act).float()
        if act == "gelu":
            want = torch.where(vals < -30, torch.zeros_like(want), want)
        assert y.isnan().sum().item() == 0
        ref = want.expand(M, -1)
        assert torch.where(ref == y, torch.zeros_like(y), (y - ref).abs() - 2.0 ** -17 * ref.abs() - 1e-30).max().item() <= 0
        odd = torch.tensor([math.inf, math.nan, -math.inf], device=DEV)
        y = ops.linear_act(x, w[:3].contiguous(), odd, act, None, torch.float32)
        assert torch.equal(y[:, 0], torch.full((M,), math.inf, device=DEV)) and y[:, 1].isnan().all()
        if act in ("none", "relu", "relu_squared"):
            assert torch.equal(y[:, 2], torch.full((M,), -math.inf if act == "none" else 0.0, device=DEV))


@pytest.mark.parametrize("M,N,K", [(8, 8960, 1536), (64, 1536, 8960), (300, 1536, 8960), (2048, 2048, 1536)])
def test_calls_on_two_streams_and_in_a_graph_do_not_meet(M, N, K):
    from infer_b200 import ops
    x, w, bias, res = _operands(M, N, K, torch.bfloat16)
    want = ops.linear_act(x, w, bias, "gelu", res)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append(ops.linear_act(x, w, bias, "gelu", res))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops.linear_act(x, w, bias, "gelu", res)
    for _ in range(2):
        x.copy_(x.flip(0).clone())
        fresh = ops.linear_act(x, w, bias, "gelu", res)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, fresh)
