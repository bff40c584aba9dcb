"""32-bit products with an activation whose operands are cut into three bfloat16 numbers beforehand.

Tolerance: as for the other products. Of a product less than 2^-24 is left out; the sum of 64 elements takes four steps of the tensor core, which
truncate (at most 2^-22 of what they hold, together), and the blocks' sums are added as floats: below 2e-6 of |x| . |w| up to K = 16,384 in any case.
"""
import math

import pytest
import torch

from test_linear_act_gpu import ACTS, DEV, _operands, check

pytestmark = pytest.mark.gpu


def _cut(x, w, bias, act, residual, width, out=None):
    import ctypes
    from infer_b200 import fast_ops, ops
    (M, K), N = x.shape, w.shape[0]
    st = fast_ops.device_state(DEV)
    out = torch.full((M, N), 7.0, device=DEV) if out is None else out
    nbytes = 6 * (M + N) * (-(-K // 8) * 8)
    scratch = torch.full((nbytes + 64,), 255, dtype=torch.uint8, device=DEV)
    ops._call(fast_ops._act_fn("lin32_cut"), x.data_ptr(), w.data_ptr(), None if bias is None else bias.data_ptr(),
              None if residual is None else residual.data_ptr(), out.data_ptr(), M, N, K, ACTS.index(act), width, scratch.data_ptr(), st.sm_count,
              st.status.data_ptr(), ops._stream())
    assert (scratch[nbytes:] == 255).all() and st.status.item() == 0
    return out


# K of one block, of a block that the two small accumulators end with in different ways (256 and 512 elements and next to them), not of 4 elements
@pytest.mark.parametrize("width", [32, 64, 96, 128])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (129, 40, 63), (8, 129, 64), (300, 301, 255), (257, 95, 256), (100, 200, 321), (65, 127, 512), (513, 260, 577),
                                   (40, 33, 1025), (2000, 1000, 130)])
def test_every_width(width, M, N, K):
    x, w, bias, res = _operands(M, N, K, torch.float32)
    for i, act in enumerate(ACTS):
        b, r = (bias if i % 2 else None), (res if i % 3 else None)
        check(_cut(x, w, b, act, r, width), x, w, b, act, r)
    h = res.clone()
    _cut(x, w, bias, "none", h, width, h)
    check(h, x, w, bias, "none", res)


@pytest.mark.parametrize("sign", [False, True])
@pytest.mark.parametrize("M,N,K", [(300, 128, 8960), (70, 64, 16384)])
def test_long_sums_keep_their_digits(M, N, K, sign):
    x, w, _, _ = _operands(M, N, K, torch.float32)
    if sign:
        x, w = x.abs(), w.abs()
    z = x.double() @ w.double().t()
    assert ((_cut(x, w, None, "none", None, 64).double() - z).norm() / z.norm()).item() < 1e-6


@pytest.mark.parametrize("up", [1e30, 1e-30, 1e-34])
def test_scales_far_apart(up):
    """The small parts are kept 2^8 and 2^16 times as large: all but a ten-thousandth of numbers near 1e-34 have all their digits."""
    x, w, bias, res = _operands(200, 150, 700, torch.float32)
    x, w = x * up, w / up
    check(_cut(x, w, bias, "gelu", res, 96), x, w, bias, "gelu", res)
    g = torch.Generator(device=DEV).manual_seed(3)
    x = x * torch.exp(3 * torch.randn(200, 1, device=DEV, generator=g))
    z, c = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    assert ((_cut(x, w, None, "none", None, 32).double() - z).abs() <= 2e-6 * c).all()


@pytest.mark.parametrize("width", [32, 128])
def test_infinities_nan_and_the_largest_numbers(width):
    x, w, _, _ = _operands(300, 200, 520, torch.float32)
    most = torch.finfo(torch.float32).max
    x[0, 5] = math.inf
    x[1, 519] = -math.inf
    x[2, 0] = math.nan
    x[3] = math.inf
    x[131, 7], x[131, 8] = math.inf, -math.inf
    x[140, 9] = most                       # (rounds to infinity in 16 bits; the results are finite)
    w[10, 5] = 0.0                         # infinity times zero
    w[150, 100] = math.inf
    w[151] = math.nan
    w[152, 3] = -most
    y = _cut(x, w, None, "none", None, width)
    z = x.double() @ w.double().t()
    want = torch.where(z.abs() > most, torch.sign(z) * math.inf, z)
    near = (z.abs() > 0.5 * most) & z.isfinite()      # a sum in another order may or may not pass the largest number on its way
    assert torch.equal(y.isnan() & ~near, want.isnan())
    assert torch.equal(y.isinf() & ~near, want.isinf() & ~near) and torch.equal(torch.sign(y)[want.isinf() & ~near], torch.sign(want.float())[want.isinf() & ~near])
    ok = want.isfinite() & ~near
    c = x.double().abs() @ w.double().abs().t()
    assert ok.sum().item() > 290 * 190 and ((y.double() - z).abs()[ok] <= 2e-6 * c[ok]).all()
    z = torch.full((300, 520), math.nan, device=DEV)
    assert _cut(z, w, None, "none", None, width).isnan().all()


def test_rows_and_results_that_start_anywhere():
    x, w, bias, res = _operands(200, 130, 260, torch.float32)
    for shift in (1, 2, 3):
        at = lambda t: torch.empty(t.numel() + shift, device=DEV)[shift:].view(t.shape).copy_(t)
        out = torch.empty(200 * 130 + shift, device=DEV)[shift:].view(200, 130)
        check(_cut(at(x), at(w), at(bias), "silu", at(res), 64, out), x, w, bias, "silu", res)


@pytest.mark.parametrize("M,N,K,cut", [(301, 2301, 1000, True), (1024, 1024, 1024, True), (500, 5003, 1000, True), (129, 1000, 1000, False), (257, 128, 16000, False),
                                       (64, 3000, 1000, False), (300, 1000, 17000, False),
                                       (2054, 3014, 65, True), (1000, 100, 500, True), (300, 300, 100, False), (65, 18000, 100, False)])
def test_the_kernel_that_a_product_takes(M, N, K, cut):
    from infer_b200 import ops
    x, w, bias, res = _operands(M, N, K, torch.float32)
    before = ops.LAUNCH_KINDS["ib_linear_f32_cut"]
    y = ops.linear_act(x, w, bias, "gelu", res)
    assert (ops.LAUNCH_KINDS["ib_linear_f32_cut"] > before) == cut
    check(y, x, w, bias, "gelu", res)


def test_calls_on_two_streams_and_in_a_graph_do_not_meet():
    from infer_b200 import ops
    x, w, bias, res = _operands(301, 2301, 1000, torch.float32)
    want = ops.linear_act(x, w, bias, "gelu", res)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append(ops.linear_act(x, w, bias, "gelu", res))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    captured = []
    for g in graphs:
        with torch.cuda.graph(g):
            captured.append(ops.linear_act(x, w, bias, "gelu", res))
    for _ in range(2):
        x.copy_(x.flip(0).clone())
        fresh = ops.linear_act(x, w, bias, "gelu", res)
        for g, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(c, fresh) for c in captured)


def test_every_result_computed_again():
    """All results infinite, the longest K: the warps that compute them again are not done before the issuer would wait, and are done in time."""
    x = torch.full((300, 16384), math.inf, device=DEV)
    w = torch.rand(260, 16384, device=DEV) + 0.5
    y = _cut(x, w, None, "none", None, 128)
    assert torch.equal(y, torch.full((300, 260), math.inf, device=DEV))
