"""Log probabilities, entropies and alternatives, from logits and from the rows in front of a head, against the definition in 64 bits.

Tolerances. With x = l - m and e = exp x: x is rounded once, x log2(e) once more and the constant is half a step off (together
2.5 x 2^-24 |x| of e), the hardware's 2^y is 2 ulp off (2^-22 of e), and S is a sum of at most 60 sums after one another (60 x 2^-24). Weighted with the
probabilities |x| is at most ln V <= 13 on average, so S is off by less than (2.5 * 13 + 4 + 60) x 2^-24 of itself and ln S by as much: below
100 x 2^-24. (l - m) - ln S is rounded twice more, each 2^-24 of something that is at most |result| + |ln S|, and ln itself is 1 ulp off:
100 x 2^-24 + 2^-22 |result| holds with room. D / S has the errors of S, those of D's terms (the same again) and |D / S| <= 13: the
entropy is off by less than 100 x 2^-24 (1 + 2 |D / S|). Logits that are a product's sums are off by themselves: where they are not whole multiples of
a step that makes every sum exact, an error of c in each logit moves logprob by at most 2 c and the entropy by 2 c times (1 + |D / S|).
With a cap: tanhf is 2 ulp off, l / cap and the product with it are rounded: 4 x 2^-24 cap in each logit.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
STEP = 2.0 ** -24


def _definition(l, z, tokens, top):
    """float64 rows l (z: what the alternatives go by): (logprob, entropy, ids, logprobs, |D / S|)."""
    l = l.double()
    T, V = l.shape
    bad = (l.isnan() | (l == math.inf)).any(1)
    m = l.masked_fill(l.isnan(), -math.inf).amax(1, keepdim=True)
    empty = (m == -math.inf)[:, 0] & ~bad
    x = l - torch.where(m.isfinite(), m, torch.zeros_like(m))
    e = x.exp()
    S = e.sum(1)
    D = torch.where(e > 0, e * x, torch.zeros_like(x)).sum(1)
    lp = x - S.log()[:, None]
    lp[bad] = math.nan
    lp[empty] = -math.inf
    entropy = S.log() - D / S
    entropy[bad] = math.nan
    entropy[empty] = 0.0
    t = torch.full((T,), -1, dtype=torch.int64, device=l.device) if tokens is None else tokens.long()
    logprob = lp.gather(1, t.clamp(0, V - 1)[:, None])[:, 0]
    logprob = torch.where(t == -1, torch.zeros_like(logprob), torch.where((t < 0) | (t >= V), torch.full_like(logprob, math.nan), logprob))
    zz = (z.double() + 0.0).masked_fill(z.isnan(), -math.inf)
    keep = min(top, V)
    ids = torch.sort(zz, dim=1, descending=True, stable=True).indices[:, :keep]
    best = lp.gather(1, ids)
    none = zz.gather(1, ids) == -math.inf
    ids, best = ids.masked_fill(none, -1), best.masked_fill(none, -math.inf)
    ids = torch.nn.functional.pad(ids, (0, top - keep), value=-1)
    best = torch.nn.functional.pad(best, (0, top - keep), value=-math.inf)
    ds = torch.where(bad | empty, torch.zeros_like(S), (D / S).abs())
    return logprob, entropy, ids, best, ds


def _near(got, want, bound, what):
    got, want = got.double(), want.double()
    finite = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    same = finite | want.isnan()
    assert torch.equal(got[~same], want[~same]), f"{what}: infinities in other places"
    assert got[finite].isfinite().all(), f"{what}: not finite"
    over = ((got - want).abs() - bound)[finite]
    assert over.numel() == 0 or over.max().item() <= 0, f"{what}: {over.max().item():.3e} beyond its bound"


def check(r, l, z, tokens, top, off=0.0):
    """``off``: how far a logit may be from l by itself."""
    logprob, entropy, ids, best, ds = _definition(l, z, tokens, top)
    assert r.logprob.dtype == r.entropy.dtype == r.top_logprobs.dtype == torch.float32 and r.top_ids.dtype == torch.int32
    assert r.top_ids.shape == r.top_logprobs.shape == (l.shape[0], top)
    assert torch.equal(r.top_ids.long(), ids), "other alternatives"
    bound = lambda v: 100 * STEP + 4 * STEP * v.double().abs().nan_to_num(0, 0, 0) + 2 * off
    _near(r.logprob, logprob, bound(logprob), "logprob")
    _near(r.top_logprobs, best, bound(best), "top_logprobs")
    _near(r.entropy, entropy, (100 * STEP + 2 * off) * (1 + 2 * ds), "entropy")


def _logits(B, V, seed, shift=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    buf = torch.randn(B * V + shift, device=DEV, generator=g) * 2.5
    l = buf[shift:].view(B, V)
    l[torch.arange(B, device=DEV), torch.randint(0, V, (B,), device=DEV, generator=g)] += 12 * torch.rand(B, device=DEV, generator=g)
    t = torch.randint(0, V, (B,), device=DEV, generator=g, dtype=torch.int32)
    if B > 1:
        t[-1] = -1
    return l, t


@pytest.mark.parametrize("B,V,top", [(1, 1, 1), (2, 2, 5), (3, 3, 0), (3, 5, 20), (1, 31, 20), (2, 301, 4), (5, 1023, 20), (1, 8192, 20), (2, 8193, 7),
                                     (3, 16389, 20), (1, 50257, 8), (37, 50257, 8), (1, 151936, 20), (64, 151936, 20), (3, 152064, 0), (700, 301, 20),
                                     (600, 9001, 3), (130, 70001, 20), (1, 262147, 20)])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_from_logits(B, V, top, shift):
    from infer_b200 import ops
    l, t = _logits(B, V, B + V + top, shift)
    check(ops.token_logprobs(l, t, top), l, l, t, top)


@pytest.mark.parametrize("V", [40, 8200, 50257])
@pytest.mark.parametrize("top", [0, 1, 20])
def test_rows_out_of_the_ordinary(V, top):
    """Masked rows, ties, sorted rows, values that are not finite, logits far from zero: one batch."""
    from infer_b200 import ops
    inf, low = math.inf, torch.finfo(torch.float32).min
    g = torch.Generator(device=DEV).manual_seed(V)
    n = lambda: torch.randn(V, device=DEV, generator=g)
    up = torch.arange(V, device=DEV).float() / 16
    rows = [torch.full((V,), -inf, device=DEV), torch.zeros(V, device=DEV), up, up.flip(0), torch.full((V,), low, device=DEV), n() * 1e-3 + 1e4,
            n() - 1e30, n() * 50]
    for k in (0, V // 2, V - 1):                                     # one token left
        r = torch.full((V,), -inf, device=DEV); r[k] = 3.0; rows.append(r)
        r = torch.full((V,), low, device=DEV); r[k] = 3.0; rows.append(r)
    rows.append(n().masked_fill(torch.rand(V, device=DEV, generator=g) < 0.9, -inf))
    rows.append(n().masked_fill(torch.arange(V, device=DEV) % 7 != 3, -inf))
    r = n(); r[V // 3] = math.nan; rows.append(r)
    r = n(); r[V // 3] = inf; rows.append(r)
    rows.append(torch.full((V,), math.nan, device=DEV))
    r = torch.full((V,), -inf, device=DEV); r[2] = math.nan; rows.append(r)
    rows.append(torch.where(torch.arange(V, device=DEV) % 2 == 0, torch.tensor(0.0, device=DEV), torch.tensor(-0.0, device=DEV)))      # -0 is 0: lowest ids
    rows.append((n() * 2).round())                                   # many ties
    r = n() - 20; r[5:25] = 10.0; rows.append(r)                     # the best ones side by side, equal
    r = n() - 20; r[torch.arange(0, V, max(1, V // 37), device=DEV)] += 30; rows.append(r)
    l = torch.stack(rows)
    t = torch.arange(len(rows), device=DEV, dtype=torch.int32) % V
    check(ops.token_logprobs(l, t, top), l, l, t, top)
    check(ops.token_logprobs(l.clone(), None, top), l, l, None, top)


def test_large_elements_that_meet_in_one_half_warp_of_a_chunk():
    from infer_b200 import ops
    V = 8192 * 3
    g = torch.Generator(device=DEV).manual_seed(3)
    l = torch.randn(40, V, device=DEV, generator=g)
    unit = torch.arange(V, device=DEV) // 4
    l[:, (unit % 512) // 16 == 11] += 9                              # half-warp 11 of every chunk
    l[20:] = l[20:].sort(1).values
    t = torch.full((40,), 7, dtype=torch.int32, device=DEV)
    check(ops.token_logprobs(l, t, 20), l, l, t, 20)


def test_scaled_and_capped():
    from infer_b200 import ops
    z, t = _logits(6, 5003, 1)
    z = z * 6
    for scale, cap in ((0.25, 0.0), (1.0, 30.0), (0.3, 8.0)):
        l = z.double() * scale
        l = cap * torch.tanh(l / cap) if cap else l
        off = 4 * STEP * (cap or l.abs().max().item())
        check(ops.token_logprobs(z, t, 9, scale=scale, softcap=cap), l, z, t, 9, off)
        masked = torch.rand(z.shape, device=DEV) < 0.5                # what is masked stays masked under a cap
        zm, lm = z.masked_fill(masked, -math.inf), l.masked_fill(masked, -math.inf)
        check(ops.token_logprobs(zm, t, 9, scale=scale, softcap=cap), lm, zm, t, 9, off)


def test_tokens_outside_the_vocabulary_and_the_status_word():
    from infer_b200 import ops
    l, _ = _logits(4, 300, 2)
    t = torch.tensor([299, 300, -1, -2], dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    r = ops.token_logprobs(l, t, 2, status)
    check(r, l, l, t, 2)
    assert status.item() == 1
    status.zero_()
    ops.token_logprobs(l, t.clamp(-1, 299), 2, status)
    assert status.item() == 0
    assert ops.token_logprobs(l[:0], t[:0], 3).top_ids.shape == (0, 3)
    from infer_b200 import fast_ops
    device_status = fast_ops.device_state(DEV).status
    device_status.zero_()
    for T in (4, 40, 300):
        x, w, _ = _head(T, 64, 300, 1)
        th = torch.full((T,), 299, dtype=torch.int32, device=DEV)
        th[1], th[2] = 300, -7
        status.zero_()
        r = ops.head_logprobs(x, w, th, 2, status=status)
        assert status.item() == 1 and r.logprob[1:3].isnan().all() and r.logprob[0].isfinite()
        ops.head_logprobs(x, w, th, 2)
    assert device_status.item() == 0, "a wrong token is the caller's: the device's word stays as it is"
    assert ops.head_logprobs(x[:0], w, th[:0], 3).top_ids.shape == (0, 3)


def test_results_that_are_given():
    from infer_b200 import ops
    from infer_b200.ops import KernelError
    l, t = _logits(5, 700, 1)
    r = ops.TokenLogprobs(torch.empty(5, device=DEV), torch.empty(5, device=DEV), torch.empty(5, 3, dtype=torch.int32, device=DEV), torch.empty(5, 3, device=DEV))
    assert ops.token_logprobs(l, t, 3, out=r) is r
    check(r, l, l, t, 3)
    for bad in (r._replace(entropy=r.entropy[:4]), r._replace(top_ids=r.top_ids.long()), r._replace(top_logprobs=r.top_logprobs.t()), r._replace(logprob=r.logprob.cpu())):
        with pytest.raises(KernelError):
            ops.token_logprobs(l, t, 3, out=bad)
    for bad in (t.long(), t[:4], t.cpu(), t.expand(5, 5)[0].expand(2, 5)):
        with pytest.raises(KernelError):
            ops.token_logprobs(l, bad, 3)
    with pytest.raises(KernelError):
        ops.token_logprobs(l.half(), t, 3)
    with pytest.raises(KernelError):
        ops.token_logprobs(l.t(), None, 3)
    with pytest.raises(KernelError):
        ops.token_logprobs(l[:, :0], t, 3)


def test_rows_beside_the_batch_are_left_as_they_are():
    """Neither results behind the last row nor the inputs around a view are written; a batch inside a larger buffer."""
    from infer_b200 import ops
    big = torch.randn(9, 5003, device=DEV)
    keep = big.clone()
    l = big[2:7]
    big[:2] = math.nan
    big[7:] = math.nan
    pads = [torch.full((12,), 7.0, device=DEV), torch.full((12,), 7.0, device=DEV), torch.full((12, 4), 7, dtype=torch.int32, device=DEV), torch.full((12, 4), 7.0, device=DEV)]
    # (against the definition: a row's sums go by how it lies to 16 bytes, so that a copy elsewhere may differ in its last bits)
    check(ops.token_logprobs(l, None, 4, out=ops.TokenLogprobs(*(p[3:8] for p in pads))), keep[2:7], keep[2:7], None, 4)
    for p in pads:
        assert (p[:3] == 7).all() and (p[8:] == 7).all()
    assert torch.equal(big[2:7], keep[2:7])


def test_calls_on_two_streams_and_in_a_graph_do_not_meet():
    from infer_b200 import ops
    l, t = _logits(3, 151936, 5)
    x, w, th = _head(200, 256, 5000, 1)
    want, want_h = ops.token_logprobs(l, t, 20), ops.head_logprobs(x, w, th, 20)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append((ops.token_logprobs(l, t, 20), ops.head_logprobs(x, w, th, 20)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = (ops.token_logprobs(l, t, 20), ops.head_logprobs(x, w, th, 20))
    l2, x2 = l.flip(0).clone(), x.flip(0).clone()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in got + [captured]:
        assert all(torch.equal(p, q) for p, q in zip(a, want)) and all(torch.equal(p, q) for p, q in zip(b, want_h))
    l.copy_(l2), x.copy_(x2)
    fresh = ops.token_logprobs(l, t, 20), ops.head_logprobs(x, w, th, 20)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(captured, fresh):
        assert all(torch.equal(p, q) for p, q in zip(a, b)), "a replay reads its inputs anew"


# ----------------------------------------------------------------------------- from the rows in front of a head

def _head(T, H, V, seed, dtype=torch.bfloat16):
    """Rows and a matrix on steps that make every sum of products a float32 number (multiples of 2^-15 below 512)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(T, H, device=DEV, generator=g) * 16).round().clamp(-64, 64).mul(2.0 ** -4).to(dtype)
    w = (torch.randn(V, H, device=DEV, generator=g) * (2048 * min(2.5 / math.sqrt(H), 0.06))).round().clamp(-255, 255).mul(2.0 ** -11).to(dtype)
    t = torch.randint(0, V, (T,), device=DEV, generator=g, dtype=torch.int32)
    if T > 1:
        t[-1] = -1
    return x, w, t


HEADS = [(1, 64, 300, 3), (8, 1536, 5000, 20), (9, 64, 301, 20), (16, 1536, 5000, 20), (32, 1536, 9000, 5), (136, 72, 700, 5), (17, 8, 1, 1), (17, 64, 5, 20), (33, 72, 130, 0), (64, 1536, 50257, 20), (100, 200, 301, 8), (128, 136, 1000, 9),
         (129, 64, 300, 20), (130, 72, 5, 20), (256, 1536, 5003, 5), (257, 520, 1000, 0), (300, 1000, 32003, 20), (513, 128, 70000, 1), (1500, 96, 9001, 20),
         (77, 3584, 40000, 20)]


@pytest.mark.parametrize("T,H,V,top", HEADS)
def test_from_a_heads_rows(T, H, V, top):
    from infer_b200 import fast_ops, ops
    x, w, t = _head(T, H, V, T + H + V)
    st = fast_ops.device_state(DEV)
    st.status.zero_()
    z = x.double() @ w.double().t()
    check(ops.head_logprobs(x, w, t, top), z, z, t, top)
    for scale, cap in ((0.5, 0.0), (1.0, 5.0)):
        l = z * scale
        l = cap * torch.tanh(l / cap) if cap else l
        check(ops.head_logprobs(x, w, t, top, scale, cap), l, z, t, top, 4 * STEP * (cap or l.abs().max().item()))
    assert st.status.item() == 0


@pytest.mark.parametrize("T,H,V,top", [(1, 7, 300, 3), (20, 65, 301, 20), (333, 1000, 3203, 3), (40, 1024, 2000, 20)])
def test_from_a_heads_rows_in_32_bits(T, H, V, top):
    from infer_b200 import ops
    x, w, t = _head(T, H, V, T + H, torch.float32)
    z = x.double() @ w.double().t()
    check(ops.head_logprobs(x, w, t, top), z, z, t, top)


def test_rows_that_do_not_keep_to_16_bytes():
    from infer_b200 import ops
    x, w, t = _head(40, 99, 700, 3)
    z = x.double() @ w.double().t()
    check(ops.head_logprobs(x, w, t, 5), z, z, t, 5)
    x, w, t = _head(40, 96, 700, 3)
    y = torch.empty(40 * 96 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(40, 96).copy_(x)
    z = x.double() @ w.double().t()
    check(ops.head_logprobs(y, w, t, 5), z, z, t, 5)


@pytest.mark.parametrize("T", [40, 300])
def test_head_with_equal_columns_and_rows_that_are_not_finite(T):
    """Equal rows of w are ties: the lowest id first. A row of x that is not finite makes its own results NaN and no one else's."""
    from infer_b200 import ops
    x, w, t = _head(T, 128, 3001, 9)
    w[1000:1300] = w[5]
    w[2000:3001] = 0
    x[3] = 0                                                        # every logit 0
    x[7, 5] = math.inf
    x[11, 0] = math.nan
    z = x.double() @ w.double().t()
    r = ops.head_logprobs(x, w, t, 20)
    odd = torch.zeros(T, dtype=torch.bool, device=DEV)
    odd[7] = odd[11] = True
    assert r.logprob[odd].isnan().all() and r.entropy[odd].isnan().all()
    ok = ~odd
    check(type(r)(*(v[ok] for v in r)), z[ok], z[ok], t[ok], 20)


@pytest.mark.parametrize("T,H,V", [(300, 1536, 9000), (64, 4096, 9000)])
def test_ordinary_rows(T, H, V):
    """Without exact sums: the tensor core's additions truncate, at most 2^-23 of the running sum of absolute products at each of H / 16 steps; for
    normal rows below 2^-23 H / 16 times the logit's own size in all (measured: 1e-5 of it at H = 8960)."""
    from infer_b200 import ops
    g = torch.Generator(device=DEV).manual_seed(H)
    x = torch.randn(T, H, device=DEV, generator=g).bfloat16()
    w = (torch.randn(V, H, device=DEV, generator=g) * (2.5 / math.sqrt(H))).bfloat16()
    t = torch.randint(0, V, (T,), device=DEV, generator=g, dtype=torch.int32)
    z = x.double() @ w.double().t()
    check(ops.head_logprobs(x, w, t, 0), z, z, t, 0, 2.0 ** -23 * H / 16 * z.abs().max().item())


def test_a_batchs_rows_do_not_depend_on_each_other():
    """A row's alternatives and tokens come out the same whatever rows are beside it; rows behind the last are not written."""
    from infer_b200 import ops
    x, w, t = _head(300, 256, 9001, 4)
    whole = ops.head_logprobs(x, w, t, 20)
    for lo, hi in ((0, 20), (100, 300), (280, 300)):
        part = ops.head_logprobs(x[lo:hi].contiguous(), w, t[lo:hi].contiguous(), 20)
        assert torch.equal(part.top_ids, whole.top_ids[lo:hi])
        assert (part.logprob - whole.logprob[lo:hi]).abs().max().item() <= 200 * STEP + 8 * STEP * whole.logprob.abs().max().item()
