"""Operators that finish a matrix product, or take up its result, where a model's answers are scored.

``token_logprobs``: from float32 logits (one row a place) the log probability of a given token, the row's entropy and the likeliest
tokens with theirs.  ``head_logprobs``: the same from the rows in front of the head and the head's matrix, without logits in memory.
``linear_act``: a matrix product with bias, activation and residual, rounded once.

With l a row of logits, m its maximum, S = sum exp(l - m) and D = sum exp(l - m) (l - m): logprob(t) = l[t] - m - ln S and
entropy = ln S - D / S.  A logit of -inf has no probability and adds nothing; where every logit of a row is -inf the log probability is
-inf and the entropy 0.  Alternatives come by falling logit, among equal ones the lowest id first; places without one hold id -1
and -inf.  A token of -1 asks for nothing: its log probability is 0.  The head's logits are scale * x . w, or with a cap
cap * tanh(scale * x . w / cap); its alternatives go by x . w, which has the same order.

In the head's cases the rows' elements are multiples of 1/16 and the matrix's of 2^-11 (seven bits of a bfloat16's eight): each sum of
products is then a float32 number, whatever the order of the additions, and the order of the alternatives is the same for everyone.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
ACTIVATIONS = ("none", "relu", "relu_squared", "gelu_tanh", "gelu", "silu")


def _logits(name, rows, vocab, top, masked=0.0):
    c = dict(op="logits", rows=rows, vocab=vocab, top=top, masked=masked)
    return dict(c, name=name) if name else c


def _head(name, rows, hidden, vocab, top, dtype="bfloat16", scale=1.0, cap=0.0):
    c = dict(op="head", rows=rows, hidden=hidden, vocab=vocab, top=top, dtype=dtype, scale=scale, cap=cap)
    return dict(c, name=name) if name else c


def _act(name, rows, n, k, act, bias, residual, dtype="bfloat16", out="bfloat16"):
    c = dict(op="act", rows=rows, n=n, k=k, act=act, bias=bias, residual=residual, dtype=dtype, out=out)
    return dict(c, name=name) if name else c


def listed():
    return [
        # One request decodes and its user asked for five alternatives of each token: latency counts.
        _logits("logprobs-1", 1, 151936, 5),
        # A full server: every request asked for as many alternatives as there are.
        _logits("logprobs-64", 64, 151936, 20),
        # Decoding under a grammar: most tokens are masked, some rows have none left; an odd vocabulary.
        _logits("logprobs-masked-37", 37, 50257, 8, 0.9),
        # A prompt's logits that are in memory already: log probabilities and entropies only.
        _logits("logprobs-1024", 1024, 152064, 0),
        # Eight requests decode, from the head's rows: the matrix is what is read.
        _head("head-8", 8, 1536, 151936, 5),
        # The ends of many short prompts scored together, a larger model with capped logits.
        _head("head-77", 77, 3584, 152064, 20, cap=30.0),
        # A prompt of the benchmark's length scored, with the likeliest five at each place: the largest case.
        _head("head-2048", 2048, 1536, 151936, 5),
        # The 32-bit path, odd sizes.
        _head("head-f32-333", 333, 1000, 32003, 3, "float32", scale=0.5),
        # A feed-forward's first product for eight decoding requests.
        _act("act-8", 8, 8960, 1536, "gelu_tanh", True, False),
        # The same for a prompt of 2,048 tokens of a larger model.
        _act("act-2048", 2048, 18944, 3584, "relu_squared", False, False),
        # A feed-forward's last product into the residual stream, a portion of a prompt of odd length.
        _act("act-500", 500, 1536, 8960, "none", True, True, out="float32"),
        # The 32-bit path, odd sizes.
        _act("act-f32-301", 301, 2301, 1000, "silu", True, False, "float32", "float32"),
    ]


def _between(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    """One more case of the same ranges: every operator as often, sizes over their logarithm, odd ones among them. (The bfloat16
    products' K are multiples of 8: rows on 16 bytes, as the framework's other products on the tensor cores want them.)"""
    kind = rng.choice(("logits", "head", "head", "act", "act"))
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    if kind == "logits":
        vocab = _between(rng, 300, 260000)
        return _logits(None, _between(rng, 1, min(2048, 160_000_000 // vocab)), vocab, rng.choice((0, rng.randint(1, 20))), rng.choice((0.0, 0.0, 0.5, 0.99)))
    if kind == "head":
        vocab = _between(rng, 300, 152064)
        hidden = 8 * _between(rng, 8, 640) if dtype == "bfloat16" else _between(rng, 64, 1600)
        most = 300_000_000_000 // (vocab * hidden) if dtype == "bfloat16" else 12_000_000_000 // (vocab * hidden)
        cap = rng.choice((0.0, 0.0, float(rng.randint(10, 60))))
        return _head(None, _between(rng, 1, max(1, min(2048, most))), hidden, vocab, rng.choice((0, rng.randint(1, 20))), dtype,
                     rng.choice((1.0, 1.0, round(rng.uniform(0.1, 2.0), 3))), cap)
    k = 8 * _between(rng, 8, 2368) if dtype == "bfloat16" else _between(rng, 64, 2400)
    n = _between(rng, 33, 18944)
    most = 140_000_000_000 // (n * k) if dtype == "bfloat16" else 6_000_000_000 // (n * k)
    residual = rng.random() < 0.3
    out = "float32" if residual or dtype == "float32" else rng.choice(("bfloat16", "bfloat16", "float32"))
    return _act(None, _between(rng, 1, max(1, min(4096, most))), n, k, rng.choice(ACTIVATIONS), rng.random() < 0.5, residual, dtype, out)


def _tokens(g, rows, vocab):
    """The tokens that are asked for; the last row of several has none, as the end of a prompt."""
    t = torch.randint(0, vocab, (rows,), generator=g, device=DEVICE, dtype=torch.int32)
    if rows > 1:
        t[-1] = -1
    return t


def _grid(g, shape, std, step, most, dtype):
    """Normal numbers on multiples of ``step``, at most ``most`` steps from zero."""
    return (torch.randn(shape, generator=g, device=DEVICE) * (std / step)).round_().clamp_(-most, most).mul_(step).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    if case["op"] == "logits":
        B, V = case["rows"], case["vocab"]
        logits = torch.randn((B, V), generator=g, device=DEVICE) * 2.5
        # a model is surer at some places than at others: up to 12 on top of a token
        logits[torch.arange(B, device=DEVICE), torch.randint(0, V, (B,), generator=g, device=DEVICE)] += 12 * torch.rand(B, generator=g, device=DEVICE)
        if case["masked"]:
            logits.masked_fill_(torch.rand((B, V), generator=g, device=DEVICE) < case["masked"], -math.inf)
            logits[B // 2, 1:] = -math.inf          # one token left
            if B > 2:
                logits[B // 3] = -math.inf          # none left
        return dict(case=case, logits=logits, tokens=_tokens(g, B, V))
    if case["op"] == "head":
        T, H, V, dt = case["rows"], case["hidden"], case["vocab"], DTYPES[case["dtype"]]
        x = _grid(g, (T, H), 1.0, 2.0 ** -4, 64, dt)
        w = _grid(g, (V, H), min(2.5 / math.sqrt(H), 0.06), 2.0 ** -11, 255, dt)
        return dict(case=case, x=x, w=w, tokens=_tokens(g, T, V))
    M, N, K, dt = case["rows"], case["n"], case["k"], DTYPES[case["dtype"]]
    x = torch.randn((M, K), generator=g, device=DEVICE).to(dt)
    w = (torch.randn((N, K), generator=g, device=DEVICE) / math.sqrt(K)).to(dt)
    bias = 0.3 * torch.randn(N, generator=g, device=DEVICE) if case["bias"] else None
    residual = torch.randn((M, N), generator=g, device=DEVICE) if case["residual"] else None
    return dict(case=case, x=x, w=w, bias=bias, residual=residual)


def _statistics(l, tokens):
    """(log probability of the tokens, entropy) of rows of float32 logits."""
    m = l.amax(1, keepdim=True)
    empty = m == -math.inf
    d = l - torch.where(empty, torch.zeros_like(m), m)
    e = torch.exp(d)
    S = e.sum(1)
    D = torch.where(e > 0, e * d, torch.zeros_like(d)).sum(1)
    at = d.gather(1, tokens.long().clamp_min(0)[:, None])[:, 0]
    none = empty[:, 0]
    logprob = torch.where(none, torch.full_like(S, -math.inf), at - torch.log(S))
    entropy = torch.where(none, torch.zeros_like(S), torch.log(S) - D / S)
    return torch.where(tokens < 0, torch.zeros_like(S), logprob), entropy, m[:, 0], S


def _alternatives(z, top):
    """The ids of the ``top`` largest of each row, among equal ones the lowest id first, -1 where only -inf is left."""
    if top == 0:
        return torch.empty((z.shape[0], 0), dtype=torch.int64, device=z.device)
    bits = (z + 0.0).view(torch.int32)                                  # (-0 is 0)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32) + ((1 << 32) - 1 - torch.arange(z.shape[1], device=z.device))
    ids = ((1 << 32) - 1 - (torch.topk(key, min(top, z.shape[1]), dim=1).values & 0xFFFFFFFF))
    ids = torch.where(z.gather(1, ids) == -math.inf, torch.full_like(ids, -1), ids)
    return torch.nn.functional.pad(ids, (0, top - ids.shape[1]), value=-1)


def _with_top(l, z, tokens, top):
    logprob, entropy, m, S = _statistics(l, tokens)
    ids = _alternatives(z, top)
    at = l.gather(1, ids.clamp_min(0)) - m[:, None] - torch.log(S)[:, None]
    return logprob, entropy, ids.to(torch.int32), torch.where(ids < 0, torch.full_like(at, -math.inf), at)


def _activate(z, act):
    if act == "relu":
        return torch.clamp_min(z, 0)
    if act == "relu_squared":
        return torch.clamp_min(z, 0) ** 2
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def run(state):
    c = state["case"]
    if own:
        from infer_b200 import ops
        if c["op"] == "logits":
            return tuple(ops.token_logprobs(state["logits"], state["tokens"], c["top"]))
        if c["op"] == "head":
            return tuple(ops.head_logprobs(state["x"], state["w"], state["tokens"], c["top"], scale=c["scale"], softcap=c["cap"]))
        return ops.linear_act(state["x"], state["w"], state["bias"], c["act"], state["residual"], DTYPES[c["out"]])
    if c["op"] == "logits":
        return _with_top(state["logits"], state["logits"], state["tokens"], c["top"])
    z = state["x"].float() @ state["w"].float().T
    if c["op"] == "head":
        l = z * c["scale"]
        if c["cap"]:
            l = c["cap"] * torch.tanh(l / c["cap"])
        return _with_top(l, z, state["tokens"], c["top"])
    if state["bias"] is not None:
        z = z + state["bias"]
    z = _activate(z, c["act"])
    if state["residual"] is not None:
        z = z + state["residual"]
    return z.to(DTYPES[c["out"]])


def work(case):
    if case["op"] == "logits":
        B, V, top = case["rows"], case["vocab"], case["top"]
        return {"bytes": 4 * B * V + 12 * B + 8 * B * top, "flops": 5 * B * V}
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "head":
        T, H, V, top = case["rows"], case["hidden"], case["vocab"], case["top"]
        return {"bytes": size * H * (T + V) + 12 * T + 8 * T * top, "flops": 2 * T * H * V}
    M, N, K = case["rows"], case["n"], case["k"]
    return {"bytes": size * K * (M + N) + (4 * N if case["bias"] else 0) + (4 * M * N if case["residual"] else 0) + M * N * (2 if case["out"] == "bfloat16" else 4),
            "flops": 2 * M * N * K}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "act":
        z = torch.matmul(s["x"].double(), s["w"].double().t())
        if s["bias"] is not None:
            z += s["bias"].double()
        act = case["act"]
        if act == "relu":
            z = z.clamp(min=0)
        elif act == "relu_squared":
            z = z.clamp(min=0).square()
        elif act == "gelu_tanh":
            z = z * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z))
        elif act == "gelu":
            z = z * 0.5 * torch.special.erfc(-z / 2 ** 0.5)
        elif act == "silu":
            z = z * torch.sigmoid(z)
        return z if s["residual"] is None else z + s["residual"].double()
    parts = []
    rows = case["rows"]
    w = s["w"].double() if case["op"] == "head" else None
    step = max(1, 64_000_000 // case["vocab"])
    for lo in range(0, rows, step):
        hi = min(rows, lo + step)
        if w is None:
            z = l = s["logits"][lo:hi].double()
        else:
            z = s["x"][lo:hi].double() @ w.t()
            l = z * case["scale"]
            if case["cap"]:
                l = case["cap"] * torch.tanh(l / case["cap"])
        lse = torch.logsumexp(l, 1, keepdim=True)
        empty = lse == -math.inf
        lp = torch.where(empty, torch.full_like(l, -math.inf), l - lse)
        p = lp.exp()
        entropy = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
        t = s["tokens"][lo:hi].long()
        logprob = torch.where(t < 0, torch.zeros_like(entropy), lp.gather(1, t.clamp(min=0)[:, None])[:, 0])
        keep = min(case["top"], case["vocab"])
        ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :keep]
        best = lp.gather(1, ids)
        ids = torch.where(z.gather(1, ids) == -math.inf, torch.full_like(ids, -1), ids)
        if keep < case["top"]:
            ids = torch.nn.functional.pad(ids, (0, case["top"] - keep), value=-1)
            best = torch.nn.functional.pad(best, (0, case["top"] - keep), value=-math.inf)
        parts.append((logprob, entropy, ids.to(torch.int32), best))
    return tuple(torch.cat([p[i] for p in parts]) for i in range(4))
