"""Products with weights in 8-bit integers and expert layers of a few tokens, as cases that can be timed and compared.

Kinds: ``linear`` is ``ops.int8.int8_linear``: rows of activations are held in 8-bit integers with a scale each, multiplied by weights in 8-bit integers with
a scale for each output channel, with a bias or as a gated pair. ``moe`` is ``ops.moe.moe_ffn_few``: the whole mixture-of-experts layer, router to sum, of
up to 64 tokens, with experts in bf16 or in 8-bit integers. Sizes are those of the presets, the tests and the mixture's benchmark, and what lies between.

A row of activations x is held as c = x / s rounded to whole numbers, halves to even, s = max(|x|, 1e-10) / 127 in fp32. A weight row is held the same way.
The router's weights are the raw probabilities of its ``top_k`` largest entries."""
from __future__ import annotations

import math

import torch

own = False          # True: the framework's operators; False: the same in elementary operations

DEV, LEAST = "cuda", 1e-10


def listed():
    return [
        # the next token of a single user, the 7 B decoder's fused projection: latency
        dict(name="linear_1_qkv", kind="linear", dtype="bfloat16", rows=1, k=4096, n=6144, gated=False, bias=False),
        # sixteen sequences' next tokens through its gate and up projection
        dict(name="linear_16_gated", kind="linear", dtype="bfloat16", rows=16, k=4096, n=22016, gated=True, bias=False),
        # the headline's decode batch through its down projection
        dict(name="linear_64_down", kind="linear", dtype="bfloat16", rows=64, k=11008, n=4096, gated=False, bias=False),
        # an fp32 model of odd sizes with a bias, on packed tokens of a few prompts
        dict(name="linear_301_odd_fp32", kind="linear", dtype="float32", rows=301, k=1411, n=1001, gated=False, bias=True),
        # three prompts of 1001 tokens through the 64 M decoder's gate and up projection
        dict(name="linear_3003_64m", kind="linear", dtype="bfloat16", rows=3003, k=512, n=4096, gated=True, bias=False),
        # prompts of the 7 B decoder: its output projection, its gate and up projection
        dict(name="linear_2048_out", kind="linear", dtype="bfloat16", rows=2048, k=4096, n=4096, gated=False, bias=True),
        dict(name="linear_8192_gated", kind="linear", dtype="bfloat16", rows=8192, k=4096, n=22016, gated=True, bias=False),
        # one token through a small mixture, as a test or a draft model has it: latency
        dict(name="moe_1_small_int8", kind="moe", weights="int8", tokens=1, d=256, f=512, experts=8, top_k=2, shared=False, residual=True),
        # the next token of a single user through a layer of the 24-layer mixture
        dict(name="moe_1_24l", kind="moe", weights="bfloat16", tokens=1, d=2048, f=5632, experts=8, top_k=2, shared=False, residual=True),
        # many small experts and one for every token
        dict(name="moe_7_many", kind="moe", weights="bfloat16", tokens=7, d=1024, f=704, experts=64, top_k=6, shared=True, residual=True),
        # sixteen sequences through the 24-layer mixture, experts in 8 bits
        dict(name="moe_16_24l_int8", kind="moe", weights="int8", tokens=16, d=2048, f=5632, experts=8, top_k=2, shared=False, residual=True),
        # a full decode batch: every expert is met
        dict(name="moe_64_24l", kind="moe", weights="bfloat16", tokens=64, d=2048, f=5632, experts=8, top_k=2, shared=False, residual=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.55:
        k, n = _log(rng, 40, 11008), _log(rng, 24, 22016)
        if rng.random() < 0.6:                                   # trained sizes are mostly whole, some are not
            k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
        gated = rng.random() < 0.4
        rows = min(_log(rng, 1, 8192), 8192 * 4096 * 22016 // (n * k))
        return dict(kind="linear", dtype=rng.choice(("bfloat16", "bfloat16", "float32")), rows=rows, k=k, n=n + n % 2 if gated else n, gated=gated,
                    bias=rng.random() < 0.4)
    experts = rng.choice((2, 4, 8, 8, 16, 37, 64))
    d, f = 16 * _log(rng, 8, 256), 16 * _log(rng, 4, 352)
    f = max(16, min(f, 8 * 2048 * 5632 // (experts * d) // 16 * 16))
    return dict(kind="moe", weights=rng.choice(("bfloat16", "int8")), tokens=_log(rng, 1, 64), d=d, f=f, experts=experts,
                top_k=rng.randrange(1, min(8, experts) + 1), shared=rng.random() < 0.3, residual=rng.random() < 0.7)


# ---------------------------------------------------------------------------------------------- sizes
def work(c):
    if c["kind"] == "linear":
        size, out = 2 if c["dtype"] == "bfloat16" else 4, c["n"] // 2 if c["gated"] else c["n"]
        return {"bytes": c["rows"] * (c["k"] + out) * size + c["n"] * (c["k"] + 4 + (size if c["bias"] else 0)), "flops": 2 * c["rows"] * c["n"] * c["k"]}
    T, E, D, F, K = c["tokens"], c["experts"], c["d"], c["f"], c["top_k"]
    met = E * (1 - (1 - K / E) ** T) + c["shared"]               # experts that some token goes to, on average
    expert = 3 * F * D * (2 if c["weights"] == "bfloat16" else 1) + (4 * (2 * F + D) if c["weights"] == "int8" else 0)
    return {"bytes": int(met * expert) + 2 * E * D + (3 if c["residual"] else 2) * 2 * T * D, "flops": 6 * T * (K + c["shared"]) * F * D}


# ---------------------------------------------------------------------------------------------- inputs
def _rows(g, rows, n, dtype):
    """Activations behind a norm: channels of unequal size."""
    x = torch.randn(rows, n, device=DEV, generator=g)
    return (x * torch.exp(0.5 * torch.randn(n, device=DEV, generator=g))).to(dtype)


def _weight(g, shape, weights, pad=16):
    """bf16 weights, or codes [.., n, k], rows on 16-byte boundaries, with a scale for each row."""
    k = shape[-1]
    w = torch.randn(*shape, device=DEV, generator=g).mul_(torch.exp(0.3 * torch.randn(*shape[:-1], 1, device=DEV, generator=g))).mul_(k ** -0.5)
    if weights == "bfloat16":
        return w.to(torch.bfloat16)
    s = w.abs().amax(-1).clamp_min(LEAST).double().div(127).float()
    q = torch.zeros(*shape[:-1], -(-k // pad) * pad, dtype=torch.int8, device=DEV)
    q[..., :k] = w.div_(s.unsqueeze(-1)).round_().clamp_(-127, 127).to(torch.int8)
    return q[..., :k], s


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if c["kind"] == "linear":
        dt = getattr(torch, c["dtype"])
        s = dict(case=c, x=_rows(g, c["rows"], c["k"], dt), w=_weight(g, (c["n"], c["k"]), "int8"))
        s["bias"] = torch.randn(c["n"], device=DEV, generator=g).to(dt) if c["bias"] else None
        return s
    T, E, D, F = c["tokens"], c["experts"], c["d"], c["f"]
    s = dict(case=c, x=_rows(g, T, D, torch.bfloat16), router=(1.5 * D ** -0.5 * torch.randn(E, D, device=DEV, generator=g)).bfloat16())
    s["gate_up"], s["down"] = _weight(g, (E, 2 * F, D), c["weights"]), _weight(g, (E, D, F), c["weights"])
    s["shared"] = (_weight(g, (2 * F, D), c["weights"]), _weight(g, (D, F), c["weights"])) if c["shared"] else None
    s["residual"] = torch.randn(T, D, device=DEV, generator=g).bfloat16() if c["residual"] else None
    return s


# ---------------------------------------------------------------------------------------------- the operators in elementary operations
def _silu_pair(y):
    a, b = y.chunk(2, -1)
    return a / (1 + torch.exp(-a)) * b


def _linear_plain(s):
    c, (q, sw) = s["case"], s["w"]
    x = s["x"].float()
    sx = (x.abs().amax(-1, keepdim=True).clamp_min(LEAST).double() / 127).float()
    codes = torch.round(x.double() / sx.double()).float()                      # 64 bits: quotients next to a half
    y = torch.matmul(codes, q.float().t()) * sx * sw                           # whole sums stay far under 2^24
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return (_silu_pair(y) if c["gated"] else y).to(s["x"].dtype)


def _float(w):
    return w.float() if isinstance(w, torch.Tensor) else w[0].float() * w[1].unsqueeze(-1)


def _moe_plain(s):
    """Every expert on every token, weighted by what the router gives it, zero for most."""
    c, x = s["case"], s["x"].float()
    T, E = c["tokens"], c["experts"]
    logits = torch.matmul(x, s["router"].float().t())
    e = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    order = torch.sort(p, dim=-1, descending=True, stable=True).indices[:, : c["top_k"]]
    chosen = torch.zeros(T, E, device=DEV).scatter_(1, order, 1.0)
    act = _silu_pair(torch.matmul(x, _float(s["gate_up"]).transpose(1, 2)))                    # [E, T, F]
    y = (torch.matmul(act, _float(s["down"]).transpose(1, 2)) * (p * chosen).t().unsqueeze(-1)).sum(0)
    if c["shared"]:
        y = y + torch.matmul(_silu_pair(torch.matmul(x, _float(s["shared"][0]).t())), _float(s["shared"][1]).t())
    if c["residual"]:
        y = y + s["residual"].float()
    return y.to(torch.bfloat16), chosen.sum(0).int()


# ---------------------------------------------------------------------------------------------- one pass
def _own_weight(w):
    from innova_b200.ops import int8
    return w if isinstance(w, torch.Tensor) else int8.Int8Weight(*w)


def _moe_own(s):
    from innova_b200.ops.moe import moe_ffn_few
    shared = None if s["shared"] is None else tuple(_own_weight(w) for w in s["shared"])
    return moe_ffn_few(s["x"], s["router"], _own_weight(s["gate_up"]), _own_weight(s["down"]), s["residual"], s["case"]["top_k"], shared)


def _linear_own(s):
    from innova_b200.ops import int8
    return int8.int8_linear(s["x"], int8.Int8Weight(*s["w"]), s["bias"], gated=s["case"]["gated"])


def run(s):
    if s["case"]["kind"] == "linear":
        return {"y": _linear_own(s) if own else _linear_plain(s)}
    y, counts = _moe_own(s) if own else _moe_plain(s)
    return {"y": y, "counts": counts}


# ---------------------------------------------------------------------------------------------- in 64 bits, from the definitions
def _exact_gate(y):
    half = y.shape[-1] // 2
    return y[..., :half] * torch.sigmoid(y[..., :half]) * y[..., half:]


def _exact_linear(c, s):
    q, sw = s["w"]
    out = []
    for rows in s["x"].double().split(1024):
        top = torch.where(rows.abs().amax(1) < LEAST, LEAST, rows.abs().amax(1))
        scale = (top / 127).to(torch.float32).double().unsqueeze(1)
        y = (torch.round(rows / scale) @ q.double().mT) * scale * sw.double()
        if c["bias"]:
            y = y + s["bias"].double()
        out.append(_exact_gate(y) if c["gated"] else y)
    return {"y": torch.cat(out)}


def _exact_matrix(w, e=None):
    q, scale = (w, None) if isinstance(w, torch.Tensor) else w
    m = (q if e is None else q[e]).double()
    return m if scale is None else m * (scale if e is None else scale[e]).double()[:, None]


def _exact_moe(c, s):
    x = s["x"].double()
    logits = x @ s["router"].double().mT
    prob = torch.softmax(logits, 1)
    y = s["residual"].double() if c["residual"] else torch.zeros_like(x)
    taken = torch.zeros_like(prob, dtype=torch.bool)
    left = prob.clone()
    for _ in range(c["top_k"]):
        best = left.argmax(1, keepdim=True)
        taken.scatter_(1, best, True)
        left.scatter_(1, best, -1.0)
    for e in range(c["experts"]):
        rows = taken[:, e].nonzero().flatten()
        if len(rows):
            h = _exact_gate(x[rows] @ _exact_matrix(s["gate_up"], e).mT) @ _exact_matrix(s["down"], e).mT
            y = y.index_add(0, rows, h * prob[rows, e, None])
    if c["shared"]:
        y = y + _exact_gate(x @ _exact_matrix(s["shared"][0]).mT) @ _exact_matrix(s["shared"][1]).mT
    return {"y": y, "counts": taken.sum(0).int()}


def exact(c, seed):
    s = prepare(c, seed)
    return _exact_linear(c, s) if c["kind"] == "linear" else _exact_moe(c, s)
