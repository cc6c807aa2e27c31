"""Norms and rotation of query and key heads, and attention over a paged cache of 8-bit keys and values, as cases that can be timed and compared.

Kinds: ``norm`` is ``ops.qk_norm_rope``, forward alone or with its backward pass; ``append`` is ``paged_fp8.qkv_append``: the new tokens of several
sequences go from the fused projection into the pages, heads normed and rotated on the way; ``attend`` is ``paged_fp8.kv_attend``: attention of
those tokens over everything that the pages hold. Head counts are those of the presets and the tests, contexts run from the tests' lengths to long ones.

A page holds 16 tokens of one key head in float8_e4m3fn with one scale, the smallest power of two 2^e >= 2^-64 with |x| <= 448 * 2^e for all of
its tokens; where later tokens raise the scale, the earlier ones' codes are rounded again to the new one."""
from __future__ import annotations

import math
import random

import torch

own = False          # True: the framework's operators; False: the same in elementary operations

DEV, PAGE, EPS, TOP, FLOOR = "cuda", 16, 1e-6, 448.0, 2.0 ** -64


def listed():
    return [
        # a short prompt of the 64 M decoder on its way to attention: latency
        dict(name="norm_fwd_1x77", kind="norm", dtype="bfloat16", batch=1, seq=77, heads=8, kv_heads=8, dim=64, rot=64, grad=False),
        # a training step of the 64 M decoder at an odd batch and length
        dict(name="norm_grad_3x1001", kind="norm", dtype="bfloat16", batch=3, seq=1001, heads=8, kv_heads=8, dim=64, rot=64, grad=True),
        # a training step of the 7 B decoder's layers: grouped heads of 128
        dict(name="norm_grad_8x2048", kind="norm", dtype="bfloat16", batch=8, seq=2048, heads=32, kv_heads=8, dim=128, rot=128, grad=True),
        # the hybrid decoder's full-attention layers: fp32, one key head, a quarter of each head rotated
        dict(name="norm_grad_fp32_partial", kind="norm", dtype="float32", batch=2, seq=1999, heads=4, kv_heads=1, dim=64, rot=16, grad=True),
        # one decode step of the headline's batch: 64 sequences, one token each
        dict(name="append_64x1", kind="append", seqs=64, context=640, new=1, ragged=0, heads=32, kv_heads=8, dim=128, rot=128, norm=False),
        # five prompts of unequal length behind a shared conversation, normed heads
        dict(name="append_5_ragged", kind="append", seqs=5, context=1500, new=1201, ragged=7, heads=16, kv_heads=2, dim=128, rot=128, norm=True),
        # a long document's portion
        dict(name="append_2x8000", kind="append", seqs=2, context=333, new=8000, ragged=0, heads=32, kv_heads=8, dim=128, rot=128, norm=False),
        # a single user's next token: latency
        dict(name="attend_1x1_of_500", kind="attend", seqs=1, context=499, new=1, ragged=0, heads=8, kv_heads=8, dim=64, window=0),
        # the headline's decode step
        dict(name="attend_64x1_of_640", kind="attend", seqs=64, context=639, new=1, ragged=0, heads=32, kv_heads=8, dim=128, window=0),
        # long contexts of unequal length, one token each
        dict(name="attend_8x1_to_65000", kind="attend", seqs=8, context=65000, new=1, ragged=3, heads=32, kv_heads=8, dim=128, window=0),
        # verification of five drafted tokens, behind a sliding window
        dict(name="attend_12x5_window", kind="attend", seqs=12, context=4000, new=5, ragged=5, heads=16, kv_heads=4, dim=64, window=1024),
        # a portion of a long prompt over what came before it: products, not bytes
        dict(name="attend_2x1500_of_7000", kind="attend", seqs=2, context=5500, new=1500, ragged=0, heads=32, kv_heads=8, dim=128, window=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "append", "attend", "attend"))
    if kind == "norm":
        dim = rng.choice((32, 64, 80, 96, 128, 256))
        kv = rng.choice((1, 2, 3, 4, 8))
        heads = kv * rng.choice((1, 2, 4, 5, 8))
        seq = _log(rng, 1, 4000)
        dtype = rng.choice(("bfloat16", "bfloat16", "float32"))
        seq = min(seq, (8000 if dtype == "float32" else 16000) * 48 * 128 // ((heads + 2 * kv) * dim))
        batch = max(1, min(_log(rng, 1, 64), (8000 if dtype == "float32" else 16000) * 48 * 128 // (seq * (heads + 2 * kv) * dim)))
        return dict(kind=kind, dtype=dtype, batch=batch, seq=seq, heads=heads, kv_heads=kv, dim=dim,
                    rot=rng.choice((dim, 16, dim - dim // 2 // 16 * 16)), grad=rng.random() < 0.7)
    dim, kv = rng.choice((64, 128)), rng.choice((1, 2, 4, 8))
    case = dict(kind=kind, heads=kv * rng.choice((1, 2, 3, 4, 8)), kv_heads=kv, dim=dim, ragged=rng.randrange(1, 1000) if rng.random() < 0.7 else 0)
    if kind == "append":
        new = 1 if rng.random() < 0.4 else _log(rng, 2, 8000)
        seqs = max(1, min(_log(rng, 1, 200), 16000 // new))
        return dict(case, seqs=seqs, context=rng.choice((0, _log(rng, 1, 4000))), new=new, rot=rng.choice((0, 32, dim, dim)), norm=rng.random() < 0.5)
    new = rng.choice((1, 1, _log(rng, 2, 64), _log(rng, 2, 1500)))
    context = _log(rng, 1, 65000 if new == 1 else 5500)
    seqs = max(1, min(_log(rng, 1, 200), 300000 // (context + new), 3000 // new, 7 * 10 ** 10 // (new * (context + new) * case["heads"] * dim)))
    return dict(case, seqs=seqs, context=context, new=new, window=rng.choice((0, 0, 0, _log(rng, 1, 4000))))


# ---------------------------------------------------------------------------------------------- sizes
def _lengths(c):
    """Cached and new tokens of each sequence. Ragged: the first has the full lengths, the others shares of them down to an eighth, new tokens down to one."""
    n, r = c["seqs"], random.Random(c["ragged"])
    if not c["ragged"]:
        return [c["context"]] * n, [c["new"]] * n
    ctx = [c["context"]] + [int(c["context"] * 2.0 ** r.uniform(-3, 0)) for _ in range(n - 1)]
    new = [c["new"]] + [max(1, int(c["new"] * 2.0 ** r.uniform(-5, 0))) for _ in range(n - 1)]
    return ctx, new


def _visible(ctx, new, window):
    """Keys that the new tokens of one sequence see, over all of them."""
    if not window:
        return new * ctx + new * (new + 1) // 2
    return sum(min(window, ctx + i + 1) for i in range(new))


def work(c):
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "norm":
        rows, size = c["batch"] * c["seq"], 2 if c["dtype"] == "bfloat16" else 4
        whole, turned = rows * (H + 2 * G) * D * size, rows * (H + G) * D * size
        table = c["seq"] * c["rot"] * 4
        if not c["grad"]:
            return {"bytes": 2 * whole + table, "flops": 6 * rows * (H + G) * D}
        return {"bytes": 4 * whole + turned + 2 * table, "flops": 20 * rows * (H + G) * D}     # x, y; dy, x of the normed heads, dx
    ctx, new = _lengths(c)
    T = sum(new)
    if c["kind"] == "append":
        blocks = sum(-(-(a + b) // PAGE) - a // PAGE for a, b in zip(ctx, new)) * G
        return {"bytes": T * D * (2 * (H + 2 * G) + 2 * H + 2 * G) + T * c["rot"] * 4 + 8 * blocks, "flops": 8 * T * (H + G) * D}
    seen = sum(_visible(a, b, c["window"]) for a, b in zip(ctx, new))
    keys = sum(min(a + b, c["window"] + b - 1) if c["window"] else a + b for a, b in zip(ctx, new))
    return {"bytes": 2 * keys * G * D + keys // PAGE * G * 8 + 4 * T * H * D, "flops": 4 * seen * H * D}


# ---------------------------------------------------------------------------------------------- inputs
def _tables(n, rot):
    if not rot:
        return None, None
    inv = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64, device=DEV) * 2 / rot)
    a = torch.arange(n, dtype=torch.float64, device=DEV).unsqueeze(1) * inv
    return a.cos().float(), a.sin().float()


def _rows(g, rows, heads, dim, dtype):
    """Projection rows: channels of unequal size, as trained projections have them."""
    x = torch.randn(rows, heads * dim, device=DEV, generator=g)
    return (x * torch.exp(0.5 * torch.randn(heads * dim, device=DEV, generator=g))).to(dtype)


def _scale_of(amax):
    """The power of two of a block whose largest value is ``amax``."""
    m, e = torch.frexp(amax)                                   # amax = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.where(torch.isfinite(amax), torch.ldexp(torch.ones_like(amax), e.clamp(-64, 120)).clamp_min(FLOOR), torch.nan)


def _pool(g, pages, G, D):
    x = torch.randn(pages, G, PAGE, D, device=DEV, generator=g).mul_(torch.exp(0.5 * torch.randn(1, G, 1, D, device=DEV, generator=g)))
    s = _scale_of(x.abs().amax((2, 3)))
    return x.div_(s[..., None, None]).to(torch.float8_e4m3fn), s


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "norm":
        dt = getattr(torch, c["dtype"])
        s = dict(case=c, qkv=_rows(g, c["batch"] * c["seq"], H + 2 * G, D, dt).view(c["batch"], c["seq"], -1).requires_grad_(c["grad"]))
        for n in ("wq", "wk"):
            s[n] = (1 + 0.3 * torch.randn(D, device=DEV, generator=g)).to(dt).requires_grad_(c["grad"])
        s["cos"], s["sin"] = _tables(c["seq"], c["rot"])
        if c["grad"]:
            s["dy"] = torch.randn(c["batch"], c["seq"], (H + 2 * G) * D, device=DEV, generator=g).to(dt)
        return s
    ctx, new = _lengths(c)
    T, n = sum(new), c["seqs"]
    need = [-(-(a + b) // PAGE) for a, b in zip(ctx, new)]
    wide, pages = max(need), sum(need)
    order = torch.randperm(pages, device=DEV, generator=g).int()                     # pages as a long run leaves them: in no order
    at = torch.arange(wide, device=DEV).view(1, -1)
    has = at < torch.tensor(need, device=DEV).view(-1, 1)
    table = torch.zeros(n, wide, dtype=torch.int32, device=DEV)
    table[has] = order
    s = dict(case=c, page_table=table, rows=torch.arange(n, dtype=torch.int32, device=DEV), start=torch.tensor(ctx, dtype=torch.int32, device=DEV),
             cu=torch.tensor([sum(new[:i]) for i in range(n + 1)], dtype=torch.int32, device=DEV), tokens=T, max_new=max(new),
             max_len=max(a + b for a, b in zip(ctx, new)))
    s["k"], s["k_scale"] = _pool(g, pages, G, D)
    s["v"], s["v_scale"] = _pool(g, pages, G, D)
    if c["kind"] == "append":
        s["qkv"] = _rows(g, T, H + 2 * G, D, torch.bfloat16)
        s["cos"], s["sin"] = _tables(s["max_len"], c["rot"])
        for name in ("wq", "wk"):
            s[name] = (1 + 0.3 * torch.randn(D, device=DEV, generator=g)).bfloat16() if c["norm"] else None
    else:
        s["q"] = _rows(g, T, H, D, torch.bfloat16)
    return s


# ---------------------------------------------------------------------------------------------- the operators in elementary operations
def _norm_turn(x, w, cos, sin):
    """x [..., heads, D] fp32, w [D] or None, cos and sin [..., 1, rot / 2] or None."""
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    if cos is None:
        return x
    half = cos.shape[-1]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * half:]], -1)


def _norm_plain(s):
    c = s["case"]
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].float().view(c["batch"], c["seq"], H + 2 * G, D)
    cos, sin = s["cos"][: c["seq"]].unsqueeze(1), s["sin"][: c["seq"]].unsqueeze(1)
    q, k = _norm_turn(x[..., :H, :], s["wq"].float(), cos, sin), _norm_turn(x[..., H:H + G, :], s["wk"].float(), cos, sin)
    return torch.cat([q, k, x[..., H + G:, :]], 2).flatten(2).to(s["qkv"].dtype)


def _token_places(s):
    """Sequence and position of every new token."""
    seq = torch.repeat_interleave(torch.arange(s["case"]["seqs"], device=DEV), s["cu"].diff().long(), output_size=s["tokens"])
    return seq, s["start"].long()[seq] + torch.arange(s["tokens"], device=DEV) - s["cu"].long()[seq]


def _store_plain(x, codes, scale, page, slot, first, kept):
    """x [T, G, D] fp32 into slots of pages; ``first``: the page that each sequence continues, ``kept`` of whose slots hold earlier tokens."""
    amax = torch.zeros_like(scale).index_reduce_(0, page, x.abs().amax(-1), "amax")
    touched = torch.zeros(scale.shape[0], dtype=torch.bool, device=DEV).index_fill_(0, page, True)
    holds = torch.zeros(scale.shape[0], dtype=torch.int64, device=DEV).index_reduce_(0, first, kept, "amax")
    was = torch.where(holds.unsqueeze(1) > 0, scale, 0.0)
    fresh = torch.where(touched.unsqueeze(1), torch.maximum(was, _scale_of(amax)), scale)
    old = codes[first]
    moved = (old.float() * (scale / fresh)[first][..., None, None]).to(codes.dtype)
    keep = (torch.arange(PAGE, device=DEV).view(1, 1, -1, 1) < kept.view(-1, 1, 1, 1)) & (kept > 0).view(-1, 1, 1, 1)
    raw = codes.view(torch.uint8)
    raw[first] = torch.where(keep, moved.view(torch.uint8), old.view(torch.uint8))
    raw[page, :, slot] = (x / fresh[page].unsqueeze(-1)).to(codes.dtype).view(torch.uint8)
    scale.copy_(fresh)


def _append_plain(s):
    c = s["case"]
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    seq, pos = _token_places(s)
    x = s["qkv"].float().view(s["tokens"], H + 2 * G, D)
    cos, sin = (None, None) if s["cos"] is None else (s["cos"][pos].unsqueeze(1), s["sin"][pos].unsqueeze(1))
    wq, wk = (None, None) if s["wq"] is None else (s["wq"].float(), s["wk"].float())
    q, k = _norm_turn(x[:, :H], wq, cos, sin), _norm_turn(x[:, H:H + G], wk, cos, sin)
    table, start = s["page_table"].long(), s["start"].long()
    page, slot = table[s["rows"].long()[seq], pos // PAGE], pos % PAGE
    first = table[s["rows"].long(), start // PAGE]
    _store_plain(k, s["k"], s["k_scale"], page, slot, first, start % PAGE)
    _store_plain(x[:, H + G:], s["v"], s["v_scale"], page, slot, first, start % PAGE)
    return q.flatten(1).to(torch.bfloat16)


def _attend_plain(s):
    c = s["case"]
    H, G, D, n = c["heads"], c["kv_heads"], c["dim"], c["seqs"]
    seq, pos = _token_places(s)
    table = s["page_table"].long()[s["rows"].long()]
    k, v = ((s[p][table].float() * s[p + "_scale"][table][..., None, None]).permute(0, 2, 1, 3, 4).reshape(n, G, -1, D) for p in ("k", "v"))
    q = torch.zeros(n, s["max_new"], H, D, device=DEV)                               # padded to the longest sequence
    at = torch.arange(s["tokens"], device=DEV) - s["cu"].long()[seq]
    q[seq, at] = s["q"].float().view(-1, H, D) * D ** -0.5
    where = torch.zeros(n, s["max_new"], dtype=torch.int64, device=DEV)
    where[seq, at] = pos
    j, p = torch.arange(k.shape[2], device=DEV), where.view(n, 1, 1, -1, 1)
    seen = j <= p
    if c["window"]:
        seen = seen & (j > p - c["window"])
    score = torch.matmul(q.view(n, -1, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(n, G, -1, D), k.transpose(2, 3))
    score = score.view(n, G, H // G, s["max_new"], -1).masked_fill_(~seen, -torch.inf)
    e = score.sub_(score.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(e.view(n, G, -1, e.shape[-1]), v).view(n, G, H // G, -1, D) / e.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(n, -1, H * D)[seq, at].to(torch.bfloat16)


# ---------------------------------------------------------------------------------------------- one pass
def _norm_own(s):
    from innova_b200 import ops
    c = s["case"]
    return ops.qk_norm_rope(s["qkv"], s["wq"], s["wk"], s["cos"], s["sin"], c["heads"], c["kv_heads"], c["dim"], eps=EPS)


def _paged_own(s):
    from innova_b200.ops import paged_fp8
    c = s["case"]
    pages = paged_fp8.Fp8Pages(s["k"], s["v"], s["k_scale"], s["v_scale"])
    new = paged_fp8.NewTokens(s["rows"], s["cu"], s["start"], s["max_new"], s["max_len"])
    if c["kind"] == "append":
        return paged_fp8.qkv_append(s["qkv"], c["heads"], c["kv_heads"], c["dim"], pages, s["page_table"], new, s["cos"], s["sin"],
                                    q_weight=s["wq"], k_weight=s["wk"], eps=EPS)
    return paged_fp8.kv_attend(s["q"], pages, s["page_table"], new, c["heads"], c["dim"] ** -0.5, window=c["window"])


def run(s):
    c = s["case"]
    if c["kind"] == "norm":
        y = _norm_own(s) if own else _norm_plain(s)
        if not c["grad"]:
            return {"y": y}
        dqkv, dwq, dwk = torch.autograd.grad(y, (s["qkv"], s["wq"], s["wk"]), s["dy"])
        return {"y": y, "dqkv": dqkv, "dwq": dwq, "dwk": dwk}
    if c["kind"] == "append":
        q = _paged_own(s) if own else _append_plain(s)
        return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    return {"out": _paged_own(s) if own else _attend_plain(s)}


# ---------------------------------------------------------------------------------------------- in 64 bits, from the definitions
def _exact_heads(x, w, pos, cos, sin):
    """Heads x [T, heads, D]; pair (i, i + rot / 2) of a token at p is turned by the table's angle of (p, i)."""
    if w is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.double()
    if cos is None:
        return x
    h, out = cos.shape[1], x.clone()
    turn = torch.complex(cos.double(), sin.double())[pos].unsqueeze(1)
    z = torch.complex(x[..., :h], x[..., h:2 * h]) * turn
    out[..., :h], out[..., h:2 * h] = z.real, z.imag
    return out


def _exact_norm(c, s):
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    T = c["batch"] * c["seq"]
    pos = torch.arange(c["seq"], device=DEV).repeat(c["batch"])
    x = s["qkv"].detach().double().view(T, H + 2 * G, D)
    q, k = _exact_heads(x[:, :H], s["wq"].detach(), pos, s["cos"], s["sin"]), _exact_heads(x[:, H:H + G], s["wk"].detach(), pos, s["cos"], s["sin"])
    y = torch.cat([q, k, x[:, H + G:]], 1).view(c["batch"], c["seq"], -1)
    if not c["grad"]:
        return {"y": y}
    dy, grads = s["dy"].double().view(T, H + 2 * G, D), []
    dx = dy.clone()
    for lo, hi, w in ((0, H, s["wq"]), (H, H + G, s["wk"])):
        back = _exact_heads(dy[:, lo:hi], None, pos, s["cos"], -s["sin"])             # the transpose turns the other way
        part = x[:, lo:hi]
        r = 1 / torch.sqrt((part * part).sum(-1, keepdim=True) / D + EPS)
        grads.append((back * part * r).sum((0, 1)))
        gw = back * w.detach().double()
        dx[:, lo:hi] = gw * r - part * r ** 3 * (gw * part).sum(-1, keepdim=True) / D
    return {"y": y, "dqkv": dx.view(c["batch"], c["seq"], -1), "dwq": grads[0], "dwk": grads[1]}


def _exact_round(x):
    """To e4m3: three bits behind the leading one down to 2^-6, steps of 2^-9 below; halves to the even step."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_append(c, s):
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    ctx, new = _lengths(c)
    pos = torch.cat([torch.arange(a, a + b, device=DEV) for a, b in zip(ctx, new)])
    x = s["qkv"].double().view(-1, H + 2 * G, D)
    q, k = _exact_heads(x[:, :H], s["wq"], pos, s["cos"], s["sin"]), _exact_heads(x[:, H:H + G], s["wk"], pos, s["cos"], s["sin"])
    out = {"q": q.flatten(1)}
    table = s["page_table"].tolist()
    for name, src in (("k", k), ("v", x[:, H + G:])):
        codes, scale = s[name].double(), s[name + "_scale"].double()
        at = 0
        for i, (a, b) in enumerate(zip(ctx, new)):
            done = 0
            while done < b:
                page, slot = table[i][(a + done) // PAGE], (a + done) % PAGE
                m = min(PAGE - slot, b - done)
                part = src[at + done:at + done + m].transpose(0, 1)                     # [G, m, D]
                amax = part.abs().amax((1, 2))
                e = torch.exp2(torch.round(torch.log2(amax.clamp_min(1e-30) / TOP)))
                e = torch.where(amax > TOP * e, 2 * e, torch.where(amax <= TOP / 2 * e, e / 2, e)).clamp_min(FLOOR)
                if slot:
                    e = torch.maximum(e, scale[page])
                    codes[page, :, :slot] = _exact_round(codes[page, :, :slot] * (scale[page] / e)[:, None, None])
                codes[page, :, slot:slot + m] = _exact_round(part / e[:, None, None])
                scale[page] = e
                done += m
            at += b
        out[name], out[name + "_scale"] = codes, scale
    return out


def _exact_attend(c, s):
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    ctx, new = _lengths(c)
    if sum(_visible(a, b, c["window"]) for a, b in zip(ctx, new)) * H * D > 3e11:
        return None
    outs, at = [], 0
    for i, (a, b) in enumerate(zip(ctx, new)):
        pages = s["page_table"][i, : -(-(a + b) // PAGE)].long()
        kv = [(s[p][pages].double() * s[p + "_scale"][pages].double()[..., None, None]).transpose(1, 2).reshape(-1, G, D)[: a + b] for p in ("k", "v")]
        for t in range(0, b, 256):
            rows = s["q"][at + t:at + min(t + 256, b)].double().view(-1, G, H // G, D)
            score = torch.einsum("tghd,jgd->ghtj", rows, kv[0]) / math.sqrt(D)
            p, j = torch.arange(a + t, a + t + rows.shape[0], device=DEV).view(-1, 1), torch.arange(a + b, device=DEV)
            hidden = (j > p) | (j <= p - c["window"]) if c["window"] else j > p
            outs.append(torch.einsum("ghtj,jgd->tghd", torch.softmax(score.masked_fill(hidden, -math.inf), -1), kv[1]).reshape(-1, H * D))
        at += b
    return {"out": torch.cat(outs)}


def exact(c, seed):
    s = prepare(c, seed)
    return {"norm": _exact_norm, "append": _exact_append, "attend": _exact_attend}[c["kind"]](c, s)
