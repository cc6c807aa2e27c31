"""The expert layer of a few tokens (ops.moe.moe_ffn_few) against its formula in 64 bits.

Tolerances. A product of K terms is summed sixteen terms an instruction, and parts of sixteen steps and more one after the other; a step of a chain is off by at most
2^-23 of the sum of the terms' sizes: (K / 16 + K / 1024 + 16) 2^-23 |a| |b|. A router's logit is a chain of K / 256 + 21 (eight terms of every 2048, five steps
among lanes, eight among warps). silu' is at most 1.1 and exp and the quotient are off
by under 2^-20. The activations between the products are rounded to bf16, half a step 2^-8 of each. Those errors go through the second product by |w|, are
weighted by the router's probabilities, which are off by twice the logits' error and 2^-20, and the result is rounded to bf16, 2^-8. On the CPU nothing is rounded
between the products and chains are as long as K."""
import pytest
import torch

from innova_b200.ops import runtime as rt
from innova_b200.ops.int8 import Int8Weight
from innova_b200.ops.moe import moe_few_supported, moe_ffn, moe_ffn_few

gpu = pytest.mark.gpu
BF = torch.bfloat16


def inputs(T, D, F, E, i8=False, shared=False, residual=True, seed=0, dtype=BF):
    g = torch.Generator().manual_seed(seed)

    def weight(*shape):
        w = torch.randn(*shape, generator=g) * shape[-1] ** -0.5
        return Int8Weight.quantize(w) if i8 else w.to(dtype)
    x = (torch.randn(T, D, generator=g) * torch.exp(0.5 * torch.randn(D, generator=g))).to(dtype)
    router = (1.5 * D ** -0.5 * torch.randn(E, D, generator=g)).to(dtype)
    a = dict(x=x, router_w=router, w_gate_up=weight(E, 2 * F, D), w_down=weight(E, D, F),
             residual=torch.randn(T, D, generator=g).to(dtype) if residual else None)
    a["shared"] = (weight(2 * F, D), weight(D, F)) if shared else None
    return a


def to(v, dev):
    if isinstance(v, Int8Weight):
        return Int8Weight(*(to(t, dev) for t in v))
    if isinstance(v, tuple):
        return tuple(to(t, dev) for t in v)
    if isinstance(v, dict):
        return {k: to(t, dev) for k, t in v.items()}
    return v.to(dev) if isinstance(v, torch.Tensor) else v


def real(w):
    return w.q.double() * w.scale.double().unsqueeze(-1) if isinstance(w, Int8Weight) else w.double()


def expert(x, gate_up, down, chain, half):
    """One expert on rows x in 64 bits, and how far it may be off."""
    steps = lambda k: chain(k) * 2.0 ** -23  # noqa: E731
    y, size = x @ gate_up.t(), x.abs() @ gate_up.abs().t() * steps(x.shape[1])
    (g, u), (eg, eu) = y.chunk(2, -1), size.chunk(2, -1)
    silu = g * torch.sigmoid(g)
    act = silu * u
    err = (1.1 * eg + 2.0 ** -20 * (1 + g.abs()) * silu.abs()) * u.abs() + silu.abs() * eu + half * act.abs()
    return act @ down.t(), err @ down.abs().t() + act.abs() @ down.abs().t() * steps(act.shape[1])


def check(a, top_k, dev, chosen=None):
    """Runs the call on ``dev`` and compares; ``chosen`` [T, top_k]: the experts, where probabilities do not tell them apart."""
    y, counts = moe_ffn_few(**to(a, dev), top_k=top_k)
    assert y.shape == a["x"].shape and y.dtype == a["x"].dtype and counts.dtype == torch.int32
    if dev == "cuda":
        rt.check_status()
    x = a["x"].reshape(-1, a["x"].shape[-1]).double()
    cpu = dev == "cpu"
    chain = (lambda k: k + 16) if cpu else (lambda k: k / 16 + k / 1024 + 16)
    half = 0.0 if cpu else 2.0 ** -8
    logits = x @ a["router_w"].double().t()
    el = (x.abs() @ a["router_w"].double().abs().t()).amax(-1, keepdim=True) * (x.shape[1] + 6 if cpu else x.shape[1] / 256 + 21) * 2.0 ** -24
    p = torch.softmax(logits, -1)
    if chosen is None:
        top, idx = p.topk(min(top_k + 1, p.shape[1]), -1)
        if top.shape[1] > top_k:     # the inputs tell the last that is taken from the first that is not, beyond the logits' error
            apart = logits.gather(1, idx[:, top_k - 1:top_k]) - logits.gather(1, idx[:, top_k:top_k + 1])
            assert bool((apart > 2 * el).all()), "inputs of this test"
        chosen = idx[:, :top_k]
    want, err = torch.zeros_like(x), torch.zeros_like(x)
    if a["residual"] is not None:
        want = want + a["residual"].reshape(x.shape).double()
    if a["shared"] is not None:
        y1, e1 = expert(x, real(a["shared"][0]), real(a["shared"][1]), chain, half)
        want, err = want + y1, err + e1
    for e in chosen.unique().tolist():
        rows = (chosen == e).any(-1).nonzero().flatten()
        y1, e1 = expert(x[rows], real(a["w_gate_up"])[e], real(a["w_down"])[e], chain, half)
        q = p[rows, e].unsqueeze(-1)
        want = want.index_add(0, rows, q * y1)
        err = err.index_add(0, rows, q * (e1 + y1.abs() * (2 * el[rows] + 2.0 ** -20)))
    off = (y.cpu().reshape(x.shape).double() - want).abs()
    tol = err * 1.01 + (2.0 ** -8 if y.dtype == BF else 2.0 ** -22) * (want.abs() + err) + 1e-30
    assert torch.isfinite(y).all() and bool((off <= tol).all()), float((off / tol).max())
    assert torch.equal(counts.cpu(), torch.bincount(chosen.reshape(-1), minlength=p.shape[1]).int())
    return y


CASES = [   # T, D, F, E, top_k, 8 bits, shared
    (1, 64, 32, 4, 2, False, False), (1, 256, 512, 8, 2, True, False), (2, 16, 16, 2, 1, True, True), (3, 8, 8, 3, 3, False, True),
    (7, 128, 88, 64, 6, False, True), (8, 208, 144, 8, 2, True, False), (9, 200, 72, 5, 2, False, False), (16, 512, 176, 16, 4, True, True),
    (17, 136, 264, 8, 8, False, False), (31, 64, 64, 200, 16, False, False), (33, 96, 160, 37, 3, True, False), (64, 256, 320, 8, 2, False, True),
    (64, 128, 48, 2, 1, True, False), (64, 64, 16, 1, 1, False, False), (40, 1032, 40, 6, 2, False, False)]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
def test_against_the_formula(case, dev):
    T, D, F, E, k, i8, shared = case
    check(inputs(T, D, F, E, i8, shared, T % 2 == 1, seed=1), k, dev)


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("T", [1, 12, 30, 64])
@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=gpu)])
def test_every_token_to_one_expert_and_ties(T, i8, dev):
    """Experts 3 and 5 lead by far and alike, the rest is alike: the lowest ones are taken."""
    a = inputs(T, 64, 48, 7, i8)
    a["x"] = a["x"].abs() + 0.5
    a["router_w"] = torch.zeros(7, 64, dtype=BF)
    a["router_w"][[3, 5]] = 0.125
    check(a, 1, dev, torch.full((T, 1), 3))
    check(a, 4, dev, torch.tensor([[3, 5, 0, 1]]).expand(T, 4))


def test_fp32_and_leading_dimensions():
    a = inputs(6, 40, 24, 5, dtype=torch.float32)
    y = check(a, 2, "cpu")
    b = dict(a, x=a["x"].view(2, 3, 40), residual=a["residual"].view(2, 3, 40))
    assert torch.equal(moe_ffn_few(**b, top_k=2)[0], y.view(2, 3, 40))


def test_refusals():
    a = inputs(4, 32, 16, 4)
    bad = lambda **kw: moe_ffn_few(**dict(a, **kw))  # noqa: E731
    with pytest.raises(TypeError, match="bf16"):
        bad(x=a["x"].half())
    with pytest.raises(ValueError, match="router"):
        bad(router_w=a["router_w"][:, :16])
    with pytest.raises(ValueError, match="w_gate_up"):
        bad(w_gate_up=a["w_gate_up"].float())
    with pytest.raises(ValueError, match="is needed"):
        bad(w_down=a["w_down"][:3])
    with pytest.raises(ValueError, match="8 bits or none"):
        bad(w_down=Int8Weight.quantize(a["w_down"]))
    with pytest.raises(ValueError, match="top_k"):
        bad(top_k=5)
    with pytest.raises(ValueError, match="top_k"):
        bad(top_k=0)
    with pytest.raises(ValueError, match="residual"):
        bad(residual=a["residual"][:3])
    with pytest.raises(ValueError, match="at most 64"):
        moe_ffn_few(**inputs(65, 32, 16, 4))
    with pytest.raises(ValueError, match="8 bits or none|2"):
        bad(shared=(a["w_gate_up"][0],))
    with pytest.raises(RuntimeError, match="no gradient"):
        bad(x=a["x"].clone().requires_grad_())
    with torch.no_grad():
        bad(x=a["x"].clone().requires_grad_())
    y, counts = bad(x=a["x"][:0], residual=None)
    assert y.shape == (0, 32) and not counts.any()


def test_supported():
    a = inputs(4, 32, 16, 4)
    args = (a["router_w"], a["w_gate_up"], a["w_down"])
    assert moe_few_supported(a["x"], *args) and not moe_few_supported(a["x"].repeat(17, 1), *args)


# ---------------------------------------------------------------------------------------------- on a GPU
@gpu
def test_refusals_gpu():
    a = to(inputs(4, 40, 24, 4), "cuda")
    moe_ffn_few(**a)
    b = to(inputs(4, 40, 24, 4, True), "cuda")
    with pytest.raises(ValueError, match="multiples of 16|one behind the other|16-byte"):
        moe_ffn_few(**b)
    c = to(inputs(4, 36, 24, 4), "cuda")
    with pytest.raises(ValueError, match="multiples of 8|16-byte"):
        moe_ffn_few(**c)
    with pytest.raises(TypeError, match="bf16"):
        moe_ffn_few(**to(inputs(4, 32, 16, 4, dtype=torch.float32), "cuda"))
    with pytest.raises(ValueError, match="on cpu"):
        moe_ffn_few(**dict(a, w_down=a["w_down"].cpu()))


@gpu
@pytest.mark.parametrize("i8", [False, True])
def test_a_token_does_not_depend_on_its_company(i8):
    a = to(inputs(64, 256, 176, 8, i8, True), "cuda")
    y, _ = moe_ffn_few(**a, top_k=3)
    for T in (1, 2, 9, 20, 33):
        b = dict(a, x=a["x"][64 - T:], residual=a["residual"][64 - T:])
        assert torch.equal(moe_ffn_few(**b, top_k=3)[0], y[64 - T:])
    b = dict(a, x=a["x"].flip(0), residual=a["residual"].flip(0))
    assert torch.equal(moe_ffn_few(**b, top_k=3)[0], y.flip(0))


@gpu
def test_a_token_that_is_not_finite_stays_alone():
    a = to(inputs(20, 128, 64, 8, False, True), "cuda")
    y, _ = moe_ffn_few(**a, top_k=2)
    a["x"][3, 5], a["x"][11, 0] = float("nan"), float("inf")
    z, counts = moe_ffn_few(**a, top_k=2)
    lost = torch.zeros(20, dtype=torch.bool)
    lost[[3, 11]] = True
    assert torch.isnan(z[lost]).all() and torch.equal(z[~lost], y[~lost]) and int(counts.sum()) == 40
    rt.check_status()


@gpu
def test_views():
    a = to(inputs(12, 64, 32, 4), "cuda")
    y, c = moe_ffn_few(**a)
    wide = torch.randn(12, 80, device="cuda", dtype=BF)
    wide[:, 8:72] = a["x"]
    odd = torch.randn(12, 80, device="cuda", dtype=BF)
    odd[:, 3:67] = a["residual"]
    b = dict(a, x=wide[:, 8:72], residual=odd[:, 3:67])
    assert torch.equal(moe_ffn_few(**b)[0], y)
    b = dict(a, x=a["x"].view(3, 2, 2, 64), residual=a["residual"].view(3, 2, 2, 64))
    assert torch.equal(moe_ffn_few(**b)[0], y.view(3, 2, 2, 64))
    b = dict(a, x=a["x"][5].expand(12, 64), residual=a["residual"][5].expand(12, 64))          # one row for all tokens
    assert torch.equal(moe_ffn_few(**b)[0], y[5].expand(12, 64))
    b = dict(a, x=a["x"].t().contiguous().t(), router_w=a["router_w"].t().contiguous().t())
    assert torch.equal(moe_ffn_few(**b)[0], y)


@gpu
@pytest.mark.parametrize("i8", [False, True])
def test_streams_and_graphs(i8):
    """Calls on two streams at once, and one captured and replayed on other inputs."""
    a = [to(inputs(T, 512, 256, 16, i8, T == 3, seed=T), "cuda") for T in (3, 50)]
    want = [moe_ffn_few(**b, top_k=4)[0] for b in a]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(30):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(moe_ffn_few(**a[i], top_k=4)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in (0, 1) for y in got[i])
    graph = torch.cuda.CUDAGraph()
    still = [dict(b, x=b["x"].clone()) for b in a]
    with torch.cuda.graph(graph):
        ys = [moe_ffn_few(**b, top_k=4) for b in still]
    for b in still:
        b["x"].mul_(-0.75)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for (y, c), b in zip(ys, still):
        z, d = moe_ffn_few(**b, top_k=4)
        assert torch.equal(y, z) and torch.equal(c, d)
    rt.check_status()


@gpu
def test_near_the_training_form():
    """moe_ffn rounds gate, up and each expert's result to bf16 as well: a handful of half steps of the parts' sizes."""
    a = to(inputs(48, 256, 512, 8), "cuda")
    y, counts = moe_ffn_few(**a)
    with torch.no_grad():
        z, _, c = moe_ffn(a["x"], a["router_w"], a["w_gate_up"], a["w_down"], a["residual"], 2)
    assert torch.equal(counts, c)
    assert float((y.float() - z.float()).norm()) <= 4 * 2.0 ** -8 * float(z.float().norm())


@gpu
@pytest.mark.parametrize("T", [1, 17, 40])
def test_every_code_is_widened_exactly(T):
    # 256 columns hold each code once in every row. Codes are exact in bf16 and the scale is a power of two, so both forms add up the same terms, sixteen at a time.
    D, F = 256, 64
    g = torch.Generator().manual_seed(3)
    codes = torch.stack([torch.arange(-128, 128).roll(37 * i) for i in range(2 * F)]).to(torch.int8)
    down = torch.stack([torch.randperm(256, generator=g)[:F] - 128 for _ in range(D)]).to(torch.int8)
    x = torch.randn(T, D, generator=g).to(BF)
    out = []
    for i8 in (True, False):
        weights = [Int8Weight(q[None], torch.full((1, len(q)), 2.0 ** -6)) if i8 else (q[None].to(BF) * 2.0 ** -6) for q in (codes, down)]
        a = to(dict(x=x, router_w=torch.zeros(1, D, dtype=BF), w_gate_up=weights[0], w_down=weights[1]), "cuda")
        out.append(moe_ffn_few(**a, top_k=1)[0])
    rt.check_status()
    assert torch.equal(*out)


@gpu
@pytest.mark.parametrize("T", [1, 40])
def test_experts_beyond_two_to_the_31(T):
    """The last two of 72 experts, by themselves and behind the others: probabilities of the others are 0."""
    E, D, F = 72, 4096, 4096
    g = torch.Generator("cuda").manual_seed(1)
    w = [Int8Weight(torch.randint(-127, 128, s, dtype=torch.int8, device="cuda", generator=g), torch.rand(s[:2], device="cuda", generator=g) * 1e-3)
         for s in ((E, 2 * F, D), (E, D, F))]
    x = torch.randn(T, D, device="cuda", generator=g).to(BF)
    x[:, 0] = 8.0
    router = torch.randn(E, D, device="cuda", generator=g).to(BF) * 0.02
    router[:E - 2, 0], router[E - 2:, 0] = -60.0, 0.0
    y, counts = moe_ffn_few(x, router, *w)
    z, _ = moe_ffn_few(x, router[E - 2:], *(Int8Weight(v.q[E - 2:], v.scale[E - 2:]) for v in w))
    assert counts.tolist() == [0] * (E - 2) + [T, T] and torch.equal(y, z)
    rt.check_status()


@gpu
@pytest.mark.parametrize("i8", [False, True])
def test_beside_products_that_hold_tensor_memory(i8):
    """Products whose clusters fit on an SM beside a CTA of the layer, on another stream: each side may find the tensor memory taken, and both end."""
    from innova_b200.ops.int8 import int8_linear
    a = to(inputs(40, 512, 256, 16, i8), "cuda")
    g = torch.Generator().manual_seed(4)
    w = Int8Weight(torch.randint(-127, 128, (4096, 512), dtype=torch.int8, generator=g).cuda(), torch.full((4096,), 1e-3).cuda())
    h = torch.randn(9, 512, generator=g).to(BF).cuda()
    want, other = moe_ffn_few(**a, top_k=4)[0], int8_linear(h, w)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(100):
        with torch.cuda.stream(streams[0]):
            got[0].append(moe_ffn_few(**a, top_k=4)[0])
        with torch.cuda.stream(streams[1]):
            got[1] += [int8_linear(h, w) for _ in range(3)]
    torch.cuda.synchronize()
    rt.check_status()
    assert all(torch.equal(y, want) for y in got[0]) and all(torch.equal(y, other) for y in got[1])


def test_weights_and_scales_that_ask_for_gradients_are_refused():
    a, b = inputs(4, 32, 16, 4, shared=True), inputs(4, 32, 16, 4, True, True)
    ask = lambda w: Int8Weight(w.q, w.scale.clone().requires_grad_()) if isinstance(w, Int8Weight) else w.clone().requires_grad_()  # noqa: E731
    for c in (a, b):
        for bad in (dict(w_gate_up=ask(c["w_gate_up"])), dict(w_down=ask(c["w_down"])), dict(shared=(ask(c["shared"][0]), c["shared"][1])),
                    dict(shared=(c["shared"][0], ask(c["shared"][1])))):
            with pytest.raises(RuntimeError, match="no gradient"):
                moe_ffn_few(**{**c, **bad})
