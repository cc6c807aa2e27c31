"""Norms of query and key heads with the rotation in the same pass: forward and gradients against the formulas in 64 bits, refusals, the model's use."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

from innova_b200 import ops
from innova_b200.models import DenseModel, MoEModel, TransformerConfig
from innova_b200.ops import runtime as rt

DEV, EPS = "cuda", 1e-5
# y = R(w x r): the mean's sum and the root lose under 2^-19, products and the rotation 2^-22 more, of the pair's size; one rounding to the type
FLOAT = 2.0 ** -18
# a sum of dw: chains of under 160 additions (a lane's heads and tokens, lanes, warps, rows) of terms that are off by 2^-19
SUM = 160 * 2.0 ** -24 + 2.0 ** -18


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def formula(x, wq, wk, cos, sin, H, G, D, pos):
    """x [T, heads, D] in 64 bits."""
    def head(h, w):
        h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * w
        if cos is None:
            return h
        n = cos.shape[1]
        c, s = cos.double()[pos].unsqueeze(1), sin.double()[pos].unsqueeze(1)
        a, b = h[..., :n], h[..., n:2 * n]
        return torch.cat([a * c - b * s, a * s + b * c, h[..., 2 * n:]], -1)
    return torch.cat([head(x[:, :H], wq), head(x[:, H:H + G], wk), x[:, H + G:]], 1)


def inputs(B, S, H, G, D, rot, dtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, S, (H + 2 * G) * D, generator=g) * torch.exp(torch.randn(B, S, 1, generator=g))).to(dtype)
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(dtype) for _ in "qk")
    dy = torch.randn(B, S, (H + 2 * G) * D, generator=g).to(dtype)
    cos, sin = ops.rope_tables(S + 40, rot) if rot else (None, None)
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    return [to(t) for t in (x, wq, wk, dy, cos, sin)]


def check(dtype, dev, B, S, H, G, D, rot, positions=None, seed=0):
    x, wq, wk, dy, cos, sin = inputs(B, S, H, G, D, rot, dtype, dev, seed)
    leaves = [t.clone().requires_grad_() for t in (x, wq, wk)]
    y = ops.qk_norm_rope(*leaves, cos, sin, H, G, D, positions, EPS)
    assert y.shape == x.shape and y.dtype == dtype
    grads = torch.autograd.grad(y, leaves, dy)
    T = B * S
    pos = torch.arange(S, device=dev).repeat(B) if positions is None else positions.reshape(-1).long()
    ref = [t.detach().double().requires_grad_() for t in (x.view(T, H + 2 * G, D), wq, wk)]
    yr = formula(*ref, cos, sin, H, G, D, pos)
    gr = torch.autograd.grad(yr, ref, dy.double().view(T, H + 2 * G, D))
    half = half_step(dtype)
    # the size of what a value is made from: its head's largest normed value or gradient
    def near(a, b, size):
        a, b = a.double().view_as(b), b.detach()
        bad = ((a - b).abs() > half * b.abs() + FLOAT * size).sum()
        assert int(bad) == 0, float(((a - b).abs() / (half * b.abs() + FLOAT * size + 1e-300)).max())
    near(y, yr, yr.detach().abs().amax(-1, keepdim=True))
    r = 1 / torch.sqrt(x.double().view(T, -1, D).square().mean(-1, keepdim=True) + EPS)
    w = torch.cat([wq.double().expand(H, D), wk.double().expand(G, D), torch.ones(G, D, device=dev)]).abs().amax(-1, keepdim=True)
    gd = dy.double().view(T, -1, D)
    # dx = r (g w - xh mean(g w xh)), |xh| <= sqrt(D), |mean| <= max |g w| : of the size of r w |g| sqrt(D)
    near(grads[0], gr[0], r * w * gd.abs().amax(-1, keepdim=True) * 2 * math.sqrt(D))
    back = gd
    if rot:
        n = cos.shape[1]
        c, s = cos.double()[pos].unsqueeze(1), sin.double()[pos].unsqueeze(1)
        a, b = gd[..., :n], gd[..., n:2 * n]
        back = torch.cat([a * c + b * s, b * c - a * s, gd[..., 2 * n:]], -1)
    terms = (back * x.double().view(T, -1, D) * r).abs()
    for a, b, t in ((grads[1], gr[1], terms[:, :H]), (grads[2], gr[2], terms[:, H:H + G])):
        assert bool(((a.double() - b).abs() <= half * b.abs() + SUM * t.sum((0, 1))).all())
    assert torch.equal(y.view(T, -1, D)[:, H + G:], x.view(T, -1, D)[:, H + G:])


SHAPES = [(1, 1, 1, 1, 64, 64), (2, 5, 4, 2, 64, 64), (1, 77, 8, 8, 64, 64), (3, 33, 6, 2, 128, 128), (1, 9, 5, 1, 80, 48), (2, 7, 3, 3, 96, 96),
          (1, 13, 4, 1, 256, 64), (2, 3, 7, 1, 16, 16), (1, 6, 2, 2, 32, 0), (1, 600, 10, 2, 64, 16), (4, 41, 1, 1, 48, 16)]


@pytest.mark.parametrize("shape", SHAPES[:7])
def test_cpu_matches_the_formula(shape):
    check(torch.float32, "cpu", *shape)


def test_cpu_gradients_against_differences():
    x, wq, wk, _, cos, sin = inputs(1, 4, 3, 1, 16, 8, torch.float64, "cpu")
    leaves = [t.requires_grad_() for t in (x, wq, wk)]
    assert torch.autograd.gradcheck(lambda *a: ops.qk_norm_rope(*a, cos, sin, 3, 1, 16), leaves)


@pytest.mark.parametrize("shape", [(2, 0, 512), (0, 3, 512), (0, 512)])
def test_cpu_no_tokens(shape):
    cos, sin = ops.rope_tables(9, 64)
    x, w = torch.zeros(shape), torch.ones(64, requires_grad=True)
    y = ops.qk_norm_rope(x, w, torch.ones(64), cos, sin, 4, 2, 64)
    assert y.shape == shape and float(torch.autograd.grad(y.sum(), w)[0].abs().sum()) == 0


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_refusals(dev):
    x, wq, wk, _, cos, sin = inputs(2, 5, 4, 2, 64, 64, torch.float32 if dev == "cpu" else torch.bfloat16, dev)
    call = lambda x=x, wq=wq, wk=wk, cos=cos, sin=sin, H=4, G=2, D=64, pos=None: ops.qk_norm_rope(x, wq, wk, cos, sin, H, G, D, pos)  # noqa: E731
    call()
    for bad in (dict(H=5), dict(G=0), dict(D=32), dict(wq=wq[:32]), dict(wk=wk.double()), dict(cos=None), dict(cos=cos.half(), sin=sin.half()),
                dict(cos=cos[:3], sin=sin[:3]), dict(pos=torch.zeros(9, dtype=torch.int32, device=dev)), dict(pos=torch.zeros(10, device=dev)),
                dict(x=x[0, 0]), dict(cos=torch.ones(9, 40, device=dev), sin=torch.ones(9, 40, device=dev))):
        with pytest.raises((ValueError, TypeError)):
            call(**bad)
    if dev == "cpu":
        with pytest.raises(ValueError):
            call(pos=torch.full((10,), 45, dtype=torch.int32))
        with pytest.raises(ValueError):
            call(pos=torch.full((10,), -1, dtype=torch.int32))
    else:
        with pytest.raises(TypeError):
            call(x=x.half(), wq=wq.half(), wk=wk.half())
        with pytest.raises(ValueError):
            ops.qk_norm_rope(x[..., :8 * 8], wq[:8], wk[:8], cos[:, :4], sin[:, :4], 4, 2, 8)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_forward_mode_is_not_dropped(dev):
    """A tangent of any input comes back right (the directional derivative that the gradients give) or is refused; without one nothing changes."""
    x, wq, wk, dy, cos, sin = inputs(1, 5, 2, 1, 32, 16, torch.float32, dev)
    call = lambda x, wq, wk: ops.qk_norm_rope(x, wq, wk, cos, sin, 2, 1, 32)  # noqa: E731
    want = call(x, wq, wk)
    assert not want.requires_grad
    for which in range(3):
        args = [x, wq, wk]
        tangent = torch.randn(args[which].shape, generator=torch.Generator().manual_seed(which)).to(dev)
        alone = lambda t: call(*[t if i == which else a for i, a in enumerate(args)])  # noqa: E731
        if dev == "cpu":
            got = torch.func.jvp(alone, (args[which],), (tangent,))[1]
            leaf = args[which].clone().requires_grad_()
            g = torch.autograd.grad(alone(leaf), leaf, dy)[0]
            a, b = (got * dy).double().sum(), (g * tangent).double().sum()          # the same sum in two orders, of terms that lose under FLOAT
            assert abs(a - b) <= 4 * FLOAT * float((got * dy).abs().sum() + (g * tangent).abs().sum())
            continue
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(alone, (args[which],), (tangent,))
        with fwd.dual_level():
            with pytest.raises((RuntimeError, NotImplementedError)):
                alone(fwd.make_dual(args[which], tangent))
            assert torch.equal(call(x, wq, wk), want)


def tiny(cls=DenseModel, **kw):
    base = dict(vocab_size=300, hidden_size=128, num_layers=2, num_heads=2, head_dim=64, ffn_hidden_size=256, num_kv_heads=1, max_seq_len=128, qk_norm=True,
                vocab_pad_to=8)
    return TransformerConfig(**{**base, **kw})


def test_model_with_head_norms_on_the_cpu(tmp_path):
    from innova_b200.formats import export
    torch.manual_seed(0)
    cfg = tiny(hidden_size=64, num_heads=4, head_dim=16, num_kv_heads=2, ffn_hidden_size=96)
    m = DenseModel(cfg, dtype=torch.float32)
    names = {n for n, _ in m.named_parameters() if "q_norm" in n or "k_norm" in n}
    assert len(names) == 4
    with torch.no_grad():
        for n, p in m.named_parameters():
            if n in names:
                p.add_(0.3 * torch.randn_like(p))
    ids = torch.randint(0, 300, (2, 9))
    m(ids, labels=ids).backward()
    assert all(float(p.grad.abs().sum()) > 0 for n, p in m.named_parameters() if n in names)
    path = str(tmp_path / "m.oil")
    export.save_model(m.eval(), path, fmt="OIL32")
    again = export.load_model(path)
    assert again.cfg.qk_norm and torch.allclose(again(ids), m(ids), atol=1e-6)
    e = MoEModel(tiny(hidden_size=64, num_heads=4, head_dim=16, num_kv_heads=2, num_experts=2, moe_ffn_hidden_size=64), dtype=torch.float32)
    state = e.state_dict_reference()
    assert "layers.1.attention.k_norm.weight" in state
    state["layers.1.attention.k_norm.weight"] = torch.full((16,), 2.0)
    e.load_reference_state(state)
    assert float(e.layers[1].attention.k_norm.weight.detach()[3]) == 2.0


def test_decoders_without_head_norms_refuse_them():
    from innova_b200.models.tp_dense import TPDenseModel
    from innova_b200.parallel.tp import TPDecoder
    with pytest.raises(NotImplementedError):
        TPDenseModel(tiny(), device="cpu", comm=object())
    with pytest.raises(NotImplementedError):
        TPDecoder(tiny(), device="cpu", single=True)
    with pytest.raises(NotImplementedError):
        TPDecoder(tiny(qk_norm=False), device="cpu", single=True, kv_format="fp8")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_gpu_matches_the_formula(shape, dtype):
    check(dtype, DEV, *shape)
    rt.check_status()


@pytest.mark.gpu
def test_gpu_positions_strides_and_empty():
    pos = torch.randint(0, 45, (2, 5), device=DEV, dtype=torch.int32)
    check(torch.bfloat16, DEV, 2, 5, 4, 2, 64, 64, pos)
    x, wq, wk, dy, cos, sin = inputs(1, 12, 4, 2, 64, 64, torch.bfloat16, DEV)
    want = ops.qk_norm_rope(x, wq, wk, cos, sin, 4, 2, 64)
    wide = torch.randn(1, 12, 8 * 64 + 40, device=DEV).bfloat16()
    for off in (0, 8, 3):                                    # rows behind one another, and one that starts off 16 bytes
        view = wide[..., off:off + 512]
        view.copy_(x)
        assert torch.equal(ops.qk_norm_rope(view, wq, wk, cos, sin, 4, 2, 64), want)
    wpad = torch.randn(80, device=DEV).bfloat16()
    wpad[3:67] = wq
    assert torch.equal(ops.qk_norm_rope(x, wpad[3:67], wk, cos, sin, 4, 2, 64), want)
    leaf = x.clone().requires_grad_()
    a = torch.autograd.grad(ops.qk_norm_rope(leaf, wq, wk, cos, sin, 4, 2, 64).sum(), leaf)[0]      # a gradient of stride zero
    b = torch.autograd.grad(ops.qk_norm_rope(leaf, wq, wk, cos, sin, 4, 2, 64), leaf, torch.ones_like(x))[0]
    assert torch.equal(a, b)
    t = dy.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(torch.autograd.grad(ops.qk_norm_rope(leaf, wq, wk, cos, sin, 4, 2, 64), leaf, t)[0],
                       torch.autograd.grad(ops.qk_norm_rope(leaf, wq, wk, cos, sin, 4, 2, 64), leaf, dy)[0])
    empty = torch.empty(2, 0, 512, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    w = wq.clone().requires_grad_()
    y = ops.qk_norm_rope(empty, w, wk, cos, sin, 4, 2, 64)
    assert y.shape == empty.shape and float(torch.autograd.grad(y.sum(), w)[0].abs().sum()) == 0
    rt.check_status()


@pytest.mark.gpu
def test_gpu_position_outside_the_table_is_reported():
    x, wq, wk, _, cos, sin = inputs(1, 4, 2, 1, 64, 64, torch.bfloat16, DEV)
    pos = torch.tensor([0, 44, 10 ** 6, -5], device=DEV, dtype=torch.int32)       # the kernel reads the nearest rows instead
    y = ops.qk_norm_rope(x, wq, wk, cos, sin, 2, 1, 64, pos)
    with pytest.raises(RuntimeError):
        rt.check_status()
    want = ops.qk_norm_rope(x, wq, wk, cos, sin, 2, 1, 64, pos.clamp(0, cos.shape[0] - 1))
    rt.check_status()
    assert torch.equal(y, want)


@pytest.mark.gpu
def test_gpu_positions_of_64_bits_are_not_cut():
    x, wq, wk, _, cos, sin = inputs(1, 4, 2, 1, 64, 64, torch.bfloat16, DEV)
    pos = torch.tensor([0, 3, 2 ** 32 + 2, -2 ** 32 + 1], device=DEV)
    y = ops.qk_norm_rope(x, wq, wk, cos, sin, 2, 1, 64, pos)
    with pytest.raises(RuntimeError):
        rt.check_status()
    assert torch.equal(y, ops.qk_norm_rope(x, wq, wk, cos, sin, 2, 1, 64, pos.clamp(0, cos.shape[0] - 1)))
    rt.check_status()


@pytest.mark.gpu
def test_gpu_gradients_repeat_and_go_to_main_grads():
    x, wq, wk, dy, cos, sin = inputs(3, 500, 8, 4, 64, 64, torch.bfloat16, DEV)
    leaves = [t.clone().requires_grad_() for t in (x, wq, wk)]
    first = torch.autograd.grad(ops.qk_norm_rope(*leaves, cos, sin, 8, 4, 64), leaves, dy)
    for _ in range(3):
        again = torch.autograd.grad(ops.qk_norm_rope(*leaves, cos, sin, 8, 4, 64), leaves, dy)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    for w in leaves[1:]:
        w.main_grad = torch.ones(64, device=DEV)
    ops.qk_norm_rope(*leaves, cos, sin, 8, 4, 64).backward(dy)
    assert leaves[1].grad is None and leaves[2].grad is None
    assert all(torch.allclose(w.main_grad - 1, g.float(), rtol=2.0 ** -7, atol=1e-3) for w, g in zip(leaves[1:], first[1:]))
    both = wq.clone().requires_grad_()                          # one weight for both norms
    both.main_grad = torch.zeros(64, device=DEV)
    ops.qk_norm_rope(x, both, both, cos, sin, 8, 4, 64).backward(dy)
    alone = [wq.clone().requires_grad_() for _ in "qk"]
    ops.qk_norm_rope(x, *alone, cos, sin, 8, 4, 64).backward(dy)
    want = alone[0].grad.float() + alone[1].grad.float()
    assert torch.allclose(both.main_grad, want, rtol=0, atol=2.0 ** -7 * float(want.abs().max()))


@pytest.mark.gpu
def test_gpu_main_grads_of_other_forms():
    """A main_grad that is not dense fp32 is added to, and nothing beside it."""
    x, wq, wk, dy, cos, sin = inputs(2, 50, 8, 4, 64, 64, torch.bfloat16, DEV)
    plain = [t.clone().requires_grad_() for t in (x, wq, wk)]
    ops.qk_norm_rope(*plain, cos, sin, 8, 4, 64).backward(dy)
    want = [w.grad.float() for w in plain[1:]]
    for shape, dtype, part in (((128,), torch.bfloat16, lambda t: t[:64]), ((64, 2), torch.float32, lambda t: t[:, 0]), ((8, 8), torch.float32, lambda t: t),
                               ((64,), torch.float64, lambda t: t)):
        some = [t.clone().requires_grad_() for t in (x, wq, wk)]
        whole = [torch.ones(shape, device=DEV, dtype=dtype) for _ in "qk"]
        for w, t in zip(some[1:], whole):
            w.main_grad = part(t)
        ops.qk_norm_rope(*some, cos, sin, 8, 4, 64).backward(dy)
        for w, t, g in zip(some[1:], whole, want):
            assert w.grad is None
            # the gradient's own rounding in `want`, the main_grad's here
            assert bool(((w.main_grad.reshape(64).float() - 1 - g).abs() <= 2.0 ** -8 * g.abs() + 2.0 ** -8 * (g + 1).abs() + 2.0 ** -20).all())
            part(t).fill_(1)
            assert bool((t == 1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("wants", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (0, 1, 1), (0, 1, 0), (0, 0, 1)])
def test_gpu_gradients_that_nobody_asked_for(wants):
    """A frozen input gets none and a frozen weight's main_grad is left alone; the others' are the same to the bit, and frozen norms save their launch."""
    x, wq, wk, dy, cos, sin = inputs(3, 50, 8, 4, 64, 64, torch.bfloat16, DEV)
    full = [t.clone().requires_grad_() for t in (x, wq, wk)]
    ops.qk_norm_rope(*full, cos, sin, 8, 4, 64).backward(dy)
    for with_main in (False, True):
        some = [t.clone().requires_grad_(bool(w)) for t, w in zip((x, wq, wk), wants)]
        if with_main:
            for w in some[1:]:
                w.main_grad = torch.ones(64, device=DEV)
        before = rt.launch_count()
        ops.qk_norm_rope(*some, cos, sin, 8, 4, 64).backward(dy)
        assert rt.launch_count() - before == (3 if wants[1] or wants[2] else 2)
        for i, (t, f, w) in enumerate(zip(some, full, wants)):
            if with_main and i:
                assert t.grad is None
                assert torch.allclose(t.main_grad - 1, f.grad.float(), rtol=2.0 ** -7, atol=1e-3) if w else bool((t.main_grad == 1).all())
            else:
                assert torch.equal(t.grad, f.grad) if w else t.grad is None


@pytest.mark.gpu
def test_gpu_captured_forward_and_backward():
    x, wq, wk, dy, cos, sin = inputs(2, 50, 4, 2, 128, 128, torch.bfloat16, DEV)
    leaves = [t.clone().requires_grad_() for t in (x, wq, wk)]

    def step():
        y = ops.qk_norm_rope(*leaves, cos, sin, 4, 2, 128)
        return [y, *torch.autograd.grad(y, leaves, dy)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        leaves[0].mul_(0.5)
        dy.add_(1)
    graph.replay()
    got = [t.clone() for t in got]
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.gpu
def test_gpu_model_trains_as_on_the_cpu():
    """Gradients of a bf16 step with head norms against the same weights in fp32 on the CPU."""
    torch.manual_seed(1)
    cpu = DenseModel(tiny(), dtype=torch.float32)
    with torch.no_grad():
        for n, p in cpu.named_parameters():
            p.copy_((p + (0.2 * torch.randn_like(p) if "_norm.weight" in n and p.dim() == 1 else 0)).bfloat16())
    gpu = DenseModel(tiny(), dtype=torch.bfloat16, device=DEV)
    gpu.load_state_dict(cpu.state_dict())
    ids = torch.randint(0, 300, (2, 65))
    lc, lg = cpu(ids, labels=ids), gpu(ids.to(DEV), labels=ids.to(DEV))
    lc.backward()
    lg.backward()
    assert abs(lc.item() - lg.item()) < 0.02 * lc.item()
    for (n, a), b in zip(cpu.named_parameters(), gpu.parameters()):
        # a value passes about forty roundings of half a bf16 step on its way through two layers and back: at most 40 * 2^-8, of random signs near 2.5 %
        assert float((b.grad.float().cpu() - a.grad).norm() / a.grad.norm()) < 0.08, n
    rt.check_status()


@pytest.mark.gpu
def test_gpu_tables_off_16_bytes():
    x, wq, wk, dy, cos, sin = inputs(2, 9, 4, 2, 64, 32, torch.bfloat16, DEV)
    off = [torch.zeros(t.numel() + 1, device=DEV)[1:].view_as(t).copy_(t) for t in (cos, sin)]
    assert all(t.data_ptr() % 16 for t in off)
    assert torch.equal(ops.qk_norm_rope(x, wq, wk, *off, 4, 2, 64), ops.qk_norm_rope(x, wq, wk, cos, sin, 4, 2, 64))
    wide = [torch.zeros(t.shape[0], t.shape[1] + 3, device=DEV)[:, 1:-2].copy_(t) for t in (cos, sin)]
    assert torch.equal(ops.qk_norm_rope(x, wq, wk, *wide, 4, 2, 64), ops.qk_norm_rope(x, wq, wk, cos, sin, 4, 2, 64))
