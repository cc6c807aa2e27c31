"""Generation from mixture decoders, and with weights in 8-bit integers: the products and the expert layer together, as they are used."""
import copy

import pytest
import torch

from innova_b200.inference.generator import Generator
from innova_b200.models import DenseModel, MoEModel, TransformerConfig
from innova_b200.ops import runtime as rt
from innova_b200.ops.int8 import Int8Linears, Int8Weight, int8_linear

gpu = pytest.mark.gpu


def mixture(dtype=torch.float32, device="cpu", shared=True, **kw):
    cfg = TransformerConfig(**{**dict(vocab_size=97, hidden_size=64, num_layers=2, num_heads=4, head_dim=16, ffn_hidden_size=96, moe_ffn_hidden_size=48, num_experts=6,
                                      top_k=2, shared_expert=shared, num_kv_heads=2, max_seq_len=160, vocab_pad_to=1), **kw})
    m = MoEModel(cfg, dtype=dtype, seed=3).eval()
    with torch.no_grad():           # routers and embeddings that tell tokens apart
        for n, p in m.named_parameters():
            if p.dim() > 1:
                p.mul_(4.0 if "router" in n else 2.0)
    return m.to(device)


def dense(dtype=torch.float32, device="cpu", **kw):
    cfg = TransformerConfig(**{**dict(vocab_size=97, hidden_size=64, num_layers=2, num_heads=4, head_dim=16, ffn_hidden_size=96, num_kv_heads=2, max_seq_len=160,
                                      vocab_pad_to=1), **kw})
    return DenseModel(cfg, dtype=dtype).eval().to(device)


def greedy(model, ids, n):
    out, cur = [], ids.clone()
    with torch.no_grad():
        for _ in range(n):
            out.append(model(cur)[:, -1].argmax(-1))
            cur = torch.cat([cur, out[-1].view(-1, 1)], 1)
    return torch.stack(out, 1).tolist()


def rounded(model):
    """The model with its blocks' weights as 8-bit integers stand for them."""
    m = copy.deepcopy(model)
    with torch.no_grad():
        for n, p in m.named_parameters():
            if p.dim() > 1 and "layers." in n and "router" not in n:
                p.copy_(Int8Weight.quantize(p).dequantize())
    return m


@pytest.mark.parametrize("shared", [False, True])
def test_mixture_generates_what_the_whole_model_says(shared):
    m = mixture(shared=shared)
    ids = torch.randint(0, 97, (2, 9), generator=torch.Generator().manual_seed(1))
    want = greedy(m, ids, 6)
    gen = Generator(m, kv_format="bf16", max_batch=2, max_seq=64)
    assert gen.generate_tokens(ids, max_new_tokens=6) == want
    assert all(int(blk.moe.last_counts.sum()) == 4 for blk in m.layers)          # two tokens, two experts each


def test_mixture_prompt_of_many_tokens():
    """More than 64 tokens run as in training, the steps behind them in the form for a few."""
    m = mixture()
    ids = torch.randint(0, 97, (1, 100), generator=torch.Generator().manual_seed(2))
    assert Generator(m, kv_format="bf16", max_batch=1, max_seq=160).generate_tokens(ids, max_new_tokens=5) == greedy(m, ids, 5)


def test_mixture_with_biased_activation_of_the_shared_expert():
    m = mixture(activation="gelu", bias=True)
    ids = torch.randint(0, 97, (1, 7), generator=torch.Generator().manual_seed(3))
    assert not m.layers[0].moe._plain_shared()
    assert Generator(m, kv_format="bf16", max_batch=1, max_seq=64).generate_tokens(ids, max_new_tokens=4) == greedy(m, ids, 4)


def test_mixture_trained_in_a_format_is_served_in_it():
    m = mixture(ste_format="oil8")
    ids = torch.randint(0, 97, (2, 9), generator=torch.Generator().manual_seed(8))
    x, h = torch.randn(4, 64), torch.randn(4, 64)
    moe = m.layers[0].moe
    with torch.no_grad():
        assert torch.allclose(moe.serve(h, x), moe(h, x)[0], rtol=1e-5, atol=1e-6)
    assert len(Generator(m, kv_format="bf16", max_batch=2, max_seq=64, weight_format="int8").generate_tokens(ids, max_new_tokens=3)[0]) == 3


def test_int8_experts_are_their_values():
    """With experts alone in 8 bits a mixture says what the model with those values says: nothing else is rounded on the CPU."""
    m = mixture()
    r = copy.deepcopy(m)
    with torch.no_grad():
        for blk in r.layers:
            for p in (blk.moe.w_gate_up, blk.moe.w_down, blk.moe.shared.gate_up_proj.weight, blk.moe.shared.down_proj.weight):
                p.copy_(Int8Weight.quantize(p).dequantize())
    h = torch.randn(5, 64)
    x = torch.randn(5, 64)
    for a, b in zip(m.layers, r.layers):
        y, z = a.moe.serve(h, x, a.moe.int8_weights()), b.moe.serve(h, x)
        assert torch.allclose(y, z, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("make", [dense, mixture])
def test_int8_generation_cpu(make):
    """Every projection is the 8-bit product: the generator says what one with that product as its linear_fn says, and is near the plain one."""
    m = make()
    ids = torch.randint(0, 97, (2, 9), generator=torch.Generator().manual_seed(4))
    gen = Generator(m, kv_format="bf16", max_batch=2, max_seq=64, weight_format="int8")
    assert isinstance(gen.linear, Int8Linears)
    lin = m.layers[0].attention.qkv_proj
    x = torch.randn(3, 64)
    assert torch.equal(gen.linear(x, lin), int8_linear(x, Int8Weight.quantize(lin.weight)))
    y = gen._forward(ids, [0, 0])
    with torch.no_grad():
        want = rounded(m)(ids)[:, -1]
    # activations of every product are off by at most half a step of 1/127 of their row's largest value: some 4 / 254 of the usual one, over a few layers
    assert float((y - want).norm()) < 0.1 * float(want.norm())
    assert len(gen.generate_tokens(ids, max_new_tokens=5)[0]) == 5


def test_int8_refusals():
    m = dense()
    with pytest.raises(ValueError, match="weight_format"):
        Generator(m, kv_format="bf16", weight_format="int4")
    with pytest.raises(ValueError, match="linear_fn"):
        Generator(m, kv_format="bf16", weight_format="int8", linear_fn=lambda x, lin: lin(x))


@gpu
@pytest.mark.parametrize("fmt", ["bf16", "fp8"])
def test_mixture_generation_gpu(fmt):
    """The steps' form and the training form give the same logits up to roundings to bf16, and steps the same as a prompt."""
    kw = dict(vocab_pad_to=128, hidden_size=256, num_heads=4, head_dim=64, moe_ffn_hidden_size=192, num_experts=8)
    m = mixture(torch.bfloat16, "cuda", **kw)
    ids = torch.randint(0, 97, (3, 20), generator=torch.Generator().manual_seed(5)).cuda()
    gen = Generator(m, kv_format=fmt, max_batch=3, max_seq=64)
    few = gen._forward(ids, [0] * 3).float()                            # 60 tokens: the form for a few
    with torch.no_grad():
        whole = m(ids)[:, -1].float()
    # a handful of roundings to bf16 a layer, 2^-8 each, two layers
    assert float((few - whole).norm()) < 16 * 2.0 ** -8 * float(whole.norm())
    out = gen.generate_tokens(ids, max_new_tokens=8)
    assert [len(o) for o in out] == [8, 8, 8] and gen.generate_tokens(ids, max_new_tokens=8) == out
    rt.check_status()


@gpu
@pytest.mark.parametrize("make", [dense, mixture])
def test_int8_generation_gpu(make):
    kw = dict(vocab_pad_to=128, hidden_size=256, num_heads=4, head_dim=64, ffn_hidden_size=512)
    m = make(torch.bfloat16, "cuda", **kw)
    gen = Generator(m, kv_format="bf16", max_batch=2, max_seq=160, weight_format="int8")
    ids = torch.randint(0, 97, (2, 30), generator=torch.Generator().manual_seed(6)).cuda()
    y = gen._forward(ids, [0, 0]).float()
    with torch.no_grad():
        want = rounded(m)(ids)[:, -1].float()
    assert float((y - want).norm()) < 0.15 * float(want.norm())         # the activations' steps as on the CPU, and bf16's
    out = gen.generate_tokens(ids, max_new_tokens=12)
    assert [len(o) for o in out] == [12, 12] and gen.generate_tokens(ids, max_new_tokens=12) == out
    long = torch.randint(0, 97, (2, 100), generator=torch.Generator().manual_seed(7)).cuda()      # tiles, and mixtures as in training
    assert [len(o) for o in gen.generate_tokens(long, max_new_tokens=3)] == [3, 3]
    rt.check_status()


def of_their_values(layer):
    """The layer with its experts' weights as 8-bit integers stand for them."""
    r = copy.deepcopy(layer)
    with torch.no_grad():
        for p in (r.w_gate_up, r.w_down) + ((r.shared.gate_up_proj.weight, r.shared.down_proj.weight) if r._plain_shared() else ()):
            p.copy_(Int8Weight.quantize(p).dequantize())
    return r


@pytest.mark.parametrize("kw", [{}, dict(num_experts=260, moe_ffn_hidden_size=8), dict(num_experts=20, top_k=17, moe_ffn_hidden_size=8), dict(activation="gelu", bias=True)])
@pytest.mark.parametrize("T", [1, 64, 65, 150, 600])
def test_int8_experts_whatever_the_number_of_tokens(T, kw):
    """Long prompts, many experts and many choices run on the 8-bit experts too, not on the weights that these were made from."""
    m = mixture(**kw).layers[0].moe
    g = torch.Generator().manual_seed(T)
    h, x = torch.randn(2, T, 64, generator=g)[:, :T], torch.randn(2, T, 64, generator=g)
    w = m.int8_weights()
    with torch.no_grad():
        y, want, plain = m.serve(h, x, w), of_their_values(m)(h, x)[0], m(h, x)[0]
    assert y.shape == h.shape and int(m.last_counts.sum()) == 2 * T * m.cfg.top_k
    # fp32 sums in another order: chains of 64 + 48 + 18 steps at most, each off by half a step of what is added up, which stays below the largest value; twice that
    # for the activation between. The rounding of the weights to 8 bits is to be seen beyond it.
    tol = 200 * 2.0 ** -24 * float(want.abs().max())
    assert float((y - want).abs().max()) <= tol < 0.5 * float((y - plain).abs().max())
    assert float((m.serve(h[:1, :1], x[:1, :1], w) - y[:1, :1]).abs().max()) <= tol


def test_int8_experts_of_several_ranks_are_refused():
    m = mixture()
    m.layers[1].moe.ep = object()
    with pytest.raises(ValueError, match="several ranks"):
        Generator(m, kv_format="bf16", weight_format="int8")


def test_dequantised_in_a_type():
    w = Int8Weight.quantize(torch.randn(3, 5, 40))
    assert torch.equal(w.dequantize(torch.bfloat16), w.dequantize().bfloat16()) and torch.equal(w.dequantize(), w.q.float() * w.scale.unsqueeze(-1))
    asked = Int8Weight(w.q, w.scale.clone().requires_grad_())
    asked.dequantize(torch.bfloat16).sum().backward()
    assert asked.scale.grad is not None


@gpu
def test_int8_experts_whatever_the_number_of_tokens_gpu():
    kw = dict(vocab_pad_to=128, hidden_size=256, num_heads=4, head_dim=64, moe_ffn_hidden_size=192, num_experts=8)
    m = mixture(torch.bfloat16, "cuda", **kw).layers[0].moe
    w, r = m.int8_weights(), of_their_values(m)
    g = torch.Generator("cuda").manual_seed(1)
    h, x = (torch.randn(1, 3000, 256, device="cuda", generator=g).bfloat16() for _ in range(2))
    with torch.no_grad():
        few = torch.cat([m.serve(h[:, i:i + 60], x[:, i:i + 60], w) for i in range(0, 3000, 60)], 1)
        for T in (65, 130, 400, 512):
            assert torch.equal(m.serve(h[:, :T], x[:, :T], w), few[:, :T])       # chunks: the same to the last bit
        many, want = m.serve(h, x, w), r(h, x)[0]
        assert torch.equal(many, want)                                            # the training form on the same rounded weights
        # a handful of roundings to bf16 in each form
        assert float((many.float() - few.float()).norm()) < 6 * 2.0 ** -8 * float(few.float().norm())
        odd = mixture(torch.bfloat16, "cuda", **{**kw, "hidden_size": 248, "num_heads": 31, "num_kv_heads": 31, "head_dim": 8}).layers[0].moe      # no form in 8 bits for a few
        for T in (3, 100):
            assert torch.equal(odd.serve(h[:, :T, :248], x[:, :T, :248], odd.int8_weights()), of_their_values(odd)(h[:, :T, :248], x[:, :T, :248])[0])
    rt.check_status()
