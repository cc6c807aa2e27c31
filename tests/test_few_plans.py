"""How products in 8-bit integers and expert layers of a few tokens are cut and launched (csrc/int8_linear.cu, csrc/moe_few.cu): every product of grid and index
stays within what it indexes, over sizes drawn from all that the calls take; and results, codes and workspaces that lie between guard values, on a GPU."""
import ctypes
import random

import pytest
import torch

from innova_b200 import _native
from innova_b200.ops import int8, moe
from innova_b200.ops import runtime as rt
from innova_b200.ops.int8 import Int8Weight

gpu = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
SMEM, SM = 227 * 1024, 228 * 1024                   # of a CTA, of an SM; a CTA takes 1 KB more than it asks for


def sizes(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def product_plan(T, N, K, gated):
    out = (ctypes.c_int * 13)()
    assert _native.cuda().inv_int8_plan(T, N, K, int(gated), ctypes.addressof(out)) == 0
    return dict(zip("route cols grid cluster threads smem tiles t_tiles tb per kb parts stages".split(), out))


def hold_product(T, N, K, gated):
    p = product_plan(T, N, K, gated)
    route, cols, tb, per, stages = p["route"], p["cols"], p["tb"], p["per"], p["stages"]
    what = (T, N, K, gated, p)
    assert cols == (N // 2 if gated else N) and 0 < p["smem"] <= SMEM and 32 <= p["threads"] <= 1024 and p["threads"] % 32 == 0, what
    assert p["grid"] % p["cluster"] == 0 and 1 <= p["cluster"] <= 8 and p["grid"] < 2 ** 31, what
    if route == 0:
        width = -(-K // (512 if T <= 2 else 128)) * (512 if T <= 2 else 128)
        assert T <= 4 and tb == T and (p["tiles"] - 1) * per < cols <= p["tiles"] * per and p["grid"] == min(p["tiles"], 296), what
        assert p["smem"] == T * (width + (16 if T > 2 else 0)) and p["smem"] + 1024 + 20 * 1024 <= SM // 2, what       # codes; two CTAs an SM beside the static part
        assert per * (2 if gated else 1) <= (512 if T <= 2 else 32) and (T <= 2 or per == (16 if gated else 32)), what     # sums of a tile
        assert per * (2 if gated else 1) * (-(-K // 512)) * 8 < 2 ** 31, what                                           # units x warps
        return
    assert p["t_tiles"] * tb >= T > (p["t_tiles"] - 1) * tb and p["kb"] * 128 >= K > (p["kb"] - 1) * 128, what
    c_tiles = p["tiles"] // p["t_tiles"]
    assert c_tiles * p["t_tiles"] == p["tiles"] < 2 ** 31 and c_tiles * per >= cols > (c_tiles - 1) * per, what
    if route == 1:
        parts, stage = p["parts"], (128 + tb) * 128
        assert tb in (16, 32, 64, 128) and 1 <= parts <= min(4, p["kb"]) and p["cluster"] == parts and p["grid"] == parts * p["tiles"], what
        cut = [r * p["kb"] // parts for r in range(parts + 1)]
        assert all(b > a for a, b in zip(cut, cut[1:])), what
        assert 1 <= stages <= 12 and stages * stage >= tb * 512, what                                                   # the sums lie in the stages
        assert 1023 + stages * stage + (2 * 12 + 1) * 8 + 8 + 4 * tb <= p["smem"], what                                 # alignment, barriers, slot and flag, scales
        assert p["smem"] >= 48 * 1024 and p["smem"] + 1024 > SM - (i8t_smem() + 1024), what                             # beside no pair of CTAs
        assert p["tiles"] * parts <= 128 or 2 * (p["smem"] + 1024) <= SM, what
    else:
        assert T > 128 and p["cluster"] == 2 and p["grid"] == 2 * min(74, p["tiles"]) and tb == 256 and per == (128 if gated else 256) and stages == 5, what
        assert 1023 + stages * 256 * 128 + 8 * 4096 + 8 * 1024 + (2 * 5 + 4) * 8 + 8 <= p["smem"], what


def i8t_smem():
    return product_plan(4096, 8192, 512, False)["smem"]


def test_plans_of_products():
    rng, seen = random.Random(1), set()
    for i in range(30000):
        T = rng.choice((1, 2, 3, 4, 5, 16, 17, 32, 33, 64, 65, 128, 129, sizes(rng, 1, 300), sizes(rng, 129, 70000)))
        K, N = sizes(rng, 1, int8.MAX_K), sizes(rng, 2, 400000)
        gated = rng.random() < 0.5
        hold_product(T, N + N % 2, K, gated)
        seen.add((product_plan(T, N + N % 2, K, gated)["route"], gated))
    assert len(seen) == 6
    for T in (129, 256, 300, 1000, 2500, 9472, 18944, 18945):             # at the border of 148 tiles of 128 rows
        edge = 148 // -(-T // 128)
        for n in (128 * edge - 1, 128 * edge, 128 * edge + 1, 64 * edge, 64 * edge + 1):
            for gated in (False, True):
                if n > 0:
                    hold_product(T, 2 * n if gated else n, 300, gated)


def layer_plan(T, D, F, E, k, shared, i8):
    out, places = (ctypes.c_int * 20)(), (ctypes.c_long * 7)()
    assert _native.cuda().inv_moe_few_plan(T, D, F, E, k, int(shared), int(i8), ctypes.addressof(out), ctypes.addressof(places)) == 0
    names = ("slots ld_act f_tiles d_tiles experts n_counters gate_steps down_steps down_per down_parts tb slices grid threads smem per_sm stages step cols tmem "
             "choice weight counters act sums bytes items").split()
    return dict(zip(names, list(out) + list(places)))


def hold_layer(T, D, F, E, k, shared, i8):
    p = layer_plan(T, D, F, E, k, shared, i8)
    what = (T, D, F, E, k, shared, i8, p)
    assert p["slots"] == T * (k + shared) and p["tb"] >= T and p["tb"] in (16, 32, 64), what
    assert p["f_tiles"] * 64 >= F > (p["f_tiles"] - 1) * 64 and p["d_tiles"] * 128 >= D > (p["d_tiles"] - 1) * 128 and F <= p["ld_act"] and p["ld_act"] % 8 == 0, what
    assert p["gate_steps"] * p["step"] >= D > (p["gate_steps"] - 1) * p["step"] and p["down_steps"] * p["step"] >= F > (p["down_steps"] - 1) * p["step"], what
    # every part of K has a step, none more than it may, and they make the whole
    parts = [min(p["down_per"], p["down_steps"] - i * p["down_per"]) for i in range(p["down_parts"])]
    assert all(1 <= n <= 12 for n in parts) and sum(parts) == p["down_steps"], what
    # places in the workspace, one behind the other
    need = [("choice", 4 * T * k, "weight"), ("weight", 4 * T * k, "counters"), ("counters", 4 * p["n_counters"], "act"), ("act", 2 * p["slots"] * p["ld_act"], "sums"),
            ("sums", 4 * p["down_parts"] * p["slots"] * D, "bytes")]
    assert all(p[a] % 256 == 0 and p[a] + n <= p[b] for a, n, b in need) and p["bytes"] == moe._few_bytes(T, D, F, E, k, shared, i8), what
    met = min(T * k, E) + shared
    assert p["experts"] == met and p["n_counters"] == 1 + met + p["d_tiles"], what
    assert p["items"] == met * (p["f_tiles"] + p["d_tiles"] * p["down_parts"]) + p["d_tiles"] * -(-T // 4) and 1 <= p["grid"] <= min(p["items"], 148 * p["per_sm"]), what
    static = 24 * 1024 if i8 else 12 * 1024
    assert p["smem"] <= SMEM - static + 12 * 1024 and p["per_sm"] * (p["smem"] + 12 * 1024 + 1024) <= SM, what
    assert 1 <= p["stages"] <= 12 and 1023 + p["stages"] * (128 * 128 + (2 if i8 else 1) * p["tb"] * 128) <= p["smem"] and p["threads"] >= 256, what
    assert p["cols"] <= p["tmem"] <= 512 // p["per_sm"] and p["tmem"] & (p["tmem"] - 1) == 0, what
    # slots and tokens in 16 and 8 bits
    assert p["slots"] < 2 ** 16 and p["slices"] in (1, 2, 4, 8), what


def test_plans_of_layers():
    rng = random.Random(2)
    for i in range(30000):
        i8 = rng.random() < 0.5
        grain = 16 if i8 else 8
        E = rng.choice((1, 2, 4, 8, 37, 64, 200, 256))
        hold_layer(rng.choice((1, 4, 16, 17, 32, 33, 64, rng.randint(1, 64))), grain * sizes(rng, 1, 2 ** 20 // grain), grain * sizes(rng, 1, 2 ** 18 // grain), E,
                   rng.randint(1, min(16, E)), rng.random() < 0.4, i8)


# ---------------------------------------------------------------------------------------------- guard values
PAGE = 4096


class Guarded:
    """Bytes between two stretches of a known value."""

    def __init__(self, n):
        self.n, self.all = n, torch.full((n + 2 * PAGE,), 0xA5, dtype=torch.uint8, device="cuda")
        self.all[PAGE:PAGE + n] = 0xFF                                     # NaN in every float type
        self.ptr = self.all.data_ptr() + PAGE

    def view(self, dtype, *shape):
        return self.all[PAGE:PAGE + self.n].view(dtype).view(*shape)

    def whole(self):
        return bool((self.all[:PAGE] == 0xA5).all()) and bool((self.all[PAGE + self.n:] == 0xA5).all())


def guarded_product(rng, T, N, K, f32, out_f32, bias, gated):
    g = torch.Generator(device="cuda").manual_seed(rng.randrange(1 << 30))
    wide, cols, dt = -(-K // 16) * 16, N // 2 if gated else N, F32 if f32 else BF
    x, q = Guarded(T * K * (4 if f32 else 2)), Guarded(N * wide)
    x.view(dt, T, K).copy_(torch.randn(T, K, device="cuda", generator=g).to(dt))
    q.view(torch.int8, N, wide)[:, :K] = torch.randint(-127, 128, (N, K), dtype=torch.int8, device="cuda", generator=g)
    sw, b, sx = Guarded(4 * N), Guarded(4 * N), Guarded(4 * T)
    sw.view(F32, N).copy_(torch.rand(N, device="cuda", generator=g) * K ** -0.5 / 73)
    b.view(F32, N).copy_(torch.randn(N, device="cuda", generator=g))
    out, codes = Guarded(T * cols * (4 if out_f32 else 2)), Guarded(T * wide)
    alone = T <= 4 and rt.lib().inv_int8_alone(T, N, K)
    rt.check(rt.lib().inv_int8_linear(int8._CALL(x.ptr, q.ptr, sw.ptr, b.ptr if bias else 0, out.ptr, 0 if alone else codes.ptr, 0 if alone else sx.ptr,
                                                 rt.status_ptr(x.all), rt.stream_ptr(), T, N, K, K, wide, cols, 0 if alone else wide, f32, out_f32, True, gated)), "inv_int8_linear")
    rt.check_status()
    what = (T, N, K, f32, out_f32, bias, gated)
    assert all(v.whole() for v in (x, q, sw, b, sx, out, codes)), what
    # Against 64 bits. Three roundings to fp32 of the sum and one of the whole: under 4 half steps of A = |sum| + |bias|, 2^-22 A. silu of g, |g| <= A: 1.1 of that, and
    # (6 + 1.16 A) 2^-23 A of its own; times up (|up| <= B, off by 2^-22 B) and rounded: A B (5.6 + 0.6 A) 2^-22 < A B (1 + A) 2^-19. The result's type adds a half step.
    xd = x.view(dt, T, K).double()
    s = (xd.abs().amax(1).float().clamp(min=1e-10).double() / 127).float().double().unsqueeze(1)
    y = torch.round(xd / s) @ q.view(torch.int8, N, wide)[:, :K].double().t() * s * sw.view(F32, N).double()
    size = y.abs()
    if bias:
        y, size = y + b.view(F32, N).double(), size + b.view(F32, N).double().abs()
    tol = 2.0 ** -22 * size
    if gated:
        (gate, up), (A, B) = y.chunk(2, 1), size.chunk(2, 1)
        y, tol = gate * torch.sigmoid(gate) * up, 2.0 ** -19 * A * B * (1 + A)
    got = out.view(F32 if out_f32 else BF, T, cols).double()
    assert torch.isfinite(got).all() and bool(((got - y).abs() <= 1.01 * tol + (2.0 ** -24 if out_f32 else 2.0 ** -8) * y.abs() + 1e-30).all()), what


@gpu
@pytest.mark.parametrize("seed", range(4))
def test_products_between_guards(seed):
    """Sizes drawn from a seed, odd ones among them; each form of the product in each type."""
    rng = random.Random(seed)
    for rows in ((1, 1), (2, 2), (3, 4), (5, 16), (17, 64), (65, 128), (129, 700)):
        for gated in (False, True):
            T, K, N = rng.randint(*rows), sizes(rng, 1, 1500), sizes(rng, 1, 1200) * 2
            K = K if rng.random() < 0.5 else -(-K // 16) * 16
            guarded_product(rng, T, N, K, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5, gated)
    for f32, gated in ((False, False), (True, False), (False, True), (True, True)):
        T = rng.randint(2300, 3100)
        cols = 128 * (150 * 128 // T + 2) // (2 if gated else 1) + rng.randint(0, 300)
        guarded_product(rng, T, 2 * cols if gated else cols, sizes(rng, 1, 500), rng.random() < 0.5, f32, rng.random() < 0.5, gated)


@gpu
@pytest.mark.parametrize("seed", range(4))
def test_layers_between_guards(seed):
    """The same sizes as a call that lays everything out by itself: alike to the last bit, nothing beside the result and the workspace written."""
    rng = random.Random(seed)
    for T in (1, rng.randint(2, 16), rng.randint(17, 32), rng.randint(33, 64)):
        for i8 in (False, True):
            grain = 16 if i8 else 8
            E, shared = rng.choice((1, 2, 8, 37, 64, 200)), rng.random() < 0.5
            D, F, k = grain * sizes(rng, 1, 600 // grain), grain * sizes(rng, 1, 900 // grain), rng.randint(1, min(16, E))
            g = torch.Generator(device="cuda").manual_seed(seed)

            def weight(*shape):
                w = torch.randn(*shape, device="cuda", generator=g) * shape[-1] ** -0.5
                return Int8Weight.quantize(w) if i8 else w.to(BF)
            x, router, res = (torch.randn(n, D, device="cuda", generator=g).to(BF) for n in (T, E, T))
            w, w2 = weight(E, 2 * F, D), weight(E, D, F)
            sh = (weight(2 * F, D), weight(D, F)) if shared else None
            want, counts = moe.moe_ffn_few(x, router, w, w2, res, k, sh)
            size = moe._few_bytes(T, D, F, E, k, shared, i8)
            out, work, c = Guarded(2 * T * D), Guarded(size), Guarded(4 * E)
            q = lambda v: v.q.data_ptr() if i8 else v.data_ptr()  # noqa: E731
            s = lambda v: v.scale.data_ptr() if i8 else 0  # noqa: E731
            a, b = sh or (None, None)
            rt.check(rt.lib().inv_moe_few(moe._FEW(x.data_ptr(), router.data_ptr(), res.data_ptr(), q(w), q(w2), s(w), s(w2), q(a) if sh else 0, q(b) if sh else 0,
                                                   s(a) if sh else 0, s(b) if sh else 0, out.ptr, c.ptr, work.ptr, rt.status_ptr(x), rt.stream_ptr(), T, D, F, E, k, D, D, i8,
                                                   size)), "inv_moe_few")
            rt.check_status()
            what = (T, D, F, E, k, shared, i8)
            assert out.whole() and work.whole() and c.whole(), what
            assert torch.equal(out.view(BF, T, D), want) and torch.equal(c.view(torch.int32, E), counts), what
            assert int(counts.sum()) == T * k, what


@gpu
def test_back_to_back_over_changing_states():
    """Hundreds of calls that nothing waits between, each form behind each other one, over inputs that change: what the last calls give is what they give alone."""
    g = torch.Generator(device="cuda").manual_seed(7)
    states = []
    for T, K, N, dt, gated in ((1, 640, 1000, BF, False), (2, 333, 514, F32, True), (4, 640, 1000, BF, False), (16, 1024, 2048, BF, True), (64, 1411, 1002, F32, False),
                               (200, 300, 900, BF, False), (2500, 128, 1026, F32, False), (2500, 200, 2052, BF, True)):
        for _ in range(3):
            x = torch.randn(T, K, device="cuda", generator=g).to(dt)
            w = Int8Weight.quantize(torch.randn(N, K, device="cuda", generator=g))
            states.append(lambda x=x, w=w, gated=gated: int8.int8_linear(x, w, gated=gated))
    for T, D, F, E, k, i8 in ((1, 256, 512, 8, 2, True), (7, 512, 176, 64, 6, False), (30, 256, 320, 8, 2, True), (64, 512, 256, 16, 4, False)):
        for _ in range(3):
            x, router = (torch.randn(n, D, device="cuda", generator=g).to(BF) for n in (T, E))
            w = [torch.randn(*s, device="cuda", generator=g) * s[-1] ** -0.5 for s in ((E, 2 * F, D), (E, D, F))]
            w = [Int8Weight.quantize(v) if i8 else v.to(BF) for v in w]
            states.append(lambda x=x, router=router, w=w, k=k: moe.moe_ffn_few(x, router, *w, x, k)[0])
    alone = []
    for run in states:
        alone.append(run())
        torch.cuda.synchronize()
    rng = random.Random(3)
    for _ in range(20):
        order = list(range(len(states))) * 3
        rng.shuffle(order)
        last = {i: states[i]() for i in order}
    torch.cuda.synchronize()
    rt.check_status()
    assert all(torch.equal(y, alone[i]) for i, y in last.items())
