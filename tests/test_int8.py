"""Products with weights and activations in 8-bit integers (ops.int8), against their definition in 64 bits.

Tolerances. The sum of code products is exact. Behind it stand the conversion of the sum to fp32, the product with the token's scale, and the product with the
channel's scale together with the bias, each off by at most half a step, 2^-24 of the value in hand: 3 * 2^-24 (|y - b|) + 2^-24 |b|. silu(g) = g / (1 + exp(-g)):
the exponential is off by at most 2 + 1.16 |g| units of 2^-23, the quotient by 2, the rest by one: (6 + 1.16 |g|) 2^-23, on top of what g's own error does, times
|silu'| <= 1.1. A bf16 result adds half a step of its own, 2^-8 of the value. The largest values carry a factor of two on all of this."""
import pytest
import torch

from innova_b200.ops import int8
from innova_b200.ops import runtime as rt
from innova_b200.ops.int8 import Int8Rows, Int8Weight, int8_linear, quantize_rows

gpu = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
E24 = 2.0 ** -24


def rows(T, K, dtype, seed=0, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, K, generator=g) * torch.exp(0.5 * torch.randn(K, generator=g))
    return x.to(dtype).to(device)


def weight(N, K, seed=1, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    q = torch.full((N, (K + 15) // 16 * 16), 77, dtype=torch.int8)           # what stands behind a row does not count
    q[:, :K] = torch.randint(-127, 128, (N, K), generator=g)
    s = torch.exp(0.3 * torch.randn(N, generator=g)) * K ** -0.5 / 73
    return Int8Weight(q.to(device)[:, :K], s.to(device))


def definition(x):
    """(codes, scales) of rows in 64 bits; 1e-10 is the fp32 number, and the scale is rounded to fp32 as it is stored."""
    s = (x.float().abs().amax(-1).clamp(min=1e-10).double() / 127).float()
    return torch.round(x.double() / s.double().unsqueeze(-1)), s


def expected(codes, s, w, bias=None, gated=False):
    """Result in 64 bits and how far it may be from it in fp32."""
    y = codes.double() @ w.q.double().t() * s.double().unsqueeze(-1) * w.scale.double()
    err = 3 * E24 * y.abs()
    if bias is not None:
        y, err = y + bias.double(), err + E24 * (bias.double().abs() + y.abs())
    if gated:
        g, u = y.chunk(2, -1)
        eg, eu = err.chunk(2, -1)
        silu = g * torch.sigmoid(g)
        es = 1.1 * eg + (6 + 1.16 * g.abs()) * 2 * E24 * silu.abs()
        y, err = silu * u, es * u.abs() + eu * silu.abs() + 2 * E24 * (silu * u).abs()
    return y, err


def close(out, y, err):
    tol = 2 * err + (2.0 ** -8 * y.abs() if out.dtype == BF else E24 * y.abs()) + 1e-30
    off = (out.double() - y).abs()
    assert torch.isfinite(out).all() and bool((off <= tol).all()), float((off / tol).max())


# ---------------------------------------------------------------------------------------------- rows
def ties(dtype):
    """Rows whose quotients lie on halves, one step beside them, and at the ends."""
    scale = torch.tensor([127.0, 254.0, 127.0 / 64, 127 * 2.0 ** 40, 127 * 2.0 ** -30])
    half = torch.arange(-126, 127).float() + 0.5
    body = torch.cat([half, half.to(dtype).float() * (1 + torch.finfo(dtype).eps), half * (1 - torch.finfo(dtype).eps), torch.tensor([127.0, -127.0, 0.0])])
    return (body * scale.unsqueeze(1) / 127).to(dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_are_rounded_halves_to_even(dtype):
    x = ties(dtype)
    r, (c, s) = quantize_rows(x), definition(x)
    assert torch.equal(r.scale, s) and torch.equal(r.q.double(), c)


def test_rows_small_zero_and_not_finite():
    x = torch.tensor([[0.0, 0, 0], [1e-12, -1e-11, 0], [1, float("nan"), 2], [float("inf"), 1, 2], [3, 2, 1]])
    r = quantize_rows(x)
    assert torch.equal(r.q[0], torch.zeros(3, dtype=torch.int8)) and float(r.scale[0]) == pytest.approx(1e-10 / 127)
    assert r.q[1].tolist() == [1, -13, 0]
    assert torch.isnan(r.scale[2]) and torch.isnan(r.scale[3]) and not r.q[2:4].any()
    w = weight(4, 3)
    y = int8_linear(x, w)
    assert torch.isnan(y[2:4]).all() and torch.isfinite(y[[0, 1, 4]]).all()


# ---------------------------------------------------------------------------------------------- products on the CPU
@pytest.mark.parametrize("dtype,bias,gated", [(F32, False, False), (F32, True, True), (BF, True, False), (BF, False, True)])
def test_linear_cpu(dtype, bias, gated):
    x, w = rows(7, 45, dtype), weight(22, 45)
    b = torch.randn(22).to(dtype) if bias else None
    y = int8_linear(x.view(7, 1, 45), w, b, gated=gated)
    assert y.shape == (7, 1, 11 if gated else 22) and y.dtype == dtype
    close(y[:, 0], *expected(*definition(x), w, b, gated))
    assert torch.equal(int8_linear(quantize_rows(x), w, b, dtype, gated), y[:, 0])
    assert int8_linear(quantize_rows(x), w).dtype == BF


def test_quantised_weight_is_near():
    w = rows(9, 50, F32)
    q = Int8Weight.quantize(torch.stack([w, 2 * w]))
    assert q.q.shape == (2, 9, 50) and q.scale.shape == (2, 9)
    assert bool(((q.dequantize() - torch.stack([w, 2 * w])).abs() <= q.scale.unsqueeze(-1) * 0.5000001).all())


def test_refusals():
    w = weight(6, 32)
    x = rows(2, 32, F32)
    with pytest.raises(ValueError, match="x of"):
        int8_linear(rows(2, 31, F32), w)
    with pytest.raises(TypeError, match="bf16 or fp32"):
        int8_linear(x.half(), w)
    with pytest.raises(TypeError, match="result"):
        int8_linear(x, w, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="bias"):
        int8_linear(x, w, torch.zeros(5))
    with pytest.raises(ValueError, match="pairs"):
        int8_linear(x, Int8Weight(w.q[:5], w.scale[:5]), gated=True)
    with pytest.raises(ValueError, match="weight of"):
        int8_linear(x, Int8Weight(w.q.float(), w.scale))
    with pytest.raises(ValueError, match="weight of"):
        int8_linear(x, Int8Weight(w.q, w.scale.double()))
    with pytest.raises(ValueError, match="32 bits"):
        int8_linear(torch.zeros(1, 140000), Int8Weight(torch.zeros(1, 140000, dtype=torch.int8), torch.ones(1)))
    with pytest.raises(ValueError, match="rows of"):
        int8_linear(Int8Rows(quantize_rows(x).q, torch.ones(3)), w)
    with pytest.raises(TypeError):
        quantize_rows(torch.ones(3, 4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no gradient"):
        int8_linear(x.clone().requires_grad_(), w)
    with torch.no_grad():
        int8_linear(x.clone().requires_grad_(), w)


def test_nothing_to_do():
    w = weight(6, 32)
    assert int8_linear(torch.zeros(0, 32), w).shape == (0, 6)
    empty = Int8Weight(torch.zeros(4, 0, dtype=torch.int8), torch.ones(4))
    assert torch.equal(int8_linear(torch.zeros(2, 0), empty, torch.arange(4.0)), torch.arange(4.0).expand(2, 4))


# ---------------------------------------------------------------------------------------------- on a GPU
@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_gpu(dtype):
    for x in (ties(dtype), rows(3, 1, dtype), rows(65, 1411, dtype), rows(5, 4096, dtype, 3), rows(2, 20000, dtype, 4)):
        r, (c, s) = quantize_rows(x.cuda()), definition(x)
        assert torch.equal(r.scale.cpu(), s) and torch.equal(r.q.cpu().double(), c)
    big = rows(9, 40, dtype)
    for view in (big[:, 1:37], big[1:, 3:], big[::2], big.t(), big.expand(2, 9, 40)):       # rows off 16-byte boundaries, apart, without unit stride
        r, (c, s) = quantize_rows(big.cuda().as_strided(view.shape, view.stride(), view.storage_offset())), definition(view)
        assert torch.equal(r.scale.cpu(), s) and torch.equal(r.q.cpu().double(), c)
    x = torch.tensor([[0.0] * 40, [1e-12] * 40, [1] * 39 + [float("nan")], [float("-inf")] + [1] * 39], dtype=dtype)
    r, c = quantize_rows(x.cuda()), quantize_rows(x)
    assert torch.equal(r.q.cpu(), c.q) and torch.equal(r.scale.cpu().nan_to_num(7), c.scale.nan_to_num(7))


@gpu
def test_scales_and_codes_of_all_sizes_gpu():
    """Scales are the nearest to a 127th over all exponents; codes of random and of nearly tied quotients are the definition's."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(1 << 20, 1, generator=g) * torch.exp2(torch.randint(-126, 127, (1 << 20, 1), generator=g).float())
    r, (c, s) = quantize_rows(x.cuda()), definition(x)
    assert torch.equal(r.scale.cpu(), s) and torch.equal(r.q.cpu().double(), c)
    x = torch.randn(64, 8192, generator=g)
    x[:, 0] = 127 * (1 + torch.rand(64, generator=g))                              # the largest: quotients n + 1/2 and their neighbours
    x[:, 1:4096] = ((torch.randint(-120, 120, (64, 4095), generator=g) + 0.5) * (x[:, :1] / 127) * (1 + torch.randint(-3, 4, (64, 4095), generator=g) * 2.0 ** -23))
    for rows_, many in ((x, False), (x.repeat(20, 1), True)):
        r, (c, s) = quantize_rows(rows_.cuda()), definition(rows_)
        assert torch.equal(r.scale.cpu(), s) and torch.equal(r.q.cpu().double(), c)


FEW = [1, 2, 8, 9, 16, 17, 32, 33, 63, 64]
MANY = [65, 100, 128, 129, 255, 257, 300, 600]
WIDE = [(1, 1), (16, 2), (17, 34), (40, 64), (127, 130), (128, 256), (129, 258), (512, 1000), (1411, 1002), (4096, 514)]


def product(T, K, N, dtype, out_dtype, bias, gated, seed=0):
    x, w = rows(T, K, dtype, seed), weight(N, K, seed + 1)
    b = None if bias is None else torch.randn(N, generator=torch.Generator().manual_seed(seed + 2)).to(bias)
    y = int8_linear(x.cuda(), Int8Weight(weight(N, K, seed + 1, "cuda").q, w.scale.cuda()), None if b is None else b.cuda(), out_dtype, gated)
    assert y.is_contiguous() and y.dtype == (out_dtype or dtype)
    rt.check_status()
    close(y.cpu(), *expected(*definition(x), w, b, gated))


@gpu
@pytest.mark.parametrize("T", FEW)
def test_linear_few_rows(T):
    for i, (K, N) in enumerate(WIDE):
        product(T, K, N, BF if i % 3 else F32, None, (None, BF, F32)[(i + T) % 3], i % 2 == 1, i)
        product(T, K, N, BF, F32, None, i % 2 == 0 and N % 2 == 0, i + 50)


@gpu
@pytest.mark.parametrize("T", MANY)
def test_linear_many_rows(T):
    for i, (K, N) in enumerate(WIDE):
        product(T, K, N, BF if i % 3 else F32, None, (None, BF, F32)[(i + T) % 3], i % 2 == 1, i)
        product(T, K, N, BF, F32, None, i % 2 == 0 and N % 2 == 0, i + 50)


@gpu
def test_linear_many_tiles_and_long_rows():
    product(3000, 200, 5000, BF, None, BF, False)
    product(3000, 200, 5000, BF, None, None, True)
    product(2, 30000, 70, BF, None, None, False)
    product(70, 30000, 70, BF, F32, None, False)


@gpu
def test_largest_sums():
    """127 * 127 * K just below 2^31, every sign alike."""
    K = int8.MAX_K // 16 * 16
    for T in (1, 70):
        x = torch.full((T, K), 3.0, device="cuda")
        w = Int8Weight(torch.full((4, K), 127, dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda"))
        w.q[1] = -127
        y = int8_linear(x, w).cpu().double()
        want = 127.0 * K * 3.0 * torch.tensor([1, -1, 1, 1], dtype=torch.float64)
        assert bool(((y - want).abs() <= 4 * E24 * want.abs()).all())


@gpu
@pytest.mark.parametrize("T", [5, 64, 200])
def test_rows_that_are_not_finite_stay_alone(T):
    x, w = rows(T, 256, BF).cuda(), weight(300, 256, device="cuda")
    fine = int8_linear(x, w)
    x[T // 2, 7], x[0, 0] = float("nan"), float("-inf")
    y = int8_linear(x, w)
    lost = torch.zeros(T, dtype=torch.bool)
    lost[[0, T // 2]] = True
    assert torch.isnan(y[lost]).all() and torch.equal(y[~lost], fine[~lost])


@gpu
def test_a_token_does_not_depend_on_its_company():
    x, w = rows(300, 1000, BF).cuda(), weight(777, 1000, device="cuda")
    y = int8_linear(x, w)
    for T in (1, 8, 20, 64, 65, 150):
        assert torch.equal(int8_linear(x[:T], w), y[:T])
        assert torch.equal(int8_linear(quantize_rows(x[:T]), w), y[:T])


@gpu
def test_linear_views_and_leading_dimensions():
    wide = rows(24, 200, BF).cuda()
    w = weight(96, 101, device="cuda")
    x = wide[:, 3:104]
    want = int8_linear(x.contiguous(), w)
    assert torch.equal(int8_linear(x, w), want)
    assert torch.equal(int8_linear(x.unflatten(0, (2, 3, 4)), w), want.view(2, 3, 4, 96))
    assert torch.equal(int8_linear(x.t().contiguous().t(), w), want)
    assert torch.equal(int8_linear(x[5], w), want[5])
    r = quantize_rows(x)
    assert torch.equal(int8_linear(Int8Rows(r.q.contiguous(), r.scale), w), want)      # rows of codes off 16-byte boundaries
    one = Int8Rows(r.q[3].expand(24, 101), r.scale[3].expand(24))                      # one row for all tokens
    assert torch.equal(int8_linear(one, w), want[3].expand(24, 96)) and torch.equal(int8_linear(x[3].expand(24, 101), w), want[3].expand(24, 96))
    with pytest.raises(ValueError, match="overlap"):
        int8_linear(x, Int8Weight(w.q[:1].expand(96, 101), w.scale))
    with pytest.raises(ValueError, match="16-byte"):
        int8_linear(x, Int8Weight(w.q.contiguous(), w.scale))
    with pytest.raises(ValueError, match="x on"):
        int8_linear(x.cpu(), w)


@gpu
def test_linear_streams_and_graphs():
    """Calls on two streams at once, and one captured and replayed on other inputs."""
    w = [weight(1000, 640, s, "cuda") for s in (1, 2)]
    x = [rows(T, 640, BF, T).cuda() for T in (20, 300)]
    want = [[int8_linear(a, b) for a in x] for b in w]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = [int8_linear(a, w[i]) for a in x]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in (0, 1) for a, b in zip(got[i], want[i]))
    still = [a.clone() for a in x]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ys = [int8_linear(a, w[0]) for a in still]
    for a in still:
        a.mul_(-0.75)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(y, int8_linear(a, w[0])) for y, a in zip(ys, still))
    rt.check_status()


@gpu
@pytest.mark.parametrize("T", [1, 2, 3, 4])
def test_up_to_four_rows(T):
    """Columns that do not fill the last CTA's share, slices of K that the warps share unevenly, more columns than one pass over the GPU takes."""
    for i, (K, N) in enumerate([(511, 888), (513, 6146), (1030, 2050), (4100, 1186), (5632, 592), (48, 160002), (16, 320006)]):
        product(T, K, N, (BF, F32)[i % 2], None, (None, F32, BF)[i % 3], False, i)
        product(T, K, N, BF, F32, (BF, None)[i % 2], True, i + 20)
    x, w = rows(4, 1030, BF).cuda(), weight(1200, 1030, device="cuda")
    fine = int8_linear(x[:T], w)
    assert torch.equal(int8_linear(quantize_rows(x[:T]), w), fine)
    x[T - 1, 1029] = float("nan")
    y = int8_linear(x[:T], w)
    assert torch.isnan(y[-1]).all() and torch.equal(y[:-1], fine[:-1])


@gpu
def test_one_row_and_a_large_weight():
    product(1, 4100, 9000, BF, None, BF, False)
    product(1, 4100, 9000, BF, None, None, True)


@gpu
@pytest.mark.parametrize("T", [1, 2, 4, 64, 300])
def test_weights_beyond_two_to_the_31(T):
    N, K = 66000, 32768
    w = Int8Weight(torch.randint(-127, 128, (N, K), dtype=torch.int8, device="cuda"), torch.rand(N, device="cuda") / 1000)
    x = rows(T, K, BF).cuda()
    y = int8_linear(x, w)
    g = int8_linear(x, w, gated=True)
    for a, b in ((0, 200), (N - 300, N)):                      # results are exact up to one rounding, however the rows are cut
        assert torch.equal(y[:, a:b], int8_linear(x, Int8Weight(w.q[a:b], w.scale[a:b])))
    half = N // 2
    few = Int8Weight(torch.cat([w.q[half - 100:half], w.q[N - 100:]]), torch.cat([w.scale[half - 100:half], w.scale[N - 100:]]))
    assert torch.equal(g[:, half - 100:], int8_linear(x, few, gated=True))
    rt.check_status()


@gpu
def test_clusters_beside_pairs():
    """Small clusters on one stream and tiles of CTA pairs on another: neither waits for tensor memory that the other holds."""
    few, many = rows(9, 128, BF).cuda(), rows(3000, 200, BF).cuda()
    w, v = weight(4096, 128, device="cuda"), weight(2050, 200, device="cuda")
    want = int8_linear(few, w), int8_linear(many, v)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(50):
        with torch.cuda.stream(streams[0]):
            got[0] += [int8_linear(few, w) for _ in range(4)]
        with torch.cuda.stream(streams[1]):
            got[1].append(int8_linear(many, v))
    torch.cuda.synchronize()
    rt.check_status()
    assert all(torch.equal(y, want[i]) for i in (0, 1) for y in got[i])


def test_the_longest_rows_hold_every_code():
    """-128 in rows of the caller's own and in weights: the longest K that is taken has sums below 2^31, the next is refused."""
    assert 128 * 128 * int8.MAX_K < 2 ** 31 <= 128 * 128 * (int8.MAX_K + 1)
    K = 131200
    with pytest.raises(ValueError, match="32 bits"):
        int8_linear(torch.ones(1, K), Int8Weight(torch.full((1, K), -128, dtype=torch.int8), torch.ones(1)))


@gpu
@pytest.mark.parametrize("T", [1, 2, 4, 20, 70])
def test_largest_sums_of_every_code(T):
    K = int8.MAX_K // 16 * 16
    w = Int8Weight(torch.full((4, K), -128, dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda"))
    w.q[1] = 127
    x = Int8Rows(torch.full((T, K), -128, dtype=torch.int8, device="cuda"), torch.ones(T, device="cuda"))
    y = int8_linear(x, w, out_dtype=F32).cpu().double()
    want = 128.0 * K * torch.tensor([128, -127, 128, 128], dtype=torch.float64)
    assert bool(((y - want).abs() <= 2 * E24 * want.abs()).all())            # one conversion to fp32; scales of one
    rt.check_status()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_nothing_to_add_up_behind_leading_dimensions(device):
    b = torch.arange(4.0, device=device)
    w = Int8Weight(torch.zeros(4, 0, dtype=torch.int8, device=device), torch.ones(4, device=device))
    x = torch.zeros(2, 3, 0, device=device)
    assert torch.equal(int8_linear(x, w, b), b.expand(2, 3, 4)) and not int8_linear(x, w).any()
    assert torch.equal(int8_linear(x, w, b, gated=True), (torch.nn.functional.silu(b[:2]) * b[2:]).expand(2, 3, 2))
    assert torch.equal(int8_linear(quantize_rows(x), w, b, F32), b.expand(2, 3, 4))
    v = weight(6, 32, device=device)
    for shape in ((0, 5, 32), (3, 0, 32), (0, 32)):
        assert int8_linear(torch.zeros(shape, device=device), v).shape == (*shape[:-1], 6)


@pytest.mark.parametrize("size", [1e36, 1e-9])
@pytest.mark.parametrize("T", [1, 3, 20, 200, 3000])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_rows_of_any_size(size, T, device):
    """Results that fp32 holds, though a sum of codes times the token's scale is beyond it."""
    K, N = 64, (2050 if T == 3000 else 66)
    x, w = rows(T, K, F32) * size, weight(N, K)
    assert float((127 * 73 * K ** 0.5) * x.abs().amax() / 127) > (2.0 ** 128 if size > 1 else 0)
    y = int8_linear(x.to(device), Int8Weight(weight(N, K, device=device).q, w.scale.to(device)))
    if device == "cuda":
        rt.check_status()
    want, err = expected(*definition(x), w)
    assert float(want.abs().max()) < 2.0 ** 127
    close(y.cpu(), want, err)


def test_sizes_beyond_32_bits_are_refused():
    """By the entries, before they ask for a device: no pointer is looked at."""
    from innova_b200 import _native
    lib, bad = _native.cuda(), -7
    at = 1 << 20
    call = lambda T, N, K: int8._CALL(at, at, at, 0, at, at, at, at, 0, T, N, K, K, (K + 15) // 16 * 16, N, (K + 15) // 16 * 16, 0, 0, 0, 0)  # noqa: E731
    assert lib.inv_int8_rows(call(1, 0, 2 ** 32 + 5)) == bad and lib.inv_int8_rows(call(2 ** 31, 0, 8)) == bad
    for T, N, K in ((2 ** 31, 16, 16), (16, 2 ** 31, 16), (16, 16, 131072), (2 ** 32 + 1, 16, 16)):
        assert lib.inv_int8_linear(call(T, N, K)) == bad


def test_scales_that_ask_for_gradients_are_refused():
    w, x = weight(6, 32), rows(2, 32, F32)
    r = quantize_rows(x)
    with pytest.raises(RuntimeError, match="no gradient"):
        int8_linear(x, Int8Weight(w.q, w.scale.clone().requires_grad_()))
    with pytest.raises(RuntimeError, match="no gradient"):
        int8_linear(Int8Rows(r.q, r.scale.clone().requires_grad_()), w)


def test_which_products_go_through_tiles():
    """What the tests below mean to reach."""
    import ctypes
    from innova_b200 import _native
    out = (ctypes.c_int * 13)()
    for T, N, gated, route in ((3001, 2050, 0, 2), (2500, 2052, 1, 2), (2500, 896, 0, 1), (2500, 897, 0, 2), (2500, 896, 1, 1), (2500, 898, 1, 2), (128, 1 << 20, 0, 1), (129, 9473, 0, 2)):
        assert _native.cuda().inv_int8_plan(T, N, 101, gated, ctypes.addressof(out)) == 0 and out[0] == route


@gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype,out_dtype", [(BF, BF), (F32, F32), (BF, F32), (F32, BF)])
def test_tiles(dtype, out_dtype, gated):
    """Both results' boxes and rows off 16-byte boundaries, biases of both types, ends of K, of rows and of columns."""
    for i, (T, K, N) in enumerate([(3001, 101, 2050), (2500, 129, 2052), (2561, 384, 4096), (2700, 257, 2064), (2400, 40, 3002)]):
        product(T, K, N, dtype, out_dtype, (BF, F32, None)[(i + gated) % 3], gated, i)
        product(T, K, N, dtype, out_dtype, (F32, None, BF)[(i + gated) % 3], gated, i + 10)


@gpu
@pytest.mark.parametrize("gated", [False, True])
def test_on_both_sides_of_the_tiles_border(gated):
    for T, N in ((2500, 896), (2500, 898), (129, 9472), (129, 9474), (300, 6272), (300, 6400)):
        product(T, 200, N, BF, F32, F32, gated)
        product(T, 77, N, F32, BF, None, gated, 3)
    x, w = rows(2500, 200, BF).cuda(), weight(898, 200, device="cuda")
    y = int8_linear(x, w)                                                    # tiles
    assert torch.equal(int8_linear(x[:300], w), y[:300]) and torch.equal(int8_linear(x[-7:], w), y[-7:])      # a cluster's
