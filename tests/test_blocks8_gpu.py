"""8-bit block operators on the GPU against their definitions in 64 bits (written here, apart from the package)."""
import math

import pytest
import torch

from trenowanie_generatora_obrazkow_b200.ops import blocks8 as B8
from trenowanie_generatora_obrazkow_b200.ops._ext import check_errors, ext

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(autouse=True)
def _no_kernel_errors():
    yield
    if torch.cuda.is_available():
        check_errors(DEV)


def rnd(*shape, seed=0, std=1.0, spread=0.5, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(*shape, device=DEV, generator=g) * std
    return (x * torch.exp(torch.randn(shape[-1], device=DEV, generator=g) * spread)).to(dtype)


def held(x):
    """The values that 8 bits hold of x [M, K] with blocks along the rows, in 64 bits."""
    x = x.detach().double()
    M, K = x.shape
    nb = -(-K // 128)
    v = torch.nn.functional.pad(x, (0, nb * 128 - K)).view(M, nb, 128)
    fin = v.isfinite()
    top = torch.where(fin, v.abs(), 0.0).amax(-1, keepdim=True)
    e = torch.full_like(top, -127.0)
    for k in range(-127, 121):  # the smallest whole e with top <= 448 2^e
        e = torch.where(top > 448 * 2.0 ** (k - 1), max(k, -127), e) if k > -127 else e
    u = v / torch.exp2(e)
    p = torch.frexp(u.abs().clamp_min(2.0 ** -6))[1] - 1  # e4m3: 3 bits behind the leading one, steps of 2^-9 at least
    step = torch.exp2((p - 3).double())
    q = torch.round(u / step) * step * torch.exp2(e)
    return torch.where(fin, q, math.nan).view(M, nb * 128)[:, :K]


def held_t(x):
    return held(x.t()).t()


HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def product_tol(a, b, dtype, y):
    """|error| of a product of held values a [M, K], b [N, K]: the tensor core adds 32 products at a time to an fp32 sum and
    drops bits below 2^-23 of the largest term in each step (one for the 32 terms, one for the sum), so 2^-22 S a step
    with S = sum |a b|; parts of 4096 (128 steps) join in fp32 for fp32 results, other sums run through."""
    S = a.abs() @ b.abs().t()
    steps = -(-a.shape[1] // 32)
    if dtype == torch.float32:
        steps = min(steps, 128) + -(-a.shape[1] // 4096)
    return S * (steps + 2) * 2.0 ** -22 + y.abs() * HALF[dtype] + TINY[dtype]


def assert_within(got, want, tol):
    assert got.shape == want.shape
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    worst = (err / tol).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the tolerance"


# ------------------------------------------------------------------------------------------------------------ packing
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 100), (128, 128), (129, 513), (300, 1000), (77, 777), (256, 640)])
def test_pack_and_unpack(M, K, dtype):
    x = rnd(M, K, dtype=dtype, seed=M + K)
    r, c = B8.quantize_blocks(x, "both")
    assert r.shape == (M, K) and c.shape == (K, M)
    assert torch.equal(B8.dequantize_blocks(r, torch.float32).double(), held(x))
    assert torch.equal(B8.dequantize_blocks(c, torch.float32).double(), held_t(x).t())
    for one, two in ((B8.quantize_blocks(x), r), (B8.quantize_blocks(x, "cols"), c)):
        assert torch.equal(one.codes.view(torch.uint8), two.codes.view(torch.uint8)) and torch.equal(one.scales, two.scales)
    # the bytes are those of the CPU's definition, padding included
    for got, want in ((r, B8.quantize_blocks(x.cpu())), (c, B8.quantize_blocks(x.cpu(), "cols"))):
        assert torch.equal(got.scales.cpu(), want.scales)
        assert torch.equal(got.codes.cpu().view(torch.uint8) & 0x7f, want.codes.view(torch.uint8) & 0x7f)  # but -0


@pytest.mark.parametrize("dtype", TYPES)
def test_pack_special_values(dtype):
    x = rnd(130, 260, dtype=dtype, seed=3)
    top = torch.finfo(dtype).max
    x[0] = 0
    x[1, 5], x[1, 200] = math.nan, math.inf
    x[2, :] = -math.inf
    x[3, 7] = top
    x[4, :] = torch.finfo(dtype).tiny
    x[5, 9] = -0.0
    x[:, 11] = 0
    x[6, 0:128] = 448.0
    x[7, 0:128] = 449.0
    x[8, 130] = math.nan
    for side, want in (("rows", held(x)), ("cols", held_t(x).t())):
        got = B8.dequantize_blocks(B8.quantize_blocks(x, side), torch.float32)
        want = want.float()  # the largest bf16 and fp32 round up to 2^128 in 8 bits, which fp32 shows as infinity
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


def test_pack_reads_strided_rows_in_place_and_copies_others():
    big = rnd(200, 1000, seed=5)
    for x in (big[:, 3:259], big[10:150:2, 8:520], big.t(), big[:, ::2], big[:1].expand(50, 1000)):
        got = B8.dequantize_blocks(B8.quantize_blocks(x), torch.float32)
        assert torch.equal(got.double(), held(x))


def test_pack_of_no_rows():
    x = torch.empty(0, 300, device=DEV, dtype=torch.bfloat16)
    r, c = B8.quantize_blocks(x, "both")
    assert r.shape == (0, 300) and c.shape == (300, 0)
    assert B8.dequantize_blocks(r).shape == (0, 300) and B8.dequantize_blocks(c).shape == (300, 0)


# ----------------------------------------------------------------------------------------------------------- products
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(128, 128, 128), (128, 256, 512), (1, 1, 1), (7, 33, 100), (129, 257, 513), (300, 777, 1000),
                                   (333, 96, 640), (64, 128, 4480), (250, 130, 9000)])
def test_gemm(M, N, K, dtype):
    a, b = rnd(M, K, seed=1, dtype=torch.float32), rnd(N, K, seed=2, std=K ** -0.5, dtype=torch.float32)
    qa, qb = held(a), held(b)
    want = qa @ qb.t()
    got = B8.gemm_blocks(B8.quantize_blocks(a), B8.quantize_blocks(b), dtype=dtype)
    assert got.dtype == dtype
    assert_within(got, want, product_tol(qa, qb, dtype, want))


@pytest.mark.parametrize("M,N,K", [(2500, 4096, 256), (4000, 2570, 384), (2048, 5504, 1280)])
def test_gemm_of_many_tiles(M, N, K):
    a, b = rnd(M, K, seed=3, dtype=torch.float32), rnd(N, K, seed=4, dtype=torch.float32)
    qa, qb = held(a), held(b)
    want = qa @ qb.t()
    for dtype in (torch.bfloat16, torch.float32):
        got = B8.gemm_blocks(B8.quantize_blocks(a), B8.quantize_blocks(b), dtype=dtype)
        assert_within(got, want, product_tol(qa, qb, dtype, want))


def test_gemm_sums_of_one_sign():
    """Long sums of positive products: what the tensor core drops does not add up past the parts of 4096."""
    K = 32768
    a, b = rnd(256, K, seed=5, spread=0).abs(), rnd(128, K, seed=6, spread=0).abs()
    qa, qb = held(a), held(b)
    want = qa @ qb.t()
    got = B8.gemm_blocks(B8.quantize_blocks(a), B8.quantize_blocks(b), dtype=torch.float32)
    assert ((got.double() - want).norm() / want.norm()).item() < 128 * 2.0 ** -24  # a part's 128 steps, half a step each


@pytest.mark.parametrize("N", [64, 61])
def test_gemm_into_out(N):
    a, b = rnd(70, 5000, seed=7), rnd(N, 5000, seed=8)
    A, Bb = B8.quantize_blocks(a), B8.quantize_blocks(b)
    qa, qb = held(a), held(b)
    want = qa @ qb.t()
    tol = product_tol(qa, qb, torch.float32, want)
    big = torch.full((70, 200), 3.0, device=DEV)
    out = big[:, 40:40 + N]
    assert B8.gemm_blocks(A, Bb, out=out) .data_ptr() == out.data_ptr()
    assert_within(out, want, tol)
    B8.gemm_blocks(A, Bb, out=out, accumulate=True)
    assert_within(out, 2 * want, 2 * tol + 2 * want.abs() * 2.0 ** -23)
    assert (big[:, :40] == 3).all() and (big[:, 40 + N:] == 3).all()
    bias = rnd(N, seed=9, dtype=torch.float32)
    got = B8.gemm_blocks(A, Bb, bias=bias, dtype=torch.float32)
    assert_within(got, want + bias.double(), tol + (want + bias.double()).abs() * 2.0 ** -23)


def test_gemm_is_deterministic():
    a, b = rnd(512, 20000, seed=10), rnd(512, 20000, seed=11)
    A, Bb = B8.quantize_blocks(a), B8.quantize_blocks(b)
    first = B8.gemm_blocks(A, Bb, dtype=torch.float32)
    for _ in range(3):
        assert torch.equal(first, B8.gemm_blocks(A, Bb, dtype=torch.float32))


# ------------------------------------------------------------------------------------------------------------- linear
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 5, 8, 9, 16, 17, 130])
@pytest.mark.parametrize("N,K,bias", [(48, 128, False), (33, 100, True), (1, 1, True), (777, 1000, True), (96, 1290, False)])
def test_linear_frozen(M, N, K, bias, dtype):
    x, w = rnd(M, K, seed=M, dtype=dtype), rnd(N, K, seed=1, std=K ** -0.5, dtype=torch.float32)
    b = rnd(N, seed=2, dtype=torch.float32) if bias else None
    qx, qw = held(x), held(w)
    want = qx @ qw.t() + (b.double() if bias else 0)
    got = B8.linear_blocks(x, B8.quantize_blocks(w), b)
    assert got.dtype == dtype
    assert_within(got, want, product_tol(qx, qw, dtype, want) + want.abs() * 2.0 ** -22)


def train_linear(x, w, b, dy, fn=B8.linear_blocks):
    leaves = [t.detach().clone().requires_grad_() for t in (x, w)] + ([b.detach().clone().requires_grad_()] if b is not None else [])
    y = fn(*leaves)
    y.backward(dy)
    return [y.detach()] + [t.grad for t in leaves]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K,bias", [(1, 16, 128, True), (77, 96, 128, False), (130, 777, 100, True), (513, 128, 1000, True),
                                        (5000, 64, 72, True), (4000, 2600, 1500, False), (12000, 700, 2048, True)])
def test_linear_gradients(M, N, K, bias, dtype):
    x, w, dy = rnd(M, K, seed=1, dtype=dtype), rnd(N, K, seed=2, std=K ** -0.5, dtype=torch.float32), rnd(M, N, seed=3, std=0.1, dtype=dtype)
    b = rnd(N, seed=4, dtype=torch.float32) if bias else None
    got = train_linear(x, w, b, dy)
    y = held(x) @ held(w).t() + (b.double() if bias else 0)
    assert_within(got[0], y, product_tol(held(x), held(w), dtype, y) + y.abs() * 2.0 ** -22)
    dx = held(dy) @ held_t(w)
    assert_within(got[1], dx, product_tol(held(dy), held_t(w).t(), dtype, dx))
    dw = held_t(dy).t() @ held_t(x)
    assert got[2].dtype == torch.float32
    assert_within(got[2], dw, product_tol(held_t(dy).t(), held_t(x).t(), torch.float32, dw))
    if bias:  # fp32 sums of at most 128 rows, then of the tiles: each step half a unit of the running sum
        db = dy.double().sum(0)
        assert_within(got[3], db, dy.double().abs().sum(0) * (16 + M / 128) * 2.0 ** -24 + 1e-30)


def test_linear_gradient_against_differences():
    """Where packing is exact (small whole numbers), the operator is linear and its gradient is that of differences."""
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randint(-7, 8, (130, 260), device=DEV, generator=g).float()
    w = torch.randint(-7, 8, (72, 260), device=DEV, generator=g).float()
    dy = torch.randint(-7, 8, (130, 72), device=DEV, generator=g).float()
    y, dx, dw = train_linear(x, w, None, dy)
    f = lambda x_, w_: (B8.linear_blocks(x_, w_).double() * dy.double()).sum()  # noqa: E731
    for _ in range(5):
        i, j, k = (int(torch.randint(0, n, (1,), generator=torch.Generator().manual_seed(_ + n))) for n in (130, 260, 72))
        d = torch.zeros_like(x)
        d[i, j] = 1
        assert (f(x + d, w) - f(x - d, w)).item() / 2 == dx[i, j].item()
        d = torch.zeros_like(w)
        d[k, j] = 1
        assert (f(x, w + d) - f(x, w - d)).item() / 2 == dw[k, j].item()


@pytest.mark.parametrize("wtype", [torch.bfloat16, torch.float16])
def test_linear_of_16_bit_weights(wtype):
    x, w, dy = rnd(200, 256, seed=1), rnd(96, 256, seed=2, std=1 / 16, dtype=wtype), rnd(200, 96, seed=3)
    got = train_linear(x, w, None, dy)
    dw = held_t(dy).t() @ held_t(x)
    assert got[2].dtype == wtype
    assert_within(got[2], dw, product_tol(held_t(dy).t(), held_t(x).t(), wtype, dw))


def test_linear_leading_dims_module_and_accumulation():
    lin = torch.nn.Linear(256, 96, device=DEV)
    x = rnd(2, 65, 256, seed=1).requires_grad_()
    y = B8.linear_blocks(x, lin)
    assert y.shape == (2, 65, 96)
    dy = rnd(2, 65, 96, seed=2)
    y.backward(dy)
    first = lin.weight.grad.clone(), lin.bias.grad.clone()
    B8.linear_blocks(x, lin).backward(dy)
    assert torch.equal(lin.weight.grad, 2 * first[0]) and torch.equal(lin.bias.grad, 2 * first[1])
    flat = train_linear(x.detach().view(130, 256), lin.weight, lin.bias, dy.view(130, 96))
    assert torch.equal(flat[2], first[0]) and torch.equal(flat[3], first[1])


def test_linear_parts_of_the_gradient():
    x, w, dy = rnd(200, 256, seed=1), rnd(96, 256, seed=2, dtype=torch.float32), rnd(200, 96, seed=3)
    b = rnd(96, seed=4, dtype=torch.float32)
    _, dx, dw, db = train_linear(x, w, b, dy)
    for want_x in (False, True):
        for want_w in (False, True):
            for want_b in (False, True):
                if not (want_x or want_w or want_b):
                    continue
                xi, wi, bi = (t.clone().requires_grad_(r) for t, r in ((x, want_x), (w, want_w), (b, want_b)))
                B8.linear_blocks(xi, wi, bi).backward(dy)
                for t, want, full in ((xi, want_x, dx), (wi, want_w, dw), (bi, want_b, db)):
                    assert (t.grad is None) if not want else torch.equal(t.grad, full)


def test_linear_weight_used_twice_and_not_a_leaf():
    x, w, dy = rnd(200, 128, seed=1), rnd(128, 128, seed=2, std=0.1, dtype=torch.float32), rnd(200, 128, seed=3)
    wi = w.clone().requires_grad_()
    h = B8.linear_blocks(x, wi)
    B8.linear_blocks(h, wi).backward(dy)
    h0 = B8.linear_blocks(x, w)
    dw2 = train_linear(h0, w, None, dy)
    dw1 = train_linear(x, w, None, dw2[1])
    assert torch.allclose(wi.grad, dw1[2] + dw2[2], rtol=1e-6, atol=0)
    base = w.clone().requires_grad_()
    B8.linear_blocks(x, base * 2.0).backward(dy)
    assert torch.equal(base.grad, 2 * train_linear(x, 2 * w, None, dy)[2])


def test_linear_of_no_rows():
    lin = torch.nn.Linear(256, 96, device=DEV)
    x = torch.empty(0, 256, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = B8.linear_blocks(x, lin)
    assert y.shape == (0, 96)
    y.sum().backward()
    assert x.grad.shape == (0, 256) and (lin.weight.grad == 0).all() and (lin.bias.grad == 0).all()
    assert B8.linear_blocks(x.detach(), B8.quantize_blocks(lin.weight)).shape == (0, 96)


# ------------------------------------------------------------------------------------------------------------- SwiGLU
def swiglu64(ab):
    a, b = ab.double().chunk(2, dim=1)
    return a * torch.sigmoid(a) * b


def swiglu_grad64(ab, dg):
    a, b = ab.double().chunk(2, dim=1)
    s, dg = torch.sigmoid(a), dg.double()
    return torch.cat([dg * b * (s + a * s * (1 - s)), dg * a * s], dim=1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,H", [(1, 1), (3, 128), (77, 1408), (130, 100), (129, 333), (300, 1536)])
def test_swiglu(M, H, dtype):
    ab = rnd(M, 2 * H, seed=1, dtype=dtype, std=2.0).requires_grad_()
    dg = rnd(M, H, seed=2, dtype=dtype)
    g = B8.swiglu_blocks(ab)
    want = swiglu64(ab.detach())
    # the exponential is within 2^-19 for |a| < 32 in 16 bits (2 ulp + 2^-21 |a|), 2^-21 in fp32, and a few roundings
    fine = 2.0 ** -20 if dtype == torch.float32 else 2.0 ** -15
    assert_within(g, want, want.abs() * (HALF[dtype] + fine) + TINY[dtype])
    assert torch.equal(g.detach(), B8.swiglu_blocks(ab.detach()))
    g.backward(dg)
    q = torch.cat([held(v) for v in ab.detach().chunk(2, dim=1)], dim=1)
    d = swiglu_grad64(q, dg)
    a, b = q.chunk(2, dim=1)
    parts = torch.cat([dg.double() * b * (1 + a.abs()), dg.double() * a], dim=1).abs()  # 1 + a (1 - s) may cancel
    assert_within(ab.grad, d, d.abs() * HALF[dtype] + parts * fine + TINY[dtype])


# ---------------------------------------------------------------------------------------------------------------- MLP
def mlp64(x, w1, w2, dy, dtype):
    ab = (held(x) @ held(w1).t()).to(dtype)
    g = swiglu64(ab)
    y = held(g) @ held(w2).t()
    dg = (held(dy) @ held_t(w2)).to(dtype)
    dab = swiglu_grad64(held(ab), dg)
    return [y, held(dab) @ held_t(w1), held_t(dab).t() @ held_t(x), held_t(dy).t() @ held_t(g)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,H", [(1, 128, 128), (77, 100, 256), (333, 512, 1408), (1000, 576, 384)])
def test_mlp(M, K, H, dtype):
    x, w1, w2 = rnd(M, K, seed=1, dtype=dtype), rnd(2 * H, K, seed=2, std=K ** -0.5, dtype=torch.float32, spread=0), \
        rnd(K, H, seed=3, std=H ** -0.5, dtype=torch.float32, spread=0)
    dy = rnd(M, K, seed=4, std=0.1, dtype=dtype)
    want = mlp64(x, w1, w2, dy, dtype)
    leaves = [t.clone().requires_grad_() for t in (x, w1, w2)]
    y = B8.mlp_blocks(*leaves)
    y.backward(dy)
    # A value that the operator computes (a, b, g, their gradients) and that lies next to a border of its 8 bits may fall
    # on the other side: one step of e4m3, 2^-3 of it, for about one value in 2^-8 / 2^-3 of those whose 16-bit form (fp32: a
    # few 2^-24) also flipped. As shares: 2^-8 / 2^-24 ... far below 2^-7 of all, so the 2-norm is off by less than
    # 2^-3 sqrt(2^-7) < 2 %, and by half a step of the result's own type.
    for got, w in zip([y.detach()] + [t.grad for t in leaves], want):
        assert got.shape == w.shape
        assert ((got.double() - w).norm() / w.norm()).item() < 0.02
    assert torch.equal(y.detach(), B8.mlp_blocks(x, w1, w2))


def test_mlp_is_its_parts():
    """The forward and the weight gradient of the second product, from the operators on their own."""
    x, w1, w2 = rnd(200, 256, seed=1, dtype=torch.float32), rnd(512, 256, seed=2, std=1 / 16, dtype=torch.float32), \
        rnd(96, 256, seed=3, std=1 / 16, dtype=torch.float32)
    ab = B8.linear_blocks(x, w1)
    g = B8.swiglu_blocks(ab)
    y = B8.linear_blocks(g, w2)
    assert torch.equal(y, B8.mlp_blocks(x, w1, w2))  # fp32: g is not rounded on the way


def test_mlp_of_other_widths_and_no_rows():
    x, w1, w2 = rnd(50, 64, seed=1), rnd(200, 64, seed=2, dtype=torch.float32), rnd(64, 100, seed=3, dtype=torch.float32)
    assert torch.equal(B8.mlp_blocks(x, w1, w2), B8.linear_blocks(B8.swiglu_blocks(B8.linear_blocks(x, w1)), w2))
    leaves = [torch.empty(0, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True),
              rnd(256, 64, seed=2, dtype=torch.float32).requires_grad_(), rnd(64, 128, seed=3, dtype=torch.float32).requires_grad_()]
    y = B8.mlp_blocks(*leaves)
    y.sum().backward()
    assert y.shape == (0, 64) and all((t.grad == 0).all() for t in leaves[1:]) and leaves[0].grad.shape == (0, 64)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,H", [(40, 192, 128), (333, 1540, 384)])
def test_mlp_of_overflowing_activations(M, K, H, dtype):
    """One value of a is beyond its type: it is NaN in 8 bits, in y's row, dx's row, two rows of dW1 and a column of dW2."""
    r, h = M - 5, H - 3
    s_x, s_w = (200.0, 1e4) if dtype == torch.float16 else (1e12, 1e30)  # a b stays finite in fp32, a[r, h] does not
    x, w1, w2 = rnd(M, K, seed=1, dtype=torch.float32, spread=0), rnd(2 * H, K, seed=2, std=K ** -0.5, dtype=torch.float32, spread=0), \
        rnd(96, H, seed=3, std=H ** -0.5, dtype=torch.float32, spread=0)
    w1[h] = x[r] * s_w / K  # a[r, h] = s_x s_w
    x[r] *= s_x
    x, dy = x.to(dtype), rnd(M, 96, seed=4, std=0.1, dtype=dtype, spread=0)
    want = mlp64(x, w1, w2, dy, dtype)
    leaves = [t.clone().requires_grad_() for t in (x, w1, w2)]
    y = B8.mlp_blocks(*leaves)
    y.backward(dy)
    nan = [torch.zeros(t.shape, dtype=torch.bool, device=DEV) for t in want]
    nan[0][r] = nan[1][r] = nan[2][h] = nan[2][H + h] = True
    nan[3][:, h] = True
    for got, w, n in zip([y.detach()] + [t.grad for t in leaves], want, nan):
        assert torch.equal(w.isnan(), n) and torch.equal(got.isnan(), n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,H", [(1, 64, 128), (17, 100, 128), (129, 100, 384), (384, 1540, 256)])
def test_mlp_gives_the_same_whatever_it_keeps(M, K, H, dtype):
    """The forms that write a checkpoint, g's columns, both or neither agree to the bit, as do those of weights held in 8 bits."""
    x, w1, w2 = rnd(M, K, seed=1, dtype=dtype), rnd(2 * H, K, seed=2, std=K ** -0.5, dtype=torch.float32), \
        rnd(96, H, seed=3, std=H ** -0.5, dtype=torch.float32)
    dy = rnd(M, 96, seed=4, std=0.1, dtype=dtype)
    every = None
    for wants in [(1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 0, 0)]:
        leaves = [t.clone().requires_grad_(bool(w)) for t, w in zip((x, w1, w2), wants)]
        y = B8.mlp_blocks(*leaves)
        if any(wants):
            y.backward(dy)
        got = [y.detach()] + [t.grad for t in leaves]
        every = every or got
        for a, b in zip(got, every):
            assert a is None or torch.equal(a, b)
    if M > 16:  # fewer rows are summed in another order
        assert torch.equal(every[0], B8.mlp_blocks(x, B8.quantize_blocks(w1), B8.quantize_blocks(w2)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,H", [(300, 640, 384), (1000, 256, 1408)])
def test_mlp_rows_are_those_of_its_parts(M, K, H, dtype):
    x, w1, w2 = rnd(M, K, seed=1, dtype=dtype), rnd(2 * H, K, seed=2, std=K ** -0.5, dtype=torch.float32), \
        rnd(96, H, seed=3, std=H ** -0.5, dtype=torch.float32)
    a, b = B8.linear_blocks(x, w1).float().chunk(2, 1)
    g = a * torch.sigmoid(a) * b
    y = B8.gemm_blocks(B8.quantize_blocks(g), B8.quantize_blocks(w2), dtype=dtype)
    # g may be off by a few 2^-24 of itself, 2^-21 at most; e4m3's borders are at least 2^-4 of a value apart, so one value in
    # 2^-4 / 2^-20 = 2^16 falls on another side, and of the rows of H values at most one in 2^16 / H (2 %) is touched
    same = (y == B8.mlp_blocks(x, w1, w2)).all(1).double().mean().item()
    assert same > 0.9


@pytest.mark.parametrize("before", [False, True])
def test_mlp_of_one_weight_twice(before):
    """in_proj and out_proj the same parameter: its gradient is the sum of both, added to what was there."""
    H = 128
    x, w, dy = rnd(70, H, seed=1), rnd(2 * H, H, seed=2, std=H ** -0.5, dtype=torch.float32), rnd(70, 2 * H, seed=3)
    two = [w.clone().requires_grad_(), w.clone().requires_grad_()]
    B8.mlp_blocks(x, *two).backward(dy)
    one = w.clone().requires_grad_()
    if before:
        one.grad = torch.ones_like(w)
    B8.mlp_blocks(x, one, one).backward(dy)
    want = two[0].grad.double() + two[1].grad.double() + float(before)
    # two fp32 additions, each off by half a step of its result
    tol = 2.0 ** -24 * (want.abs() + (1 + two[1].grad.double()).abs() + (1 + two[0].grad.double()).abs())
    assert ((one.grad.double() - want).abs() <= tol * 1.001).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K,N", [(900, 5), (900, 40009), (1100, 20011), (2048, 4800), (4500, 2400)])
@pytest.mark.parametrize("M", [1, 8, 9, 16])
def test_few_rows_against_wide_weights(M, K, N, dtype):
    """Every number of row groups of a CTA, one wave and several, a last CTA of fewer groups and rows."""
    x, w = rnd(M, K, seed=1, dtype=dtype), rnd(N, K, seed=2, std=K ** -0.5)
    qx, qw, bias = held(x), held(w), torch.randn(N, device=DEV)
    want = qx @ qw.t()
    got = B8.linear_blocks(x, B8.quantize_blocks(w), bias)
    # the bias joins in fp32: half a step of that sum, and of the output's type
    more = (want + bias.double()).abs() * 2.0 ** -23 + bias.double().abs() * torch.finfo(dtype).eps
    assert_within(got, want + bias.double(), product_tol(qx, qw, dtype, want + bias.double()) + more)


def test_more_than_2_31_values():
    """Offsets past 31 bits: the last rows and columns of a matrix of 2.16e9 values are those of the slices by themselves."""
    M, K = 33024, 65536
    x = torch.randn(M, K, device=DEV, dtype=torch.bfloat16, generator=torch.Generator(device=DEV).manual_seed(1))
    r, c = B8.quantize_blocks(x, "both")
    tail, right = B8.quantize_blocks(x[-128:]), B8.quantize_blocks(x[:, -128:], "cols")
    assert torch.equal(r.codes[-128:].view(torch.uint8), tail.codes.view(torch.uint8)) and torch.equal(r.scales[-1:], tail.scales)
    assert torch.equal(c.codes[-128:].view(torch.uint8), right.codes.view(torch.uint8)) and torch.equal(c.scales[-1:], right.scales)
    assert torch.equal(B8.dequantize_blocks(r)[-128:], B8.dequantize_blocks(tail))
    v = x[:1].clone()
    assert torch.equal(B8.linear_blocks(v, r)[:, -128:], B8.linear_blocks(v, tail))
    few = B8.quantize_blocks(x[:64])
    want = held(x[-128:]) @ held(x[:64]).t()
    assert_within(B8.gemm_blocks(r, few)[-128:], want, product_tol(held(x[-128:]), held(x[:64]), torch.bfloat16, want))
    assert_within(B8.gemm_blocks(few, r)[:, -128:], want.t(), product_tol(held(x[:64]), held(x[-128:]), torch.bfloat16, want.t()))
    out = torch.empty(M, K, device=DEV, dtype=torch.bfloat16)  # an output of as many values
    a, b = B8.quantize_blocks(x[:, :128].contiguous()), B8.quantize_blocks(x[:1, :].view(K // 128, 128).repeat(128, 1))
    B8.gemm_blocks(a, b, out=out)
    want = held(x[-128:, :128]) @ held(x[:1].view(K // 128, 128)).t()
    tol = product_tol(held(x[-128:, :128]), held(x[:1].view(K // 128, 128)), torch.bfloat16, want)
    assert_within(out[-128:, -K // 128:], want, tol)
    del out, r, c
    ab, dg = x.requires_grad_(), torch.ones(M, K // 2, device=DEV, dtype=torch.bfloat16)
    end = x.detach()[-128:].clone().requires_grad_()
    g, h = B8.swiglu_blocks(ab), B8.swiglu_blocks(end)
    g.backward(dg), h.backward(dg[-128:])
    assert torch.equal(g[-128:], h) and torch.equal(ab.grad[-128:], end.grad)


# ----------------------------------------------------------------------------------------------------- streams, graphs
def test_captured_and_replayed():
    lin = torch.nn.Linear(256, 384, device=DEV)
    x, dy = rnd(300, 256, seed=1).requires_grad_(), rnd(300, 384, seed=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            B8.linear_blocks(x, lin).backward(dy)
    torch.cuda.current_stream().wait_stream(side)
    x.grad = lin.weight.grad = lin.bias.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = B8.linear_blocks(x, lin)
        y.backward(dy)
    new_x, new_dy = rnd(300, 256, seed=3), rnd(300, 384, seed=4)
    with torch.no_grad():
        x.copy_(new_x)
        dy.copy_(new_dy)
    got = [x.grad, lin.weight.grad, lin.bias.grad]
    graph.replay()
    torch.cuda.synchronize()
    want = train_linear(new_x, lin.weight, lin.bias, new_dy)
    assert torch.equal(y.detach(), want[0])
    assert all(torch.equal(a, b) for a, b in zip(got, want[1:]))


@pytest.mark.parametrize("op", ["mlp", "swiglu", "few", "many"])
def test_two_graphs_of_the_other_operators(op):
    """Two captured graphs, replayed in turn and on other inputs, give what eager calls give."""
    w1, w2 = rnd(512, 192, seed=1, std=192 ** -0.5, dtype=torch.float32), rnd(160, 256, seed=2, std=1 / 16, dtype=torch.float32)
    held_w = B8.quantize_blocks(w1), B8.quantize_blocks(w2)

    def run(x):
        if op == "few" or op == "many":
            with torch.no_grad():
                return [B8.mlp_blocks(x, *held_w), B8.linear_blocks(x, held_w[0])]
        leaves = [x] + [w.detach().requires_grad_() for w in ((w1, w2) if op == "mlp" else ())]
        y = B8.mlp_blocks(*leaves) if op == "mlp" else B8.swiglu_blocks(x)
        y.backward(y.detach())
        return [y.detach()] + [t.grad for t in leaves]
    rows = 9 if op == "few" else 300
    xs = [rnd(rows, 192, seed=k).requires_grad_(op in ("mlp", "swiglu")) for k in (3, 4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(xs[0].detach().clone().requires_grad_(xs[0].requires_grad))
    torch.cuda.current_stream().wait_stream(side)
    graphs, got = [], []
    for x in xs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(run(x))
    with torch.no_grad():
        for k, x in enumerate(xs):
            x.copy_(rnd(rows, 192, seed=5 + k))
    for k in (0, 1, 0):
        graphs[k].replay()
    for x, g in zip(xs, got):
        want = run(x.detach().clone().requires_grad_(x.requires_grad))
        assert len(want) == len(g) and all(torch.equal(a, b) for a, b in zip(g, want))


def test_other_stream():
    x, w = rnd(300, 256, seed=1), rnd(96, 256, seed=2, dtype=torch.float32)
    want = train_linear(x, w, None, rnd(300, 96, seed=3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = train_linear(x, w, None, rnd(300, 96, seed=3))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    x, w = rnd(20, 128, seed=1), rnd(32, 128, seed=2, dtype=torch.float32)
    w8 = B8.quantize_blocks(w)
    with pytest.raises(ValueError):
        B8.quantize_blocks(x, "diagonal")
    with pytest.raises(ValueError):
        B8.quantize_blocks(x[0])
    with pytest.raises(ValueError):
        B8.quantize_blocks(x[:, :0])
    with pytest.raises(RuntimeError, match="bf16, fp16 or fp32"):
        B8.quantize_blocks(x.double())
    with pytest.raises(ValueError):
        B8.linear_blocks(x[:, :64], w)
    with pytest.raises(ValueError):
        B8.linear_blocks(x[:, :64], w8)
    with pytest.raises(RuntimeError, match="bias"):
        B8.linear_blocks(x, w, w[:, 0][:5])
    with pytest.raises(TypeError):
        B8.linear_blocks(x, "weight")
    with pytest.raises(RuntimeError, match="no gradient"):
        B8.linear_blocks(x.clone().requires_grad_(), w8)
    with pytest.raises(RuntimeError, match="expected"):
        B8.linear_blocks(x, w.cpu())
    with pytest.raises(RuntimeError, match="scales"):
        B8.linear_blocks(x, B8.Blocks8(w8.codes, w8.scales[:, :, :16], 128))
    with pytest.raises(RuntimeError, match="codes"):
        B8.linear_blocks(x, B8.Blocks8(w8.codes.view(torch.uint8), w8.scales, 128))
    with pytest.raises(RuntimeError, match="codes"):
        B8.dequantize_blocks(B8.Blocks8(w8.codes[:, ::2], w8.scales, 64))
    with pytest.raises(ValueError):
        B8.gemm_blocks(w8, B8.quantize_blocks(x[:, :100]))
    with pytest.raises(ValueError):
        B8.gemm_blocks(w8, w8, accumulate=True)
    with pytest.raises(RuntimeError, match="out"):
        B8.gemm_blocks(w8, w8, out=torch.empty(32, 31, device=DEV))
    with pytest.raises(RuntimeError, match="rows"):
        B8.gemm_blocks(w8, w8, out=torch.empty(32, 32, device=DEV).t())
    with pytest.raises(ValueError):
        B8.swiglu_blocks(x[:, :127])
    with pytest.raises(ValueError):
        B8.mlp_blocks(x, w, w)
    with pytest.raises(ValueError, match="bias"):
        B8.mlp_blocks(x, torch.nn.Linear(128, 256, device=DEV), w)


def test_higher_derivatives_are_refused():
    x, w = rnd(20, 128, seed=1).requires_grad_(), rnd(32, 128, seed=2, dtype=torch.float32).requires_grad_()
    y = B8.linear_blocks(x, w)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))
        for call in (lambda: B8.linear_blocks(dual, w), lambda: B8.swiglu_blocks(dual),
                     lambda: B8.mlp_blocks(dual, rnd(256, 128, seed=3), rnd(64, 128, seed=4))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_launch_counts():
    x, w = rnd(300, 256, seed=1), rnd(96, 256, seed=2, dtype=torch.float32)
    w8 = B8.quantize_blocks(w)
    for call, n in ((lambda: B8.quantize_blocks(x, "both"), 1), (lambda: B8.linear_blocks(x[:9], w8), 1),
                    (lambda: B8.linear_blocks(x, w8), 2), (lambda: B8.linear_blocks(x, w), 2)):
        before = ext().launch_count()
        call()
        assert ext().launch_count() - before == n


@pytest.mark.parametrize("tile", [0, 1, 2])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (130, 300, 700), (520, 513, 1500), (300, 61, 4500), (2100, 2600, 640)])
def test_every_tile(M, N, K, tile):
    a, b = rnd(M, K, seed=3, dtype=torch.float32), rnd(N, K, seed=4, dtype=torch.float32)
    A, Bb, qa, qb = B8.quantize_blocks(a), B8.quantize_blocks(b), held(a), held(b)
    want = qa @ qb.t()
    ext().set_gemm8_tile(tile)
    try:
        for dtype in TYPES:
            assert_within(B8.gemm_blocks(A, Bb, dtype=dtype), want, product_tol(qa, qb, dtype, want))
        out = torch.ones(M, N, device=DEV)
        B8.gemm_blocks(A, Bb, out=out, accumulate=True)
        assert_within(out, want + 1, product_tol(qa, qb, torch.float32, want) + (want + 1).abs() * 2.0 ** -23 + 2.0 ** -23)
    finally:
        ext().set_gemm8_tile(-1)


@pytest.mark.parametrize("tile", [0, 1, 2])
@pytest.mark.parametrize("M,N,K", [(700, 96, 300), (9000, 640, 520), (2300, 3000, 1800), (300, 4096, 8192)])
def test_gradients_of_a_layer_in_one_launch(M, N, K, tile):
    """The input's and the weight's gradient share a launch, whichever has the longer sums and however the tiles fill it."""
    x, w, dy = rnd(M, K, seed=1), rnd(N, K, seed=2, std=K ** -0.5, dtype=torch.float32), rnd(M, N, seed=3, std=0.1)
    ext().set_gemm8_tile(tile)
    try:
        got = train_linear(x, w, None, dy)
        alone = B8.gemm_blocks(B8.quantize_blocks(dy), B8.quantize_blocks(w, "cols")), \
            B8.gemm_blocks(B8.quantize_blocks(dy, "cols"), B8.quantize_blocks(x, "cols"), dtype=torch.float32)
    finally:
        ext().set_gemm8_tile(-1)
    assert torch.equal(got[1], alone[0]) and torch.equal(got[2], alone[1])
    dw = held_t(dy).t() @ held_t(x)
    assert_within(got[2], dw, product_tol(held_t(dy).t(), held_t(x).t(), torch.float32, dw))


def test_backward_called_from_another_stream():
    x, lin, dy = rnd(4096, 512, seed=1), torch.nn.Linear(512, 2048, device=DEV), rnd(4096, 2048, seed=3)
    want = train_linear(x, lin.weight, lin.bias, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    leaf = x.clone().requires_grad_()
    with torch.cuda.stream(side):
        y = B8.linear_blocks(leaf, lin)
    torch.cuda.current_stream().wait_stream(side)
    y.backward(dy)  # runs where the forward ran; what it wrote is there for this stream
    got = [leaf.grad.clone(), lin.weight.grad.clone(), lin.bias.grad.clone()]
    assert all(torch.equal(a, b) for a, b in zip(got, want[1:]))
