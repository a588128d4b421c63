"""8-bit block operators at their edges on the GPU: scales and sigmoids far out, blocks without a finite value, weights that are
frozen or released between forward and backward, sizes that give every unit several tiles."""
import math

import pytest
import test_blocks8_gpu as plain
import torch
from test_blocks8_gpu import HALF, TYPES, held, held_t, rnd

from trenowanie_generatora_obrazkow_b200.ops import blocks8 as B8
from trenowanie_generatora_obrazkow_b200.ops._ext import check_errors

pytestmark = pytest.mark.gpu
DEV = "cuda"
WIDE = [torch.bfloat16, torch.float32]  # types with fp32's range


@pytest.fixture(autouse=True)
def _no_kernel_errors():
    yield
    if torch.cuda.is_available():
        check_errors(DEV)


# ---------------------------------------------------------------------------------------------------------- far scales
@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("M", [1, 8, 9, 16, 17, 130])
def test_scales_whose_product_is_out_of_range(M, dtype):
    """The largest values of x's and W's blocks do not meet: the scales' product is beyond fp32, the sums are not."""
    x, w = torch.zeros(M, 256, device=DEV), torch.zeros(5, 256, device=DEV)
    x[:, 0], x[:, 1], x[:, 130] = 2.0 ** 100, 2.0 ** 84, 1.0
    w[:, 2] = 2.0 ** 60                   # beside x's zeros
    w[1, 1] = 2.0 ** 43                   # 2^127
    w[2, 1], w[2, 130] = -(2.0 ** 43), 3.0  # -2^127
    w[3, 130] = 5.0                       # 5, from the second block alone
    got = B8.linear_blocks(x.to(dtype), B8.quantize_blocks(w))
    want = (held(x) @ held(w).t()).to(dtype)
    assert want[0].tolist() == [0.0, 2.0 ** 127, -(2.0 ** 127), 5.0, 0.0]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("M", [1, 8, 9, 16, 17, 130])
@pytest.mark.parametrize("e", [-149, -150, -154])
def test_scales_whose_product_is_too_small(M, dtype, e):
    """Sums of 49 2^19 2^e, normal numbers of fp32, from scales whose product is not."""
    x = torch.full((M, 128), 448 * 2.0 ** -70, device=DEV, dtype=dtype)
    w = torch.full((3, 128), 448 * 2.0 ** (e + 70), device=DEV)
    x[:, 64:], w[1, :64] = 0, 0
    got = B8.linear_blocks(x, B8.quantize_blocks(w))
    want = torch.tensor([49 * 2.0 ** (18 + e), 0.0, 49 * 2.0 ** (18 + e)], device=DEV, dtype=torch.float64).to(dtype)
    assert torch.equal(got, want.expand(M, 3))


# ------------------------------------------------------------------------------------------------- no finite value at all
@pytest.mark.parametrize("dtype", TYPES)
def test_scale_bytes_of_blocks_without_a_finite_value(dtype):
    x = rnd(300, 400, dtype=dtype, seed=3)
    x[1, 128:256], x[2], x[3, 256:] = math.nan, -math.inf, math.inf
    x[128:256, 7], x[:, 9], x[256:, 11] = math.nan, math.inf, -math.inf
    x[4, 0:128:2], x[4, 1:128:2] = math.nan, math.inf
    want = B8.quantize_blocks(x.cpu(), "both")
    for got in (B8.quantize_blocks(x, "both"), (B8.quantize_blocks(x), B8.quantize_blocks(x, "cols"))):
        for a, b in zip(got, want):
            assert torch.equal(a.scales.cpu(), b.scales)
            assert torch.equal(a.codes.cpu().view(torch.uint8) & 0x7f, b.codes.view(torch.uint8) & 0x7f)


# ----------------------------------------------------------------------------------------------------------- far sigmoids
FAR = [-88.0, -96.0, -104.0, -120.0, -144.0, -160.0, -80.0, 0.0, -1.0, -20.0, 88.0, 160.0]


def far_activations(dtype):
    """[256, 256]: a [256, 128], the first six of FAR in the rows of the first tile, all of them in those of the second, and b =
    +-2^k with k falling along the columns. 8 bits hold each value, along the rows and along the columns."""
    m = torch.arange(256, device=DEV)
    a = torch.tensor(FAR, device=DEV)[torch.where(m < 128, m % 6, m % 12)][:, None].expand(256, 128)
    k = torch.arange(128, device=DEV) % 8
    return torch.cat([a, torch.exp2(118.0 - k) * (1 - 2 * (m % 2))[:, None]], 1).to(dtype)


@pytest.mark.parametrize("dtype", WIDE)
def test_swiglu_of_sigmoids_below_the_range_of_fp32(dtype):
    """a down to -160 with b large enough for results in range. exp(-160) is 0 in fp32."""
    ab = far_activations(dtype).requires_grad_()
    assert all(torch.equal(held(v), v.double()) for v in (ab.detach()[:, :128], ab.detach()[:, 128:], ab.detach().t()))
    dg = torch.full((256, 128), 2.0 ** 4, device=DEV, dtype=dtype)
    g = B8.swiglu_blocks(ab)
    g.backward(dg)
    # exp(a / 2) from an argument rounded to 2^-24 of itself (|a| / 2 < 80: 2^-17.7) and two units in the last place, squared
    fine = 2.0 ** -16
    low = 2.0 ** -126  # below it bits go
    want, d = plain.swiglu64(ab.detach()), plain.swiglu_grad64(ab.detach(), dg)
    plain.assert_within(g, want, want.abs() * (HALF[dtype] + fine) + low)
    a, b = ab.detach().double().chunk(2, 1)
    s = torch.sigmoid(a)
    parts = torch.cat([dg.double() * b * s * (1 + a.abs()), dg.double() * a * s], 1).abs()  # 1 + a (1 - s) may cancel
    plain.assert_within(ab.grad, d, d.abs() * HALF[dtype] + parts * fine + low)
    assert (want.abs() > 2.0 ** -60).double().mean() > 0.5


def in_8_bits(got, want, dim):
    """got are the held values of `want` up to 2^-14 of it: half a step of e4m3 or of the block's smallest step."""
    w = want if dim == 1 else want.t()
    top = w.abs().view(w.shape[0], -1, 128).amax(-1, keepdim=True).expand(-1, -1, 128).reshape(w.shape)
    tol = torch.maximum(w.abs() * 2.0 ** -4, top / 224 * 2.0 ** -10) * (1 + 2.0 ** -8)
    plain.assert_within(got, want, (tol if dim == 1 else tol.t()) + 2.0 ** -126)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("held_w", [False, True])
def test_mlp_of_sigmoids_below_the_range_of_fp32(dtype, held_w):
    """x and W2 the identity: y is g in 8 bits, dW1 the gradient of [a | b] in 8 bits."""
    ab, eye = far_activations(torch.float32), torch.eye(256, device=DEV)
    x, w1, w2 = eye.to(dtype), ab.t().contiguous(), torch.eye(128, device=DEV)
    want = plain.swiglu64(ab)
    if held_w:
        for rows in (256, 9):
            y = B8.mlp_blocks(x[:rows], B8.quantize_blocks(w1), B8.quantize_blocks(w2))
            in_8_bits(y.double(), want[:rows], 1)
        return
    leaves = [t.requires_grad_() for t in (x, w1, w2)]
    dy = torch.full((256, 128), 2.0 ** 4, device=DEV, dtype=dtype)
    y = B8.mlp_blocks(*leaves)
    y.backward(dy)
    in_8_bits(y.detach().double(), want, 1)
    in_8_bits(leaves[1].grad.double().t(), plain.swiglu_grad64(ab, dy), 0)


# ---------------------------------------------------------------------------- weights frozen or released in between
@pytest.mark.parametrize("op", ["linear", "mlp"])
@pytest.mark.parametrize("late", [(1,), (2,), (1, 2)])
@pytest.mark.parametrize("x_too", [False, True])
def test_weights_released_after_the_forward_get_no_gradient(op, late, x_too):
    """As everywhere in autograd, a tensor without requires_grad in the forward is not part of the graph."""
    def tensors():
        x, w = rnd(70, 128, seed=1), rnd(256, 128, seed=2, std=1 / 11, dtype=torch.float32)
        return [x, w, rnd(256, seed=3, dtype=torch.float32) if op == "linear" else rnd(72, 128, seed=3, std=1 / 11, dtype=torch.float32)]
    fn = B8.linear_blocks if op == "linear" else B8.mlp_blocks
    dy = rnd(70, 256 if op == "linear" else 72, seed=4)

    def run(release):
        ts = tensors()
        for i, t in enumerate(ts):
            t.requires_grad_(x_too if i == 0 else i not in late)
        y = fn(*ts)
        if not y.requires_grad:
            return None
        if release:
            for i in late:
                ts[i].requires_grad_()
        y.backward(dy)
        return [t.grad for t in ts]
    want, got = run(False), run(True)
    if want is None:
        assert late == (1, 2) and not x_too
        return
    for a, b in zip(got, want):
        assert (a is None) == (b is None) and (a is None or torch.equal(a, b))
    assert all(got[i] is None for i in late)


@pytest.mark.parametrize("op", ["linear", "mlp"])
@pytest.mark.parametrize("late", [(1,), (2,), (1, 2)])
def test_weights_frozen_after_the_forward_get_no_gradient(op, late):
    x, w = rnd(70, 128, seed=1), rnd(256, 128, seed=2, std=1 / 11, dtype=torch.float32)
    v = rnd(256, seed=3, dtype=torch.float32) if op == "linear" else rnd(72, 128, seed=3, std=1 / 11, dtype=torch.float32)
    fn = B8.linear_blocks if op == "linear" else B8.mlp_blocks
    dy = rnd(70, 256 if op == "linear" else 72, seed=4)
    full = [t.clone().requires_grad_() for t in (x, w, v)]
    fn(*full).backward(dy)
    ts = [t.clone().requires_grad_() for t in (x, w, v)]
    y = fn(*ts)
    for i in late:
        ts[i].requires_grad_(False)
    y.backward(dy)
    for i, (a, b) in enumerate(zip(ts, full)):
        assert a.grad is None if i in late else torch.equal(a.grad, b.grad)


# -------------------------------------------------------------------------------------------------- several tiles a unit
@pytest.mark.parametrize("dtype", TYPES)
def test_mlp_of_several_tiles_a_unit(dtype):
    """17 x 22 tiles of 256 x 128 for 74 pairs of CTAs and 34 x 22 of 128 x 128 for 148 SMs, an odd last row: every unit's
    accumulators, stages, maxima and staging are used again. Row by row and column by column."""
    M, K, H, N = 4301, 192, 2816, 160
    x, w1, w2 = rnd(M, K, seed=1, dtype=dtype), rnd(2 * H, K, seed=2, std=K ** -0.5, dtype=torch.float32, spread=0), \
        rnd(N, H, seed=3, std=H ** -0.5, dtype=torch.float32, spread=0)
    dy = rnd(M, N, seed=4, std=0.1, dtype=dtype)

    def run(rows, wants=(1, 1, 1)):
        leaves = [t.detach().clone().requires_grad_(bool(k)) for t, k in zip((x[rows], w1, w2), wants)]
        y = B8.mlp_blocks(*leaves)
        y.backward(dy[rows])
        return [y.detach()] + [t.grad for t in leaves]
    got = run(slice(None))
    # rows of y and dx are their own sums, whatever is computed beside them
    for lo, hi in ((0, 640), (1024, 2176), (4096, M), (4224, M)):
        part = run(slice(lo, hi))
        assert torch.equal(got[0][lo:hi], part[0]) and torch.equal(got[1][lo:hi], part[1])
    # with and without the checkpoint, g along its columns, or weights that are packed in the call
    for wants in ((1, 0, 0), (0, 1, 0), (0, 0, 1)):
        for a, b in zip(run(slice(None), wants), got):
            assert a is None or torch.equal(a, b)
    assert torch.equal(got[0], B8.mlp_blocks(x, w1, w2))
    assert torch.equal(got[0], B8.mlp_blocks(x, B8.quantize_blocks(w1), B8.quantize_blocks(w2)))
    # Of the 160 to 5632 values that a row's or a column's results sum over, fewer than 2^-5 fall on the other side of a border
    # of their 8 bits (2^-7 at most of all, and chance), by 2^-3 of themselves: 2^-3 2^-2.5 in the 2-norm, and a rounding
    for g, w in zip(got, plain.mlp64(x, w1, w2, dy, dtype)):
        for dim in (0, 1):
            off = (g.double() - w).norm(dim=dim) / w.norm(dim=dim)
            assert off.max().item() < 2.0 ** -5.5 + HALF[dtype], (tuple(g.shape), dim, off.argmax().item(), off.max().item())
