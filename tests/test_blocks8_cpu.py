"""8-bit block operators: the CPU definitions, their gradients and refusals."""
import math

import pytest
import torch

from trenowanie_generatora_obrazkow_b200.ops import blocks8 as B8


def slow_held(row):
    """The values that 8 bits hold of one row, number by number."""
    out = []
    for lo in range(0, len(row), 128):
        block = [float(v) for v in row[lo:lo + 128]]
        top = max([abs(v) for v in block if math.isfinite(v)], default=0.0)
        e = -127
        while top > 448.0 * 2.0 ** e:
            e += 1
        for v in block:
            if not math.isfinite(v):
                out.append(math.nan)
                continue
            u = v / 2.0 ** e
            p = max(-6, math.frexp(u)[1] - 1) if u else -6
            step = 2.0 ** (p - 3)
            out.append(round(u / step) * step * 2.0 ** e)  # round: ties to even
    return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("M,K", [(1, 1), (3, 100), (5, 128), (2, 300)])
def test_held_values(M, K):
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(K)) * torch.logspace(-3, 3, K)
    b = B8.quantize_blocks(x)
    assert b.shape == (M, K) and b.codes.dtype == torch.float8_e4m3fn and b.codes.shape[1] % 128 == 0
    got = B8.dequantize_blocks(b, torch.float32)
    assert torch.equal(got.double(), torch.stack([slow_held(r) for r in x]))
    r, c = B8.quantize_blocks(x, "both")
    assert torch.equal(c.codes.view(torch.uint8), B8.quantize_blocks(x.t()).codes.view(torch.uint8))
    assert torch.equal(r.scales, b.scales)


def test_special_values():
    x = torch.zeros(4, 260)
    x[0, 3], x[0, 200] = math.inf, math.nan
    x[0, 5] = 2.0
    x[1, 0] = 448.0
    x[2, 0] = 448.5
    x[3, :] = 2.0 ** -130
    got = B8.dequantize_blocks(B8.quantize_blocks(x), torch.float32)
    want = torch.stack([slow_held(r) for r in x]).float()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0), want.nan_to_num(0))


def test_error_of_a_value():
    """Half a step of e4m3, 2^-4 of the value, or half the smallest step where a value is far below its block's largest."""
    x = torch.randn(64, 512, generator=torch.Generator().manual_seed(0))
    got = B8.dequantize_blocks(B8.quantize_blocks(x), torch.float32)
    top = x.abs().view(64, 4, 128).amax(-1, keepdim=True).expand(-1, -1, 128).reshape(64, 512)
    assert ((got - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, top / 224 * 2.0 ** -10)).all()


def test_linear_and_mlp_gradients_follow_their_formulas():
    g = torch.Generator().manual_seed(1)
    x, w, b = (torch.randn(*s, generator=g).requires_grad_() for s in ((20, 130), (24, 130), (24,)))
    dy = torch.randn(20, 24, generator=g)
    y = B8.linear_blocks(x, w, b)
    y.backward(dy)
    q = lambda t: torch.stack([slow_held(r) for r in t.detach()])  # noqa: E731
    assert torch.allclose(y.double(), q(x) @ q(w).t() + b.double(), rtol=1e-5, atol=1e-5)
    assert torch.allclose(x.grad.double(), q(dy) @ q(w.t()).t(), rtol=1e-5, atol=1e-5)
    assert torch.allclose(w.grad.double(), q(dy.t()) @ q(x.t()).t(), rtol=1e-5, atol=1e-5)
    assert torch.allclose(b.grad, dy.sum(0), rtol=1e-5, atol=1e-6)
    x, w1, w2 = (torch.randn(*s, generator=g).requires_grad_() for s in ((20, 40), (256, 40), (12, 128)))
    y = B8.mlp_blocks(x, w1, w2)
    dy = torch.randn(20, 12, generator=g)
    y.backward(dy)
    ab = (q(x) @ q(w1).t()).float()
    gated = torch.nn.functional.silu(ab[:, :128]) * ab[:, 128:]
    assert torch.allclose(y.double(), q(gated) @ q(w2).t(), rtol=1e-3, atol=1e-3)
    assert torch.allclose(w2.grad.double(), q(dy.t()) @ q(gated.t()).t(), rtol=1e-3, atol=1e-3)
    assert x.grad.shape == x.shape and w1.grad.shape == w1.shape


def test_swiglu_gradient_against_differences():
    ab = (torch.randint(-7, 8, (6, 256), generator=torch.Generator().manual_seed(2)) / 4.0).double()  # held exactly
    f = lambda t: (torch.nn.functional.silu(t[:, :128]) * t[:, 128:]).sum()  # noqa: E731
    leaf = ab.float().requires_grad_()
    B8.swiglu_blocks(leaf).sum().backward()
    for i, j in ((0, 0), (3, 77), (5, 200)):
        d = torch.zeros_like(ab)
        d[i, j] = 1e-4
        assert abs((f(ab + d) - f(ab - d)).item() / 2e-4 - leaf.grad[i, j].item()) < 1e-5


def test_serving_form_and_refusals():
    x, w = torch.randn(3, 130), torch.randn(16, 130)
    w8 = B8.quantize_blocks(w)
    assert torch.equal(B8.linear_blocks(x, w8), B8.gemm_blocks(B8.quantize_blocks(x), w8, dtype=torch.float32))
    assert B8.linear_blocks(x.view(1, 3, 130), w8).shape == (1, 3, 16)
    with pytest.raises(RuntimeError, match="no gradient"):
        B8.linear_blocks(x.clone().requires_grad_(), w8)
    with pytest.raises(ValueError):
        B8.quantize_blocks(x, "all")
    with pytest.raises(ValueError):
        B8.quantize_blocks(x[0])
    with pytest.raises(ValueError):
        B8.linear_blocks(x[:, :5], w)
    with pytest.raises(ValueError):
        B8.gemm_blocks(w8, B8.quantize_blocks(x[:, :100]))
    with pytest.raises(ValueError):
        B8.swiglu_blocks(x[:, :129])
    with pytest.raises(ValueError):
        B8.mlp_blocks(x, w, w)
    with pytest.raises(TypeError):
        B8.mlp_blocks(x, w8, w)
    with pytest.raises(ValueError, match="bias"):
        B8.mlp_blocks(x, torch.nn.Linear(130, 256), torch.randn(16, 128))
    leaf = x.clone().requires_grad_()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(B8.linear_blocks(leaf, w).sum(), leaf, create_graph=True)[0].sum(), leaf)


def test_swiglu_of_sigmoids_below_the_range_of_fp32():
    a = torch.tensor([-63.5, -64.5, -88.0, -96.0, -120.0, -160.0, -20.0, 0.0, 88.0]).repeat(15)[:128].expand(4, 128)
    ab = torch.cat([a, torch.full((4, 128), 2.0 ** 118)], dim=1)
    leaf = ab.clone().requires_grad_()
    B8.swiglu_blocks(leaf).backward(torch.full((4, 128), 16.0))
    a, b = (torch.stack([slow_held(r) for r in v]) for v in ab.chunk(2, dim=1))  # what the backward reads
    s = torch.sigmoid(a)
    low = 2.0 ** -126
    assert torch.allclose(leaf.grad.double(), 16 * torch.cat([b * s * (1 + a * (1 - s)), a * s], dim=1), rtol=1e-5, atol=low)
    a, b = ab.double().chunk(2, dim=1)
    assert torch.allclose(B8.swiglu_blocks(ab).double(), a * torch.sigmoid(a) * b, rtol=1e-5, atol=low)


def test_no_rows():
    r, c = B8.quantize_blocks(torch.empty(0, 300), "both")
    assert r.shape == (0, 300) and c.shape == (300, 0)
    assert B8.dequantize_blocks(r).shape == (0, 300) and B8.dequantize_blocks(c).shape == (300, 0)
    w, b, w1, w2 = (torch.randn(s).requires_grad_() for s in ((12, 300), (12,), (256, 300), (8, 128)))
    for fn, ws, n in ((B8.linear_blocks, (w, b), 12), (B8.mlp_blocks, (w1, w2), 8)):
        x = torch.empty(2, 0, 300, requires_grad=True)
        y = fn(x, *ws)
        y.sum().backward()
        assert y.shape == (2, 0, n) and x.grad.shape == x.shape and all((t.grad == 0).all() for t in ws)
    ab = torch.empty(0, 256, requires_grad=True)
    B8.swiglu_blocks(ab).sum().backward()
    assert ab.grad.shape == (0, 256)
    assert B8.linear_blocks(torch.empty(0, 300), B8.quantize_blocks(w.detach())).shape == (0, 12)
