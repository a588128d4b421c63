"""Expert routing, expert dispatch / combine, sandwich norms and multi-axis rotary positions on the GPU against plain
implementations in 64 bits.

Tolerances: every kernel computes in fp32 and rounds each output once, so an output of type T may differ from the 64-bit
value by half a unit of T (relative UNIT[T], here with a factor 2 of room) and by the fp32 rounding of its terms: at most
OPS roundings of 2^-24 each of the sum of the magnitudes of the terms. OPS = 64 covers a chain of about 20 operations,
a reduction of depth 5 + 5 + 8 and the functions' own few units.
"""
import math

import pytest
import torch

from trenowanie_generatora_obrazkow_b200.ops import fused as Fz
from trenowanie_generatora_obrazkow_b200.ops import reference as R
from trenowanie_generatora_obrazkow_b200.ops import routing as Rt

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10, torch.float32: 2.0 ** -23}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -24, torch.float32: 0.0}  # fp16: half a subnormal step
OPS = 64
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def check(got, want, terms, name=""):
    """|got - want| <= UNIT |want| + OPS 2^-24 terms, elementwise (want, terms: 64 bits)."""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    tol = UNIT[got.dtype] * want.abs() + OPS * 2.0 ** -24 * torch.as_tensor(terms, device=want.device) + TINY[got.dtype]
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all(), name
    assert (err <= tol).all(), (name, (err - tol).max().item(), err.max().item())


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rnd(g, *shape, std=1.0, mean=0.0, dtype=F32):
    return (torch.randn(*shape, device="cuda", generator=g) * std + mean).to(dtype)


# ----------------------------------------------------------------------------------------------------------------
# routing
# ----------------------------------------------------------------------------------------------------------------
# (N, E, k, score, bias, groups, top_groups, renorm, scale, dtype)
ROUTES = [(1, 1, 1, "softmax", False, 1, 1, True, 1.0, F32), (1, 64, 8, "sigmoid", True, 8, 4, True, 2.5, F32),
          (257, 8, 2, "softmax", False, 1, 1, True, 1.0, F32), (1000, 8, 8, "softmax", True, 2, 2, False, 1.5, F32),
          (333, 7, 3, "sigmoid", False, 1, 1, False, 1.0, F32), (130, 16, 4, "softmax", False, 4, 2, False, 1.0, BF16),
          (65, 30, 6, "sigmoid", True, 5, 2, True, 2.5, F32), (129, 60, 4, "softmax", False, 1, 1, True, 1.0, F16),
          (77, 96, 8, "softmax", True, 8, 3, True, 1.0, F32), (100, 160, 6, "softmax", False, 8, 3, False, 16.0, F32),
          (515, 256, 8, "sigmoid", True, 8, 4, True, 2.5, F32), (33, 256, 32, "softmax", False, 1, 1, True, 1.0, BF16),
          (50, 384, 8, "sigmoid", True, 1, 1, True, 2.8, F32), (19, 512, 10, "softmax", False, 32, 5, False, 1.0, F32),
          (40, 500, 7, "sigmoid", False, 20, 1, True, 1.0, F16)]


@pytest.mark.parametrize("N,E,k,score,bias,groups,top,renorm,scale,dtype", ROUTES)
def test_route(N, E, k, score, bias, groups, top, renorm, scale, dtype):
    g = gen(1)
    logits = rnd(g, N, E, std=2.0, dtype=dtype)
    b = rnd(g, E, std=0.1) if bias else None
    dw = rnd(g, N, k)
    kw = dict(score=score, bias=b, groups=groups, top_groups=top, renorm=renorm, scale=scale)
    x = logits.clone().requires_grad_()
    w, idx = Rt.route_experts(x, k, **kw)
    w.backward(dw)
    # the choice is a function of the 32-bit scores: the same rule in 32 bits decides it
    _, want_idx = R.route_experts(logits.float(), k, **kw)
    key = logits.float() if score == "softmax" else torch.sigmoid(logits.float())
    same = (idx == want_idx).all(1)
    if not same.all():  # only scores within the sigmoid's own rounding may swap
        assert score == "sigmoid" and (~same).float().mean() < 0.01
    assert idx.dtype == torch.int32 and (idx >= 0).all() and (idx < E).all()
    assert (idx.sort(1).values.diff(dim=1) > 0).all()
    if b is not None:
        key = key + b
    if groups == 1:
        assert (key.gather(1, idx.long()).diff(dim=1) <= 1e-6).all()
    y = logits.double().requires_grad_()
    p = torch.softmax(y, -1) if score == "softmax" else torch.sigmoid(y)
    want = p.gather(1, idx.long())
    if renorm:
        want = want / (want.sum(-1, keepdim=True) + 1e-20)
    want = want * scale
    want.backward(dw.double())
    check(w, want.detach(), want.detach().abs(), "w")
    terms = (want.detach().abs() * dw.abs().double()).sum(1, keepdim=True) + dw.abs().double().amax(1, keepdim=True) * scale
    check(x.grad, y.grad, terms.expand_as(y.grad), "dlogits")
    with torch.no_grad():  # the form without autograd gives the same
        w2, idx2 = Rt.route_experts(logits, k, **kw)
    assert torch.equal(w2, w) and torch.equal(idx2, idx)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups", [(8, 1), (64, 4), (256, 8)])
def test_route_edges(score, E, groups):
    """Ties go to the lowest index, -0 equals +0, switched-off experts (-inf, the type's lowest) come last, a token with
    every expert off has weights of 0 (softmax) and no NaN, NaN logits never displace a number, padding rows get -1."""
    k, top = 4, max(1, groups // 2)
    kw = dict(score=score, groups=groups, top_groups=top)
    low = torch.finfo(F32).min
    rows = torch.zeros(9, E, device="cuda")
    rows[1, ::2] = -0.0
    rows[2] = -math.inf
    rows[3] = low
    rows[4, 1:] = -math.inf
    rows[5, : E // 2] = low
    rows[6, 0] = math.nan
    rows[7] = torch.arange(E, device="cuda").float()
    rows[8] = 100.0
    valid = torch.ones(9, dtype=torch.bool, device="cuda")
    valid[8] = False
    leaf = rows.clone().requires_grad_()
    w, idx = Rt.route_experts(leaf, k, valid=valid, **kw)
    first = torch.arange(k, device="cuda", dtype=torch.int32)
    for r in (0, 1, 2, 3):
        assert torch.equal(idx[r], first), r
    assert torch.equal(idx[8], torch.full_like(first, -1)) and (w[8] == 0).all()
    assert idx[4, 0] == 0 and w[4, 0] == 1.0 and (w[4, 1:] == 0).all()
    assert (w[2] == 0).all() if score == "softmax" else torch.isfinite(w[2]).all()
    assert (idx[6] != 0).all() and (idx[:8] >= 0).all() and (idx[:8] < E).all()
    if groups == 1:
        assert torch.equal(idx[7], torch.arange(E - 1, E - 1 - k, -1, device="cuda", dtype=torch.int32))
        assert (idx[5] >= E // 2).all()
    want_w, want_idx = R.route_experts(rows, k, valid=valid, **kw)
    keep = [0, 1, 2, 3, 4, 5, 7, 8]
    assert torch.equal(idx, want_idx)
    assert torch.allclose(w[keep], want_w[keep], rtol=1e-6, atol=1e-7)
    w[keep].sum().backward()
    assert torch.isfinite(leaf.grad[keep]).all() and (leaf.grad[8] == 0).all()


def test_route_gradient_by_differences():
    """Central differences of the weights in 64 bits around the kernel's gradient (the choice held fixed)."""
    g = gen(3)
    N, E, k = 5, 24, 4
    logits, dw = rnd(g, N, E), rnd(g, N, k)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            x = logits.clone().requires_grad_()
            w, idx = Rt.route_experts(x, k, score=score, renorm=renorm)
            w.backward(dw)

            def f(l):
                p = torch.softmax(l, -1) if score == "softmax" else torch.sigmoid(l)
                v = p.gather(1, idx.long())
                return ((v / v.sum(-1, keepdim=True) if renorm else v) * dw.double()).sum(-1)
            h = 1e-5
            for e in range(E):
                d = torch.zeros(N, E, device="cuda", dtype=torch.float64)
                d[:, e] = h
                num = (f(logits.double() + d) - f(logits.double() - d)) / (2 * h)
                assert (num - x.grad[:, e].double()).abs().max() < 2e-6  # h^2 third derivative + fp32 gradient


@pytest.mark.parametrize("N,E,k,score,bias,groups,top,renorm,dtype", [
    (30011, 256, 3, "sigmoid", True, 8, 4, True, F32), (40003, 256, 1, "softmax", True, 1, 1, False, BF16),
    (30001, 240, 6, "sigmoid", True, 10, 3, True, F32), (30007, 500, 2, "softmax", False, 1, 1, True, F16),
    (60005, 100, 2, "softmax", True, 5, 2, True, F32), (90001, 61, 1, "sigmoid", False, 1, 1, False, BF16),
    (300007, 8, 1, "softmax", False, 2, 1, True, F32)])
def test_route_many_tokens_as_few(N, E, k, score, bias, groups, top, renorm, dtype):
    """A warp takes several tokens one after the other when there are many: each token's result is that of a short call."""
    g = gen(33)
    logits = rnd(g, N, E, std=2.0, dtype=dtype)
    logits[::97, ::3] = -math.inf
    logits[5::1013] = math.nan
    valid = torch.rand(N, device="cuda", generator=g) > 0.1
    kw = dict(score=score, bias=rnd(g, E, std=0.1) if bias else None, groups=groups, top_groups=top, renorm=renorm)
    w, idx = Rt.route_experts(logits, k, valid=valid, **kw)
    for a in range(0, N, 2048):
        rows = slice(a, min(N, a + 2048))
        w1, idx1 = Rt.route_experts(logits[rows], k, valid=valid[rows], **kw)
        assert torch.equal(idx[rows], idx1), a
        assert torch.equal(w[rows].nan_to_num(nan=-7.0), w1.nan_to_num(nan=-7.0)), a


@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True)])
def test_route_padding_rows_stop_gradients(score, renorm):
    """NaN that reaches a padding row's weights does not reach its logits; an error reaches second derivatives."""
    g = gen(14)
    logits = rnd(g, 6, 40).requires_grad_()
    valid = torch.tensor([True, False, True, True, False, True], device="cuda")
    w, _ = Rt.route_experts(logits, 3, score=score, renorm=renorm, valid=valid)
    dw = rnd(g, 6, 3)
    dw[~valid] = math.nan
    w.backward(dw)
    assert torch.isfinite(logits.grad).all() and (logits.grad[~valid] == 0).all() and (logits.grad[0] != 0).any()
    w, _ = Rt.route_experts(logits, 3)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(w.sum(), logits, create_graph=True)


def test_broadcast_rows_share_their_gradient():
    """One modulation row expanded over the samples (stride 0): its gradient is the sum over them."""
    g = gen(15)
    ins = sandwich_inputs(g, 3, 20, 256, True, True, True, True, F32)
    one = {n: ins[n][:1].clone().requires_grad_() for n in ("gate", "shift", "scale")}
    each = {n: one[n].detach().expand(3, -1).contiguous().requires_grad_() for n in one}
    for rows in ({n: t.expand(3, -1) for n, t in one.items()}, each):
        a, b = Fz.sandwich_norm(**{**ins, **rows})
        (a.square().sum() + b.square().sum()).backward()
    for n in one:
        want = each[n].grad.sum(0, keepdim=True)
        assert torch.allclose(one[n].grad, want, rtol=1e-5, atol=1e-5 * want.abs().max().item())


def test_route_strided_rows_and_empty():
    g = gen(4)
    wide = rnd(g, 50, 40)
    a = Rt.route_experts(wide[:, 3:19], 3)
    b = Rt.route_experts(wide[:, 3:19].contiguous(), 3)
    c = Rt.route_experts(wide.t()[3:19].t(), 3)
    for x in (a, c):
        assert torch.equal(x[0], b[0]) and torch.equal(x[1], b[1])
    w, idx = Rt.route_experts(wide[:0], 3)
    assert w.shape == idx.shape == (0, 3)


# ----------------------------------------------------------------------------------------------------------------
# plan, dispatch, combine
# ----------------------------------------------------------------------------------------------------------------
def choices(g, N, E, k, pad=0.0):
    idx = (torch.rand(N, E, device="cuda", generator=g) + torch.linspace(0, 0.5, E, device="cuda")).topk(
        k, dim=1).indices.to(torch.int32)
    return idx.masked_fill((torch.rand(N, device="cuda", generator=g) < pad)[:, None], -1)


# (N, E, k, capacity, D, pad, dtype): one token, odd widths, one expert, many experts, more than one CTA of the plan
PLANS = [(1, 8, 2, None, 2048, 0.0, BF16), (1, 1, 1, None, 1, 0.0, F32), (37, 5, 3, None, 72, 0.3, BF16),
         (300, 64, 8, 16, 136, 0.1, BF16), (1031, 8, 2, 200, 577, 0.0, BF16), (5000, 16, 4, None, 64, 0.2, F32),
         (4099, 512, 2, 9, 40, 0.0, F16), (64, 40, 32, None, 1288, 0.0, BF16), (900, 3, 1, 1, 8, 0.0, F32),
         (50, 4, 2, None, 16, 1.0, BF16)]


@pytest.mark.parametrize("N,E,k,cap,D,pad,dtype", PLANS)
def test_dispatch_combine(N, E, k, cap, D, pad, dtype):
    g = gen(5)
    idx = choices(g, N, E, k, pad)
    plan = Rt.expert_plan(idx, E, capacity=cap)
    slot, offsets, counts = R.expert_plan(idx.cpu(), E, cap or 0)
    assert torch.equal(plan.slot.cpu(), slot) and torch.equal(plan.offsets.cpu(), offsets)
    assert torch.equal(plan.counts.cpu(), counts)
    x = rnd(g, N, D, dtype=dtype).requires_grad_()
    y = rnd(g, plan.rows, D, dtype=dtype).requires_grad_()
    w = torch.rand(N, k, device="cuda", generator=g).requires_grad_()
    dxs, dout = rnd(g, plan.rows, D, dtype=dtype), rnd(g, N, D, dtype=dtype)
    xs, out = Rt.expert_dispatch(x, plan), Rt.expert_combine(y, w, plan)
    torch.autograd.backward([xs, out], [dxs, dout])
    x64, y64, w64 = (t.detach().double().requires_grad_() for t in (x, y, w))
    xs64, out64 = R.expert_dispatch(x64, plan), R.expert_combine(y64, w64, plan)
    torch.autograd.backward([xs64, out64], [dxs.double(), dout.double()])
    assert torch.equal(xs.double(), xs64)  # copies
    check(out, out64.detach(), R.expert_combine(y64.detach().abs(), w64.detach(), plan), "out")
    keep = (plan.slot >= 0)
    check(x.grad, x64.grad, R.expert_combine(dxs.double().abs(), keep.double(), plan), "dx")
    check(y.grad, y64.grad, 0.0, "dy")
    ones = torch.ones_like(w64)
    mag = torch.stack([R.expert_combine(y64.detach().abs(), ones * (torch.arange(k, device="cuda") == j), plan)
                       for j in range(k)], 1)
    check(w.grad, w64.grad, (mag * dout.double().abs()[:, None]).sum(-1), "dw")


def test_dispatch_strided_and_nonfinite():
    """Rows of a wider tensor, a misaligned base, and infinities / NaN in rows that no assignment reaches."""
    g = gen(6)
    idx = choices(g, 200, 8, 2, 0.2)
    plan = Rt.expert_plan(idx, 8, capacity=40)
    wide = rnd(g, 200, 300, dtype=BF16)
    for x in (wide[:, 16:144], wide[:, 3:131], wide.t()[10:138].t()):
        assert torch.equal(Rt.expert_dispatch(x, plan), Rt.expert_dispatch(x.contiguous(), plan))
    y = rnd(g, plan.rows, 128, dtype=BF16)
    want = Rt.expert_combine(y, torch.ones(200, 2, device="cuda"), plan)
    used = torch.zeros(plan.rows + 1, dtype=torch.bool, device="cuda")
    used[plan.slot.long().reshape(-1)] = True  # -1 marks the extra last row
    y[~used[:-1]] = math.nan
    assert torch.equal(Rt.expert_combine(y, torch.ones(200, 2, device="cuda"), plan), want)
    yy, w = y.clone().requires_grad_(), torch.ones(200, 2, device="cuda").requires_grad_()
    Rt.expert_combine(yy, w, plan).sum().backward()
    assert torch.isfinite(yy.grad).all() and torch.isfinite(w.grad).all()
    empty = Rt.expert_plan(idx[:0], 8)
    assert empty.counts.sum() == 0 and (empty.offsets == 0).all() and empty.rows == 0


def test_plan_is_stable_at_size():
    """65536 x 8 assignments: the rows of an expert follow token order and tile the range exactly."""
    g = gen(7)
    N, E, k = 65536, 256, 8
    idx = choices(g, N, E, k, 0.05)
    plan = Rt.expert_plan(idx, E)
    flat = idx.reshape(-1)
    order = torch.where(flat >= 0, flat, E).argsort(stable=True)
    n = int((flat >= 0).sum())
    want = torch.full_like(flat, -1)
    want[order[:n]] = torch.arange(n, device="cuda", dtype=torch.int32)
    assert torch.equal(plan.slot.reshape(-1), want)
    assert torch.equal(plan.counts, torch.bincount(flat[flat >= 0], minlength=E).int())


# ----------------------------------------------------------------------------------------------------------------
# sandwich norm
# ----------------------------------------------------------------------------------------------------------------
def sandwich_inputs(g, B, T, D, post, gate, mod, pre, dtype):
    mods = rnd(g, B, 6, D, std=0.3, dtype=dtype)
    return dict(x=rnd(g, B, T, D, std=1.5, dtype=dtype), y=rnd(g, B, T, D, dtype=dtype),
                gate=mods[:, 2] if gate else None, post_w=rnd(g, D, std=0.1, mean=1.0) if post else None,
                w=rnd(g, D, std=0.1, mean=1.0) if pre else None, shift=mods[:, 0] if mod else None,
                scale=mods[:, 1] if mod else None)


# (B, T, D, post, gate, mod, pre, res, dtype): one row, one row per sample, odd and tiny widths, wide rows, every part
# left out in turn, a width of one channel
SANDWICH = [(1, 1, 576, True, True, True, True, 1.0, BF16), (2, 256, 576, True, True, True, True, 1.0, BF16),
            (3, 130, 2048, True, True, True, True, 0.5, BF16), (2, 33, 2560, True, False, False, True, 0.7, BF16),
            (200, 1, 128, True, True, True, True, 1.0, BF16), (4, 7, 8, True, True, True, True, 1.0, F32),
            (3, 50, 577, True, True, True, True, 1.0, BF16), (2, 40, 1000, True, True, False, True, 1.0, F16),
            (2, 65, 1024, False, True, True, True, 1.0, BF16), (2, 65, 512, False, False, False, True, 1.0, F32),
            (5, 19, 768, True, True, False, False, 2.0, BF16), (1, 300, 4096, True, False, True, True, 1.0, F32),
            (2, 9, 8192, True, True, True, True, 1.0, BF16), (1, 3, 16384, True, True, True, True, 1.0, F32),
            (1, 2000, 264, True, True, True, True, 1.0, BF16), (3, 5, 1, True, True, True, True, 1.0, F32)]


@pytest.mark.parametrize("B,T,D,post,gate,mod,pre,res,dtype", SANDWICH)
def test_sandwich_norm(B, T, D, post, gate, mod, pre, res, dtype):
    g = gen(8)
    ins = sandwich_inputs(g, B, T, D, post, gate, mod, pre, dtype)
    leaf = {n: (None if t is None else t.detach().requires_grad_()) for n, t in ins.items()}
    x_new, h = Fz.sandwich_norm(**leaf, res_scale=res)
    gx, gh = rnd(g, B, T, D, dtype=dtype), rnd(g, B, T, D, dtype=dtype)
    torch.autograd.backward([x_new] + ([h] if pre else []), [gx] + ([gh] if pre else []))
    d = {n: (None if t is None else t.detach().double().requires_grad_()) for n, t in ins.items()}
    xn64, h64 = R.sandwich_norm(**d, res_scale=res)
    torch.autograd.backward([xn64] + ([h64] if pre else []), [gx.double()] + ([gh.double()] if pre else []))
    one = torch.ones((), device="cuda", dtype=torch.float64)
    # magnitudes of the terms: u = res gate wp yn, and every gradient is a sum of products of these
    v = {n: (None if t is None else t.detach()) for n, t in d.items()}
    ry = (v["y"].square().mean(-1, keepdim=True) + 1e-6) ** -0.5 if post else one
    yn = v["y"].abs() * ry
    a = res * (v["gate"].abs()[:, None] if gate else one) * (v["post_w"].abs() if post else one)
    mag_x = v["x"].abs() + a * yn
    check(x_new, xn64.detach(), mag_x, "x_new")
    dx_mag = gx.double().abs()
    if pre:
        rx = (xn64.detach().square().mean(-1, keepdim=True) + 1e-6) ** -0.5
        sc = 1 + v["scale"].abs()[:, None] if mod else one
        n = mag_x * rx
        check(h, h64.detach(), n * v["w"].abs() * sc + (v["shift"].abs()[:, None] if mod else 0), "h")
        c = gh.double().abs() * v["w"].abs() * sc
        dx_mag = dx_mag + rx * (c + n * (c * n).mean(-1, keepdim=True))
        check(leaf["w"].grad, d["w"].grad, (gh.double().abs() * n * sc).sum((0, 1)), "dw")
        if mod:
            check(leaf["shift"].grad, d["shift"].grad, gh.double().abs().sum(1), "dshift")
            check(leaf["scale"].grad, d["scale"].grad, (gh.double().abs() * n * v["w"].abs()).sum(1), "dscale")
    check(leaf["x"].grad, d["x"].grad, dx_mag, "dx")
    s = a * dx_mag
    check(leaf["y"].grad, d["y"].grad, ry * (s + yn * (s * yn).mean(-1, keepdim=True)) if post else s, "dy")
    if post:
        check(leaf["post_w"].grad, d["post_w"].grad, (a / v["post_w"].abs() * dx_mag * yn).sum((0, 1)), "dpost_w")
    if gate:
        check(leaf["gate"].grad, d["gate"].grad,
              (res * (v["post_w"].abs() if post else one) * yn * dx_mag).sum(1), "dgate")


def test_sandwich_norm_partial_gradients_and_accumulation():
    """Only one output used, weights without a gradient, and gradients added to what .grad holds."""
    g = gen(9)
    ins = sandwich_inputs(g, 2, 40, 320, True, True, True, True, BF16)
    for use in ("x_new", "h"):
        leaf = {n: t.detach().requires_grad_(n not in ("post_w",)) for n, t in ins.items()}
        leaf["w"].grad = torch.ones_like(leaf["w"])
        x_new, h = Fz.sandwich_norm(**leaf)
        grad = rnd(g, 2, 40, 320, dtype=BF16)
        (x_new if use == "x_new" else h).backward(grad)
        d = {n: t.detach().double().requires_grad_() for n, t in ins.items()}
        xn64, h64 = R.sandwich_norm(**d)
        (xn64 if use == "x_new" else h64).backward(grad.double())
        rel = lambda p, q: ((p.double() - q).norm() / q.norm().clamp(min=1e-12)).item()
        assert rel(leaf["x"].grad, d["x"].grad) < 2 ** -8 and rel(leaf["y"].grad, d["y"].grad) < 2 ** -8
        if use == "h":
            assert rel(leaf["w"].grad - 1, d["w"].grad) < 1e-5
        else:
            assert torch.equal(leaf["w"].grad, torch.ones_like(leaf["w"]))
        assert leaf["post_w"].grad is None


def test_sandwich_norm_noncontiguous_and_repeatable():
    g = gen(10)
    ins = sandwich_inputs(g, 2, 64, 512, True, True, True, True, BF16)
    a = Fz.sandwich_norm(**ins)
    wide = torch.cat([ins["x"], ins["x"]], -1)
    b = Fz.sandwich_norm(**{**ins, "x": wide[..., :512], "shift": ins["shift"].contiguous()})
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    off = torch.empty(2 * 64 * 512 + 1, device="cuda", dtype=BF16)[1:].view(2, 64, 512).copy_(ins["x"])  # 2-byte aligned
    c = Fz.sandwich_norm(**{**ins, "x": off})  # another kernel: held to the 64-bit values by the rule above
    d = {n: t.double() for n, t in ins.items()}
    xn64, h64 = R.sandwich_norm(**d)
    yn = d["y"].abs() * (d["y"].square().mean(-1, keepdim=True) + 1e-6) ** -0.5
    mag = d["x"].abs() + d["gate"].abs()[:, None] * d["post_w"].abs() * yn
    n = mag * (xn64.square().mean(-1, keepdim=True) + 1e-6) ** -0.5
    check(c[0], xn64, mag, "misaligned x_new")
    check(c[1], h64, n * d["w"].abs() * (1 + d["scale"].abs()[:, None]) + d["shift"].abs()[:, None], "misaligned h")
    grads = []
    for _ in range(2):
        leaf = {n: t.detach().requires_grad_() for n, t in ins.items()}
        sum(o.float().square().sum() for o in Fz.sandwich_norm(**leaf)).backward()
        grads.append([t.grad for t in leaf.values()])
    assert all(torch.equal(p, q) for p, q in zip(*grads))  # fixed summation order


# ----------------------------------------------------------------------------------------------------------------
# rotary positions with several axes
# ----------------------------------------------------------------------------------------------------------------
# (B, T, Hq, Hkv, d, axes, theta, norm, interleaved, dtype)
ROPES = [(8, 1, 12, 4, 64, (64,), 1e4, True, False, BF16), (1, 1, 1, 1, 2, (2,), 1e4, True, True, F32),
         (2, 77, 16, 16, 128, (64, 64), 1e4, True, True, BF16), (1, 130, 20, 4, 128, (16, 56, 56), 1e4, True, False, BF16),
         (2, 50, 6, 2, 96, (32, 32, 32), (1e4, 1e3, 1e2), True, True, BF16), (2, 50, 3, 3, 96, (48,), 1e4, False, False, F32),
         (3, 33, 5, 1, 80, (40, 40), 1e4, True, True, F16), (1, 65, 4, 2, 256, (64, 96, 96), 1e4, True, False, BF16),
         (2, 19, 2, 2, 72, (24, 24, 24), 1e4, True, False, F32), (2, 21, 7, 7, 32, (8, 8, 8, 8), 1e4, False, True, BF16),
         (2, 9, 3, 1, 50, (10, 20), 1e4, True, True, F32), (1, 40, 2, 1, 512, (128, 128), 1e4, True, True, F32),
         (1, 40, 4, 4, 128, (2, 4), 1e4, True, False, BF16)]


@pytest.mark.parametrize("B,T,Hq,Hkv,d,axes,theta,norm,interleaved,dtype", ROPES)
def test_rope_axes(B, T, Hq, Hkv, d, axes, theta, norm, interleaved, dtype):
    g = gen(11)
    qkv = rnd(g, B, T, (Hq + 2 * Hkv) * d, dtype=dtype)
    q = qkv[..., :Hq * d].unflatten(-1, (Hq, d)).detach().requires_grad_()
    k = qkv[..., Hq * d:(Hq + Hkv) * d].unflatten(-1, (Hkv, d)).detach().requires_grad_()
    qw, kw = ((rnd(g, d, std=0.1, mean=1.0).requires_grad_() for _ in range(2)) if norm else (None, None))
    pos = torch.stack([torch.randint(-5, 100000 if a == 0 else 64, (B, T), device="cuda", generator=g)
                       for a in range(len(axes))], -1).to(torch.int32)
    dq, dk = rnd(g, B, T, Hq, d, dtype=dtype), rnd(g, B, T, Hkv, d, dtype=dtype)
    kwargs = dict(theta=theta, interleaved=interleaved)
    qo, ko = Fz.rope_axes(q, k, pos, axes, q_w=qw, k_w=kw, **kwargs)
    torch.autograd.backward([qo, ko], [dq, dk])
    q64, k64 = q.detach().double().requires_grad_(), k.detach().double().requires_grad_()
    w64 = [t.detach().double().requires_grad_() for t in (qw, kw)] if norm else [None, None]
    qo64, ko64 = R.rope_axes(q64, k64, pos, axes, q_w=w64[0], k_w=w64[1], **kwargs)
    torch.autograd.backward([qo64, ko64], [dq.double(), dk.double()])
    for name, x, out, want, g64, w, ww, up in (("q", q, qo, qo64, q64, qw, w64[0], dq), ("k", k, ko, ko64, k64, kw, w64[1], dk)):
        a = x.detach().double()
        r = (a.square().mean(-1, keepdim=True) + 1e-6) ** -0.5 if norm else 1.0
        n = a.abs() * r
        big = n.amax(-1, keepdim=True).expand_as(n) * (1.2 if norm else 1.0)
        check(out, want.detach(), 2 * big, name)
        u = up.double().abs().amax(-1, keepdim=True)
        grad = u * 2 * 1.2
        grad = r * (grad + n * grad * n.mean(-1, keepdim=True)) if norm else grad.expand_as(n)
        check(x.grad, g64.grad, 2 * grad.expand_as(n), "d" + name)
        if norm:
            check(w.grad, ww.grad, (2 * u * n).sum((0, 1, 2)), f"d{name}_w")


def test_rope_axes_is_the_2d_rope():
    """(row, column) positions with two equal axes reproduce the image model's table-driven q/k-norm + RoPE."""
    g = gen(12)
    B, h, w, H, d = 2, 6, 10, 4, 128
    q, k = rnd(g, B, h * w, H, d, dtype=BF16), rnd(g, B, h * w, H, d, dtype=BF16)
    rows, cols = torch.meshgrid(torch.arange(h), torch.arange(w), indexing="ij")
    pos = torch.stack([rows, cols], -1).view(1, h * w, 2).expand(B, -1, -1).cuda()
    qo, ko = Fz.rope_axes(q, k, pos, (d // 2, d // 2))
    cos, sin = R.rope_2d_table(h, w, d, device="cuda")
    for a, b in ((qo, q), (ko, k)):
        want = R.apply_rope(b.float(), cos, sin)
        assert (a.float() - want).abs().max() <= 2 ** -8 * want.abs().max()
    frac, _ = Fz.rope_axes(q, k, pos.float() * 0.5 - 0.25, (d // 2, d // 2))  # interpolated grids: fp32 positions
    want, _ = R.rope_axes(q.double(), k.double(), pos.float() * 0.5 - 0.25, (d // 2, d // 2))
    check(frac, want, 2 * q.double().abs().amax(), "fractions")


def test_gradients_by_differences():
    """Directional derivatives of the fp32 kernels' own forwards (central differences, h = 2^-6) against <gradient,
    direction>. The difference of the sum of n = 2 * 3 * 24 * 64 outputs of size 1 carries n^1/2 2^-24 / h = 4e-4 of
    rounding and h^2 / 6 = 4e-5 of the third derivative per unit, both far below 1e-2 of a derivative's size."""
    g = gen(16)
    ins = sandwich_inputs(g, 2, 24, 192, True, True, True, True, F32)
    up = [rnd(g, 2, 24, 192) for _ in range(2)]
    q, k = rnd(g, 2, 24, 3, 64), rnd(g, 2, 24, 1, 64)
    pos = torch.randint(0, 50, (2, 24, 2), device="cuda", generator=g)
    plan = Rt.expert_plan(choices(g, 48, 6, 2), 6, capacity=20)

    def sandwich(x, y, gate, post_w, w, shift, scale):
        return Fz.sandwich_norm(x, y, gate, post_w, w, shift, scale, res_scale=0.7)

    def rope(q, k, qw, kw):
        return Fz.rope_axes(q, k, pos, (32, 24), q_w=qw, k_w=kw)

    def rows(x, y, w):
        return Rt.expert_dispatch(x, plan), Rt.expert_combine(y, w, plan)
    cases = [(sandwich, [t.contiguous() for t in ins.values()], up),
             (rope, [q, k, rnd(g, 64, std=0.1, mean=1.0), rnd(g, 64, std=0.1, mean=1.0)],
              [rnd(g, 2, 24, 3, 64), rnd(g, 2, 24, 1, 64)]),
             (rows, [rnd(g, 48, 96), rnd(g, plan.rows, 96), torch.rand(48, 2, device="cuda", generator=g)],
              [rnd(g, plan.rows, 96), rnd(g, 48, 96)])]
    h = 2.0 ** -6
    for fn, xs, ups in cases:
        def f(args):
            with torch.no_grad():
                return sum((o.double() * u.double()).sum() for o, u in zip(fn(*args), ups)).item()
        leaves = [x.clone().requires_grad_() for x in xs]
        torch.autograd.backward(list(fn(*leaves)), ups)
        for i, leaf in enumerate(leaves):
            d = rnd(g, *leaf.shape)
            shifted = lambda s: [x + s * h * d if j == i else x for j, x in enumerate(xs)]
            num = (f(shifted(1)) - f(shifted(-1))) / (2 * h)
            want = (leaf.grad.double() * d.double()).sum().item()
            size = (leaf.grad.double().norm() * d.double().norm() / d.numel() ** 0.5).item()
            assert abs(num - want) < 1e-2 * max(size, 1.0), (fn.__name__, i, num, want, size)


def test_ops_on_a_side_stream():
    """Inputs made on one stream, used on another after it waited: results as on the default stream."""
    g = gen(13)
    ins = sandwich_inputs(g, 2, 300, 1024, True, True, True, True, BF16)
    logits = rnd(g, 500, 64)
    want = Fz.sandwich_norm(**ins) + tuple(Rt.route_experts(logits, 4))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = Fz.sandwich_norm(**ins) + tuple(Rt.route_experts(logits, 4))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rope_tables_made_while_sampling_serve_training():
    """The first call for a set of axes may come under inference_mode; a training step after it saves the same tables."""
    g = gen(31)
    q, k = rnd(g, 1, 5, 2, 32), rnd(g, 1, 5, 1, 32)
    pos = torch.arange(5, device="cuda", dtype=torch.int32).view(1, 5, 1)
    with torch.inference_mode():
        first = Fz.rope_axes(q, k, pos, (26,), theta=777.0)
    q.requires_grad_()
    again = Fz.rope_axes(q, k, pos, (26,), theta=777.0)
    again[0].sum().backward()
    assert torch.equal(first[0], again[0]) and q.grad is not None


def test_one_expert_column_of_a_wider_table():
    logits = torch.zeros(3, 8, device="cuda")[:, ::2][:, :1]
    w, idx = Rt.route_experts(logits, 1)
    assert (w == 1).all() and (idx == 0).all()


def test_sandwich_scratch_without_modulation():
    """Without gate or modulation all rows are one sample: the backward's scratch does not grow with B."""
    g = gen(32)
    x, y = (rnd(g, 20000, 1, 256, dtype=BF16).requires_grad_() for _ in range(2))
    w = torch.ones(256, device="cuda", requires_grad=True)
    x_new, h = Fz.sandwich_norm(x, y, w=w)
    d = torch.ones_like(h)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    torch.autograd.backward([h], [d])
    size = x.numel() * x.element_size()
    assert torch.cuda.max_memory_allocated() - base <= 2 * size + (16 << 20)


def test_refusals():
    """Bad arguments end in an exception before any launch."""
    x = torch.zeros(2, 4, 16, device="cuda", dtype=BF16)
    w = torch.ones(16, device="cuda")
    bad = [lambda: Rt.route_experts(torch.zeros(4, 8, device="cuda"), 9),
           lambda: Rt.route_experts(torch.zeros(4, 8, device="cuda"), 2, groups=3),
           lambda: Rt.route_experts(torch.zeros(4, 8, device="cuda"), 5, groups=4, top_groups=2),
           lambda: Rt.route_experts(torch.zeros(4, 8, device="cuda"), 2, score="relu"),
           lambda: Rt.route_experts(torch.zeros(4, 600, device="cuda"), 2),
           lambda: Rt.route_experts(torch.zeros(4, 8, device="cuda"), 2, bias=torch.zeros(7, device="cuda")),
           lambda: Rt.route_experts(torch.zeros(4, 8, device="cuda"), 2, bias=torch.zeros(8)),
           lambda: Rt.route_experts(torch.zeros(4, 8, device="cuda", dtype=torch.float64), 2),
           lambda: Rt.route_experts(torch.zeros(4, 8, device="cuda"), 2, scale=0.0),
           lambda: Rt.expert_plan(torch.zeros(4, device="cuda", dtype=torch.int32), 4),
           lambda: Rt.expert_plan(torch.zeros(4, 2, device="cuda", dtype=torch.int32), 4, capacity=0),
           lambda: Rt.expert_plan(torch.zeros(4, 2, device="cuda", dtype=torch.int32), 4, capacity=2 ** 29 - 16384),
           lambda: Rt.expert_plan(torch.zeros(4, 2, device="cuda", dtype=torch.int32), 4, capacity=2 ** 62),
           lambda: Fz.sandwich_norm(x, x[:1]), lambda: Fz.sandwich_norm(x, x, shift=x[:, 0], w=w),
           lambda: Fz.sandwich_norm(x, x, shift=x[:, 0], scale=x[:, 0]),
           lambda: Fz.sandwich_norm(x, x, gate=x[:1, 0], w=w), lambda: Fz.sandwich_norm(x, x.float(), w=w),
           lambda: Fz.sandwich_norm(x, x, w=w[:8]), lambda: Fz.sandwich_norm(x, x, w=w.cpu()),
           lambda: Fz.sandwich_norm(x, x, gate=x[:, 0].float(), w=w)]
    q, pos = torch.zeros(2, 3, 4, 16, device="cuda", dtype=BF16), torch.zeros(2, 3, 1, device="cuda", dtype=torch.int32)
    bad += [lambda: Fz.rope_axes(q, q, pos, (18,)), lambda: Fz.rope_axes(q, q, pos, (3,)),
            lambda: Fz.rope_axes(q, q, pos, (8, 8)), lambda: Fz.rope_axes(q, q[..., :8], pos, (8,)),
            lambda: Fz.rope_axes(q, q, pos, (8,), q_w=w), lambda: Fz.rope_axes(q, q.float(), pos, (8,)),
            lambda: Fz.rope_axes(q, q, pos, (8,), theta=(1.0, 2.0))]
    Fz.rope_axes(q, q, pos, (16,))
    bad += [lambda: Fz.rope_axes(q[0], q[0], pos[0], (16,)), lambda: Fz.rope_axes(q, q, pos[..., :0], (16,))]
    plan = Rt.expert_plan(torch.zeros(4, 2, device="cuda", dtype=torch.int32), 4)
    bad += [lambda: Rt.expert_dispatch(torch.zeros(5, 16, device="cuda"), plan),
            lambda: Rt.expert_combine(torch.zeros(7, 16, device="cuda"), torch.zeros(4, 2, device="cuda"), plan),
            lambda: Rt.expert_combine(torch.zeros(8, 16, device="cuda"), torch.zeros(4, 3, device="cuda"), plan),
            lambda: Rt.expert_dispatch(torch.zeros(4, 16, device="cuda", dtype=torch.int32), plan)]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            f()
            raise AssertionError(f"case {i} was accepted")
