"""The CPU definitions of the routed block's operators: gradients by finite differences in 64 bits, the plan against a
plain loop, the refusals."""
import pytest
import torch

from trenowanie_generatora_obrazkow_b200.ops import fused as Fz
from trenowanie_generatora_obrazkow_b200.ops import reference as R
from trenowanie_generatora_obrazkow_b200.ops import routing as Rt


def rnd(*shape):
    return torch.randn(*shape, dtype=torch.float64)


@pytest.mark.parametrize("score,renorm,groups", [("softmax", True, 1), ("softmax", False, 2), ("sigmoid", True, 4),
                                                 ("sigmoid", False, 1)])
def test_route_gradcheck(score, renorm, groups):
    torch.manual_seed(0)
    logits = rnd(5, 12).requires_grad_()
    f = lambda l: Rt.route_experts(l, 3, score=score, renorm=renorm, groups=groups, top_groups=max(1, groups // 2),
                                   scale=2.5)[0]
    assert torch.autograd.gradcheck(f, logits)


def test_route_against_topk():
    torch.manual_seed(1)
    logits = torch.randn(50, 10)
    w, idx = Rt.route_experts(logits, 3)
    pw, pi = logits.softmax(-1).topk(3)
    assert torch.equal(idx.long(), pi) and torch.allclose(w, pw / pw.sum(-1, keepdim=True), atol=1e-6)
    bias = torch.zeros(10)
    bias[7] = 100.0  # the bias moves the choice, not the weight
    w, idx = Rt.route_experts(logits, 1, score="sigmoid", bias=bias, renorm=False)
    assert (idx == 7).all() and torch.allclose(w[:, 0], torch.sigmoid(logits[:, 7]))
    w, idx = Rt.route_experts(logits, 2, groups=5, top_groups=1)
    assert (idx // 2 == idx[:, :1] // 2).all() and (logits.argmax(1) == idx[:, 0]).all()


@pytest.mark.parametrize("cap", [None, 3])
def test_plan_against_a_loop(cap):
    torch.manual_seed(2)
    idx = torch.randint(-1, 5, (20, 2))
    plan = Rt.expert_plan(idx, 5, capacity=cap)
    seen = [0] * 5
    counts = torch.bincount(idx[idx >= 0], minlength=5)
    start = [e * cap for e in range(5)] if cap else (counts.cumsum(0) - counts).tolist()
    for n in range(20):
        for j in range(2):
            e = int(idx[n, j])
            want = -1 if e < 0 or (cap and seen[e] >= cap) else start[e] + seen[e]
            assert plan.slot[n, j] == want
            if e >= 0:
                seen[e] += 1
    assert torch.equal(plan.counts.long(), counts) and plan.rows == (15 if cap else 40)


def test_dispatch_combine_gradcheck():
    torch.manual_seed(3)
    plan = Rt.expert_plan(torch.randint(-1, 4, (6, 2)), 4, capacity=3)
    assert torch.autograd.gradcheck(lambda x: Rt.expert_dispatch(x, plan), rnd(6, 5).requires_grad_())
    y, w = rnd(plan.rows, 5).requires_grad_(), torch.rand(6, 2).requires_grad_()
    out = Rt.expert_combine(y, w, plan)
    out.sum().backward()
    keep = plan.slot >= 0
    want = torch.where(keep, y.detach().sum(1)[plan.slot.clamp(min=0).long()], torch.zeros((), dtype=torch.float64))
    assert torch.allclose(w.grad.double(), want)


@pytest.mark.parametrize("post,gate,mod", [(True, True, True), (False, True, False), (True, False, True)])
def test_sandwich_gradcheck(post, gate, mod):
    torch.manual_seed(4)
    parts = [rnd(2, 3, 6), rnd(2, 3, 6), rnd(2, 6) if gate else None, rnd(6) if post else None, rnd(6),
             rnd(2, 6) if mod else None, rnd(2, 6) if mod else None]
    leaves = [p.requires_grad_() for p in parts if p is not None]

    def f(*ts):
        it = iter(ts)
        return Fz.sandwich_norm(*[next(it) if p is not None else None for p in parts], res_scale=0.7)
    assert torch.autograd.gradcheck(f, leaves)


def test_sandwich_reduces_to_adanorm():
    torch.manual_seed(5)
    x, y, g, s, c, w = (torch.randn(*n) for n in ((2, 4, 8), (2, 4, 8), (2, 8), (2, 8), (2, 8), (8,)))
    a = Fz.adanorm(x, y, g, w, s, c)
    b = Fz.sandwich_norm(x, y, gate=g, w=w, shift=s, scale=c)
    assert torch.allclose(a[0], b[0], atol=1e-6) and torch.allclose(a[1], b[1], atol=1e-5)


@pytest.mark.parametrize("interleaved", [True, False])
def test_rope_gradcheck_and_axes(interleaved):
    torch.manual_seed(6)
    pos = torch.randint(0, 9, (2, 3, 2))
    q, k = rnd(2, 3, 2, 10).requires_grad_(), rnd(2, 3, 1, 10).requires_grad_()
    qw, kw = rnd(10).requires_grad_(), rnd(10).requires_grad_()
    f = lambda q, k, qw, kw: Fz.rope_axes(q, k, pos, (4, 4), q_w=qw, k_w=kw, interleaved=interleaved)
    assert torch.autograd.gradcheck(f, (q, k, qw, kw))


def test_rope_axes_matches_the_tables():
    torch.manual_seed(7)
    q, k = torch.randn(2, 12, 3, 16), torch.randn(2, 12, 1, 16)
    rows, cols = torch.meshgrid(torch.arange(3), torch.arange(4), indexing="ij")
    pos = torch.stack([rows, cols], -1).view(1, 12, 2).expand(2, 12, 2)
    a, b = Fz.rope_axes(q, k, pos, (8, 8))
    cos, sin = R.rope_2d_table(3, 4, 16)
    assert torch.allclose(a, R.apply_rope(q, cos, sin), atol=1e-6)
    assert torch.allclose(b, R.apply_rope(k, cos, sin), atol=1e-6)


def test_refusals():
    l, x = torch.zeros(4, 8), torch.zeros(2, 4, 16)
    q, pos = torch.zeros(2, 3, 4, 16), torch.zeros(2, 3, 1, dtype=torch.int32)
    for f in (lambda: Rt.route_experts(l, 9), lambda: Rt.route_experts(l, 2, groups=3),
              lambda: Rt.route_experts(l, 2, score="relu"), lambda: Rt.expert_plan(torch.zeros(4), 4),
              lambda: Rt.expert_plan(torch.zeros(4, 2), 4, capacity=0), lambda: Fz.sandwich_norm(x, x[:1]),
              lambda: Fz.sandwich_norm(x, x, shift=x[:, 0], w=x[0, 0]),
              lambda: Fz.sandwich_norm(x, x, shift=x[:, 0], scale=x[:, 0]), lambda: Fz.rope_axes(q, q, pos, (18,)),
              lambda: Fz.rope_axes(q, q, pos, (8, 8)), lambda: Fz.rope_axes(q, q, pos, (3,))):
        with pytest.raises(ValueError):
            f()


def test_axes_table_is_no_inference_tensor():
    with torch.inference_mode():
        freq, axis = Fz._axes_table((10, 6), 555.0, torch.device("cpu"))
    assert not freq.is_inference() and not axis.is_inference()
