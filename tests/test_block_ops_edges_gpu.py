"""Values at the edges of the routed block's operators on the GPU (NaN inside a group of experts, weights that fill two
places, lengths and sizes at the limits), each against the definition in 64 bits or the rule that the docstrings state.
"""
import math

import pytest
import torch

from trenowanie_generatora_obrazkow_b200.ops import fused as Fz
from trenowanie_generatora_obrazkow_b200.ops import reference as R
from trenowanie_generatora_obrazkow_b200.ops import routing as Rt

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rnd(g, *shape, std=1.0, mean=0.0, dtype=F32):
    return (torch.randn(*shape, device="cuda", generator=g) * std + mean).to(dtype)


# ----------------------------------------------------------------------------------------------------------------
# routing
# ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,k", [(8, 2, 2), (30, 5, 2), (64, 4, 3), (64, 16, 2), (256, 8, 4), (512, 32, 5),
                                        (500, 20, 3)])
def test_nan_adds_nothing_to_its_group(score, E, groups, k):
    """NaN logits anywhere in a group, behind its best experts too, count as -inf for the group's worth and are chosen
    last: the choice is the definition's. The logits are multiples of 1/4, so no two different ones are within rounding."""
    g = gen(40)
    N = 200
    logits = (rnd(g, N, E) * 8).round() / 4
    logits[torch.rand(N, E, device="cuda", generator=g) < 0.3] = math.nan
    size = E // groups
    logits[0] = -3.0
    logits[0, :2] = torch.tensor([2.0, math.nan], device="cuda")  # twice the best would win
    logits[0, size:size + 2] = 1.5
    logits[1] = math.nan  # nothing but NaN in all groups but one
    logits[1, -size:] = -5.0
    logits[2, ::2] = math.inf
    logits[3, :size] = -math.inf
    top = max(1, groups // 3, -(-k // size))
    _, idx = Rt.route_experts(logits, k, score=score, groups=groups, top_groups=top)
    _, want = R.route_experts(logits, k, score, None, groups, top)
    assert torch.equal(idx, want)
    if score == "sigmoid" and top == 1:
        assert (idx[0] // size == 1).all()
    bias = torch.zeros(E, device="cuda")  # an expert that is always taken, beside one that never is
    bias[0], bias[1:size] = math.inf, -math.inf
    _, idx = Rt.route_experts(logits, k, score=score, bias=bias, groups=groups, top_groups=top)
    _, want = R.route_experts(logits, k, score, bias, groups, top)
    assert torch.equal(idx, want)


# ----------------------------------------------------------------------------------------------------------------
# gradients of the norm weights
# ----------------------------------------------------------------------------------------------------------------
def test_a_refused_backward_leaves_no_grad_behind():
    """A backward that ends in an exception (here: the allocator's limit) gives a weight no .grad of unwritten memory."""
    x, y = (torch.zeros(4, 2048, 4096, device="cuda", dtype=BF16, requires_grad=True) for _ in range(2))
    q, k = (torch.zeros(4, 2048, 32, 128, device="cuda", dtype=BF16, requires_grad=True) for _ in range(2))
    pos = torch.zeros(4, 2048, 1, device="cuda", dtype=torch.int32)
    post_w, w = (torch.ones(4096, device="cuda", requires_grad=True) for _ in range(2))
    q_w, k_w = (torch.ones(128, device="cuda", requires_grad=True) for _ in range(2))
    outs = (Fz.sandwich_norm(x, y, post_w=post_w, w=w), Fz.rope_axes(q, k, pos, (128,), q_w=q_w, k_w=k_w))
    ups = torch.ones_like(outs[0][0]), torch.ones_like(outs[1][0])
    total = torch.cuda.mem_get_info()[1]
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    try:
        torch.cuda.set_per_process_memory_fraction(torch.cuda.memory_reserved() / total)  # 64 MB gradients do not fit
        for o, up in zip(outs, ups):
            with pytest.raises(torch.OutOfMemoryError):
                torch.autograd.backward(o, [up, up], retain_graph=True)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert all(t.grad is None for t in (post_w, w, q_w, k_w))
    for o, up in zip(outs, ups):
        torch.autograd.backward(o, [up, up])
    # rows of zeros: the norm of the sum is 0, and with it every gradient of a weight
    assert all((t.grad == 0).all() for t in (post_w, w, q_w, k_w))
