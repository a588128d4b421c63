"""Values at the edges of the routed block's operators on the GPU (NaN inside a group of experts, weights that fill two
places, lengths and sizes at the limits), each against the definition in 64 bits or the rule that the docstrings state.
"""
import math

import pytest
import test_block_ops_gpu as plain
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


@pytest.mark.parametrize("E", [8, 12, 64, 256, 500])
def test_sigmoid_tells_far_negative_logits_apart(E):
    """Logits from -86 to -101 (scores down to 2^-146): the choice goes by the logits, not by the index. Scores below 2^-126
    are whole multiples of 2^-149."""
    logits = torch.full((40, E), -math.inf, device="cuda")
    rows = torch.arange(40, device="cuda")
    for i in range(8):
        logits[rows, (rows * 5 + i * 3) % 8] = -101.0 + 2 * i + rows / 80
    k = 4
    w, idx = Rt.route_experts(logits, k, score="sigmoid", renorm=False)
    want = logits.double().topk(k).indices
    assert torch.equal(idx.long(), want)
    p = torch.sigmoid(logits.double()).gather(1, want)
    assert ((w.double() - p).abs() <= p * 2.0 ** -20 + 2.0 ** -149).all()
    assert torch.equal(R.route_experts(logits, k, "sigmoid")[1], idx)
    assert torch.equal(R.route_experts(logits.cpu(), k, "sigmoid")[1], idx.cpu())
    low = torch.tensor([[-103.0, -102.0, -101.5, -101.0, -104.0, -200.0, -math.inf, -103.5]], device="cuda")
    assert Rt.route_experts(low, 3, score="sigmoid")[1].tolist() == [[3, 2, 1]]


@pytest.mark.parametrize("E,k", [(8, 2), (40, 3), (256, 8), (500, 32)])
def test_gradient_of_nearly_impossible_choices(E, k):
    """softmax, renormalised, and a bias that moves the choice to experts of a probability near 1e-20: the + 1e-20 of the
    divisor takes part, and the gradient reaches the experts that hold the probability. Tolerance: 64 fp32 roundings of
    the terms w |dw - m| and scale m, relative to the largest term of the row."""
    g = gen(44)
    N = 60
    logits = rnd(g, N, E)
    logits[:, : E // 4] += torch.linspace(0, 90, N, device="cuda")[:, None]  # chosen sums from all of it to 1e-39
    logits[::7, -1] = -math.inf
    bias = torch.zeros(E, device="cuda")
    bias[: E // 4] = -1000.0
    dw = rnd(g, N, k)
    x, y = logits.clone().requires_grad_(), logits.double().requires_grad_()
    w, idx = Rt.route_experts(x, k, bias=bias, scale=2.5)
    w64, want = R.route_experts(y, k, "softmax", bias.double(), scale=2.5)
    assert torch.equal(idx, want) and (idx >= E // 4).all()
    w.backward(dw)
    w64.backward(dw.double())
    assert (y.grad[:, : E // 4].abs().amax(1) > 1e-3).any()  # rows where it matters are among them
    terms = 2.5 * dw.double().abs().amax(1, keepdim=True) * (w64.detach().sum(1, keepdim=True) / 2.5)
    assert ((w.double() - w64).abs() <= 64 * 2.0 ** -24 * w64 + 1e-30).all()
    assert ((x.grad.double() - y.grad).abs() <= 64 * 2.0 ** -24 * terms + 1e-30).all()


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.int16])
def test_plan_of_numbers_that_are_no_expert(dtype):
    """Whatever lies outside 0 .. experts - 1 takes no row, in wide types too."""
    info = torch.iinfo(dtype)
    idx = torch.tensor([[0, 3], [4, -1], [info.max, info.min], [1, min(info.max, 2 ** 32 + 1)], [min(info.max, 2 ** 32), 2]],
                       dtype=dtype)
    plan = Rt.expert_plan(idx.cuda(), 4)
    slot, offsets, counts = R.expert_plan(idx, 4)
    assert torch.equal(plan.slot.cpu(), slot) and torch.equal(plan.counts.cpu(), counts)
    assert plan.counts.tolist() == [1, 1, 1, 1] and torch.equal(plan.offsets.cpu(), offsets)


@pytest.mark.parametrize("N,E,k,cap", [(1023, 64, 2, None), (1024, 64, 2, None), (1025, 64, 2, 30), (2049, 8, 1, None),
                                       (683, 512, 3, 4), (2000, 256, 2, None), (4096, 7, 2, 1100)])
def test_plan_on_both_sides_of_the_cluster(N, E, k, cap):
    """One CTA up to 2048 assignments, a cluster above: the same stable order."""
    idx = plain.choices(gen(48), N, E, k, 0.1)
    plan = Rt.expert_plan(idx, E, capacity=cap)
    slot, offsets, counts = R.expert_plan(idx.cpu(), E, cap or 0)
    assert torch.equal(plan.slot.cpu(), slot) and torch.equal(plan.offsets.cpu(), offsets)
    assert torch.equal(plan.counts.cpu(), counts)


# ----------------------------------------------------------------------------------------------------------------
# rotary positions
# ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("d,axes,norm,interleaved,dtype", [(776, (768,), True, True, F32), (1024, (512, 256), True, False, BF16),
                                                           (1024, (1024,), False, True, F32), (1023, (10,), True, True, F32)])
def test_rope_axes_of_the_widest_heads(d, axes, norm, interleaved, dtype):
    """Head dims up to 1024, forward and backward. Each output is rounded once (half a unit of its type, doubled) and
    carries at most 64 fp32 roundings of its largest terms: a pair's two products and the norm's mean over d channels."""
    g = gen(43)
    unit = {BF16: 2.0 ** -8, F32: 2.0 ** -23}[dtype]
    q, k, dq, dk = (rnd(g, 2, 9, h, d, dtype=dtype) for h in (3, 1, 3, 1))
    pos = torch.randint(0, 64, (2, 9, len(axes)), device="cuda", generator=g).int()
    ws = [rnd(g, d, std=0.1, mean=1.0) for _ in range(2)] if norm else [None, None]
    leaf = [t.clone().requires_grad_() if t is not None else None for t in (q, k, *ws)]
    wide = [t.double().requires_grad_() if t is not None else None for t in (q, k, *ws)]
    out = Fz.rope_axes(*leaf[:2], pos, axes, q_w=leaf[2], k_w=leaf[3], interleaved=interleaved)
    want = R.rope_axes(*wide[:2], pos, axes, q_w=wide[2], k_w=wide[3], interleaved=interleaved)
    torch.autograd.backward(list(out), [dq, dk])
    torch.autograd.backward(list(want), [dq.double(), dk.double()])
    for a, b in list(zip(out, want)) + [(a.grad, b.grad) for a, b in zip(leaf[:2], wide[:2])]:
        assert (a.double() - b).abs().max() <= (unit + 64 * 2.0 ** -24) * 2 * b.abs().max()
    for a, b in zip(leaf[2:], wide[2:]):  # sums over 18 or 54 rows
        assert a is None or (a.grad.double() - b.grad).norm() <= 64 * 2.0 ** -24 * 54 ** 0.5 * b.grad.norm()


@pytest.mark.parametrize("d", [64, 50])
def test_rope_axes_at_the_last_positions(d):
    """Integer positions up to 2^24 and fractional ones, fastest pairs included: angles to 2^-22 of a revolution (the
    two-part frequency's rest, 2^-48 relative to the first part, times 2^24 turns, and fp32 roundings of a fraction)."""
    g = gen(47)
    q = torch.ones(1, 4000, 1, d, device="cuda")
    pos = torch.randint(0, 2 ** 24, (1, 4000, 1), device="cuda", generator=g).int()
    pos[0, :4, 0] = torch.tensor([0, 1, 2 ** 24 - 1, -2 ** 24 + 1])
    for p in (pos, torch.rand(1, 4000, 1, device="cuda", generator=g) * 1000, pos.float()):
        got, _ = Fz.rope_axes(q, q, p, (d,), theta=1e4)
        want, _ = R.rope_axes(q.double(), q.double(), p, (d,), theta=1e4)
        assert (got.double() - want).abs().max() <= 2 ** 0.5 * 2 * math.pi * 2.0 ** -22 + 2.0 ** -22


# (B, T, Hq, Hkv, d, axes, interleaved, norm, kv_len, positions): one token, masked tails, a sample without keys, shared
# heads, partial rotation
@pytest.mark.parametrize("B,T,hq,hkv,d,axes,inter,norm,lens,frac", [
    (2, 77, 4, 2, 64, (16, 24, 24), True, True, (77, 30), False), (1, 130, 2, 2, 128, (64, 64), False, True, None, True),
    (3, 64, 6, 2, 128, (32, 32), False, False, (64, 1, 0), False), (2, 1, 4, 1, 64, (64,), False, True, None, False),
    (2, 33, 3, 3, 64, (20,), True, False, (33, 0), True), (1, 257, 8, 8, 128, (16, 56, 56), False, True, (200,), False)])
def test_axes_attention_core(B, T, hq, hkv, d, axes, inter, norm, lens, frac):
    """Forward and gradients against the 64-bit definition. q and k after the rotation, the probabilities and the output are
    rounded to bf16, in the backward dS and the gradients too: 2 % and 4 % of the norm, as for self_attention_core."""
    g = gen(50)
    qkv, up = rnd(g, B, T, (hq + 2 * hkv) * d, dtype=BF16), rnd(g, B, T, hq * d, dtype=BF16)
    ws = [rnd(g, d, std=0.1, mean=1.0) for _ in range(2)] if norm else [None, None]
    pos = torch.randint(0, 60, (B, T, len(axes)), device="cuda", generator=g)
    pos = pos.float() * 0.5 - 3.25 if frac else pos
    kv_len = None if lens is None else torch.tensor(lens, device="cuda", dtype=torch.int32)
    leaf = [t.clone().requires_grad_() if t is not None else None for t in (qkv, *ws)]
    out = Fz.axes_attention_core(leaf[0], pos, axes, hq, hkv, d, q_w=leaf[1], k_w=leaf[2], kv_len=kv_len, interleaved=inter)
    out.backward(up)
    wide = [t.double().requires_grad_() if t is not None else None for t in (qkv, *ws)]
    q, k, v = wide[0].view(B, T, hq + 2 * hkv, d).split([hq, hkv, hkv], dim=2)
    q, k = R.rope_axes(q, k, pos, axes, q_w=wide[1], k_w=wide[2], interleaved=inter)
    live = [b for b in range(B) if lens is None or lens[b] > 0]
    want = R.attention(q[live], k[live], v[live], None if lens is None else kv_len[live], d ** -0.5)
    want.backward(up[live].double().view(len(live), T, hq, d))
    want = want.detach().reshape(len(live), T, hq * d)
    rel = lambda a, b: ((a.double() - b).norm() / b.norm()).item()
    assert rel(out[live], want) < 2e-2 and rel(leaf[0].grad[live], wide[0].grad[live]) < 4e-2
    parts = zip(leaf[0].grad.view(B, T, -1, d).split([hq, hkv, hkv], 2), wide[0].grad.view(B, T, -1, d).split([hq, hkv, hkv], 2))
    for a, b in parts:  # dq, dk, dv (below: keys past kv_len get exactly nothing)
        assert b.norm() == 0 and a.norm() == 0 or rel(a, b) < 4e-2 or b.norm() < 1e-6 * wide[0].grad.norm()
    for b in live if lens is not None else []:
        assert (leaf[0].grad.view(B, T, -1, d)[b, lens[b]:, hq:] == 0).all()
    dead = [b for b in range(B) if b not in live]
    assert (out[dead] == 0).all() and (leaf[0].grad[dead] == 0).all()
    for a, b in zip(leaf[1:], wide[1:]):
        assert a is None or rel(a.grad, b.grad) < 4e-2 or b.grad.norm() < 1e-6 * wide[0].grad.norm()
    with torch.no_grad():
        again = Fz.axes_attention_core(qkv, pos, axes, hq, hkv, d, q_w=ws[0], k_w=ws[1], kv_len=kv_len, interleaved=inter)
    assert torch.equal(again, out)


# ----------------------------------------------------------------------------------------------------------------
# sandwich norm
# ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(1, 2 ** 31 - 1000, 1), (2 ** 20, 2 ** 11 - 1, 8), (2 ** 16, 2 ** 16, 8), (1, 4, 16385)])
def test_sandwich_norm_refuses_more_rows_than_it_counts(shape):
    """Rows are counted in 32 bits: sizes at that limit are refused before a copy or a launch (the inputs are expanded,
    so they take no memory)."""
    x = torch.zeros(1, 1, 1, device="cuda", dtype=BF16).expand(shape)
    w = torch.ones(1, device="cuda").expand(shape[2])
    Fz.err_buf("cuda")  # the device's error word is made once
    before = torch.cuda.memory_allocated()
    with pytest.raises(RuntimeError, match="rows"):
        Fz.sandwich_norm(x, x, w=w)
    assert torch.cuda.memory_allocated() == before


@pytest.mark.parametrize("B,T,D,post,gate,mod,pre,res,dtype", [
    (2, 10, 2560, True, True, True, True, 0.5, BF16), (3, 7, 2304, True, True, True, True, 1.0, F16),
    (2, 400, 2064, True, False, False, True, 1.0, BF16), (4, 90, 2560, True, True, True, True, 1.0, F32),
    (2, 31, 2056, False, True, True, True, 1.0, BF16), (2, 12, 2568, True, True, True, True, 1.0, F16)])
def test_sandwich_norm_of_2056_to_2560_channels(B, T, D, post, gate, mod, pre, res, dtype):
    """The widths whose backward takes one row per step, and one past them, against 64 bits."""
    plain.test_sandwich_norm(B, T, D, post, gate, mod, pre, res, dtype)


@pytest.mark.parametrize("B,T,D,post,gate,mod,pre,res,dtype", [
    (256, 2, 128, True, True, True, True, 1.0, BF16), (257, 1, 128, True, True, True, True, 1.0, BF16),
    (700, 3, 264, True, True, False, True, 0.5, F32), (513, 2, 577, True, False, True, True, 1.0, F16),
    (16500, 1, 64, True, True, True, True, 1.0, F32), (300, 2, 96, False, True, False, False, 1.0, F32)])
def test_sandwich_norm_of_many_samples(B, T, D, post, gate, mod, pre, res, dtype):
    """More than 256 gated or modulated samples: the weights' gradients are summed in groups of samples first."""
    plain.test_sandwich_norm(B, T, D, post, gate, mod, pre, res, dtype)


@pytest.mark.parametrize("B", [200, 700])
def test_sandwich_norm_of_many_samples_into_a_grad(B):
    """The same sums added to what .grad holds, with either weight left out. fp32; 1e-5 of the gradient's norm: sums of B 3
    products, 2^-24 of each and of the partial sums."""
    g = gen(49)
    ins = plain.sandwich_inputs(g, B, 3, 128, True, True, True, True, F32)
    up = [rnd(g, B, 3, 128) for _ in range(2)]
    d = {n: t.double().requires_grad_() for n, t in ins.items()}
    torch.autograd.backward(list(R.sandwich_norm(**d)), [u.double() for u in up])
    for only in ("both", "w", "post_w"):
        leaf = {n: t.clone().requires_grad_(n not in ("w", "post_w") or only in ("both", n)) for n, t in ins.items()}
        start = {n: rnd(g, 128) for n in ("w", "post_w") if leaf[n].requires_grad}
        for n, s in start.items():
            leaf[n].grad = s.clone()
        torch.autograd.backward(list(Fz.sandwich_norm(**leaf)), up)
        for n in ("w", "post_w"):
            if n in start:
                diff = leaf[n].grad.double() - start[n].double() - d[n].grad
                assert diff.norm() <= 1e-5 * (d[n].grad.norm() + start[n].norm())
            else:
                assert leaf[n].grad is None


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


@pytest.mark.parametrize("op", ["sandwich", "sandwich of 700 samples", "rope", "rope, any head dim", "attention"])
@pytest.mark.parametrize("given", ["none", "leaf", "twice"])
def test_one_leaf_in_both_weight_places(op, given):
    """A weight that serves as post_w and w, or as q_w and k_w: its gradient is the sum of both, also when .grad holds
    something already, and the ready hooks hear of it once. Tolerance: the sums of n fp32 products differ from the 64-bit
    ones by less than 1e-5 of their root sum of squares; bf16 attention in front of the weights' sums allows 2 %."""
    g = gen(41)
    tol = 2e-2 if op == "attention" else 1e-5
    d = {"sandwich": 256, "sandwich of 700 samples": 264, "rope": 64, "rope, any head dim": 50, "attention": 64}[op]
    weight = rnd(g, d, std=0.1, mean=1.0)
    if op.startswith("sandwich"):
        B, T = (3, 40) if op == "sandwich" else (700, 3)
        x, y, up = rnd(g, B, T, d), rnd(g, B, T, d), [rnd(g, B, T, d), rnd(g, B, T, d)]
        gate, shift, scale = (rnd(g, B, d, std=0.3) for _ in range(3))
        run = lambda w, p, c=lambda t: t: (p.sandwich_norm(c(x), c(y), c(gate), w, w, c(shift), c(scale)), [c(u) for u in up])
    elif op == "attention":
        qkv, up = rnd(g, 2, 70, 6 * d, dtype=BF16), [rnd(g, 2, 70, 4 * d, dtype=BF16)]
        pos = torch.randint(0, 50, (2, 70, 1), device="cuda", generator=g).int()

        def run(w, p, c=lambda t: t):
            if p is Fz:
                return [Fz.axes_attention_core(qkv.clone().requires_grad_(), pos, (d,), 4, 1, d, q_w=w, k_w=w)], up
            q, k, v = c(qkv).view(2, 70, 6, d).split([4, 1, 1], dim=2)
            q, k = R.rope_axes(q, k, pos, (d,), q_w=w, k_w=w)
            return [R.attention(q, k, v, None, d ** -0.5).reshape(2, 70, 4 * d)], [c(u) for u in up]
    else:
        q, k, up = rnd(g, 2, 33, 3, d), rnd(g, 2, 33, 1, d), [rnd(g, 2, 33, 3, d), rnd(g, 2, 33, 1, d)]
        pos = torch.randint(0, 50, (2, 33, 1), device="cuda", generator=g).int()
        run = lambda w, p, c=lambda t: t: (p.rope_axes(c(q), c(k), pos, (d // 2 // 2 * 2,), q_w=w, k_w=w), [c(u) for u in up])
    w64 = weight.double().requires_grad_()
    outs, ups = run(w64, R, lambda t: t.double())
    torch.autograd.backward(list(outs), ups)
    want = w64.grad
    start = torch.zeros(d, device="cuda")
    w = weight.clone().requires_grad_()
    if given != "none":
        w.grad = rnd(g, d)
        start = w.grad.clone()
    heard = []
    hook = Fz.add_grad_ready_hook(lambda p: heard.append(p))
    try:
        for _ in range(2 if given == "twice" else 1):
            outs, ups = run(w, Fz)
            torch.autograd.backward(list(outs), ups)
    finally:
        Fz.remove_grad_ready_hook(hook)
    want = want * (2 if given == "twice" else 1)
    size = want.norm()
    assert (w.grad.double() - start.double() - want).norm() <= tol * size, ((w.grad.double() - start - want).norm() / size)
    assert len(heard) == (2 if given == "twice" else 1) and all(p is w for p in heard)


def test_two_leaves_with_one_grad():
    """Two weights whose .grad is the same memory: both sums arrive there."""
    g = gen(42)
    x, y, up = rnd(g, 2, 30, 128), rnd(g, 2, 30, 128), rnd(g, 2, 30, 128)
    a, b = (rnd(g, 128, std=0.1, mean=1.0).requires_grad_() for _ in range(2))
    Fz.sandwich_norm(x, y, post_w=a, w=b)[1].backward(up)
    want = a.grad + b.grad
    both = torch.zeros(128, device="cuda")
    a.grad, b.grad = both, both.view(128)
    Fz.sandwich_norm(x, y, post_w=a, w=b)[1].backward(up)
    assert torch.allclose(both, want, rtol=1e-5, atol=1e-5 * want.abs().max().item())


def test_forward_mode_derivatives_are_refused():
    """Dual tensors: an error instead of results without their tangents, with and without requires_grad."""
    from torch.autograd import forward_ad
    g = gen(45)
    logits, x, w = rnd(g, 6, 8), rnd(g, 6, 16), torch.rand(6, 2, device="cuda", generator=g)
    plan = Rt.expert_plan(Rt.route_experts(logits, 2)[1], 8)
    y, q = rnd(g, plan.rows, 16), rnd(g, 2, 3, 2, 16)
    pos = torch.zeros(2, 3, 1, device="cuda", dtype=torch.int32)
    gate, weight = rnd(g, 2, 16), rnd(g, 16)
    x3 = x.view(2, 3, 16)
    calls = [(lambda t: Rt.route_experts(t, 2), logits), (lambda t: Rt.expert_dispatch(t, plan), x),
             (lambda t: Rt.expert_combine(t, w, plan), y), (lambda t: Rt.expert_combine(y, t, plan), w),
             (lambda t: Fz.sandwich_norm(t, x3, w=weight), x3), (lambda t: Fz.sandwich_norm(x3, x3, t, w=weight), gate),
             (lambda t: Fz.sandwich_norm(x3, x3, w=t), weight), (lambda t: Fz.rope_axes(t, q, pos, (16,)), q),
             (lambda t: Fz.rope_axes(q, q, pos, (16,), q_w=t, k_w=weight), weight)]
    for leaf in (False, True):
        with forward_ad.dual_level():
            for f, t in calls:
                dual = forward_ad.make_dual(t.clone().requires_grad_(leaf), torch.ones_like(t))
                with pytest.raises((RuntimeError, NotImplementedError)):
                    f(dual)
                with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError)):
                    f(dual)
    for f, t in calls:
        f(t)


def test_launch_counts_are_those_of_the_kernels():
    """The extension's launch counter against the kernels that torch's profiler sees."""
    from trenowanie_generatora_obrazkow_b200.ops._ext import ext
    g = gen(46)
    leaf = lambda *s: rnd(g, *s).requires_grad_()
    w, logits, pos = leaf(64), leaf(9, 8), torch.zeros(2, 3, 1, device="cuda", dtype=torch.int32)
    Fz.err_buf("cuda")

    def sandwich(B, T, weights, gate):
        x, y, m = leaf(B, T, 64), leaf(B, T, 64), leaf(B, 64)
        post_w, w = (leaf(64) if weights else torch.ones(64, device="cuda") for _ in range(2))
        a, h = Fz.sandwich_norm(x, y, m if gate else None, post_w=post_w, w=w)
        return lambda: torch.autograd.backward([a, h], [x.detach(), y.detach()])

    def rope(norm):
        q, k = leaf(2, 3, 4, 64), leaf(2, 3, 2, 64)
        a, b = Fz.rope_axes(q, k, pos, (64,), q_w=leaf(64) if norm else None, k_w=leaf(64) if norm else None)
        return lambda: torch.autograd.backward([a, b], [q.detach(), k.detach()])

    def rows(n, d, cap):
        plan = Rt.expert_plan(torch.zeros(n, 2, device="cuda", dtype=torch.int32), 4, capacity=cap)
        x, y, u = leaf(n, d), leaf(plan.rows, d), torch.ones(n, 2, device="cuda")

        def f():
            a, b = Rt.expert_dispatch(x, plan), Rt.expert_combine(y, u, plan)
            torch.autograd.backward([a, b], [y.detach(), x.detach()])
        return f
    cases = [sandwich(2, 8, True, True), sandwich(2, 8, False, True), sandwich(300, 2, True, True),
             sandwich(300, 2, False, True), sandwich(300, 2, True, False), rope(True), rope(False), rows(5, 16, None),
             rows(5, 16, 3), rows(0, 16, 3), rows(0, 16, None), rows(5, 0, None), lambda: Rt.route_experts(logits, 2),
             lambda: Rt.route_experts(logits[:0], 2), lambda: Fz.sandwich_norm(torch.zeros(0, 3, 64, device="cuda"),
                                                                               torch.zeros(0, 3, 64, device="cuda"), w=w)]
    for i, f in enumerate(cases):
        torch.cuda.synchronize()
        n0 = ext().launch_count()
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
            f()
            torch.cuda.synchronize()
        seen = sum(e.count for e in prof.key_averages() if "tgo::" in e.key)
        assert ext().launch_count() - n0 == seen, (i, ext().launch_count() - n0, seen)


def test_operators_in_a_graph():
    """Captured in a CUDA graph and replayed with other inputs in place: the results of plain calls."""
    g = gen(51)
    N, E, D = 300, 64, 256
    make = lambda: dict(logits=rnd(g, N, E), x=rnd(g, N, D, dtype=BF16), a=rnd(g, 2, 150, D, dtype=BF16),
                        b=rnd(g, 2, 150, D, dtype=BF16), gate=rnd(g, 2, D, dtype=BF16),
                        pos=torch.randint(0, 90, (2, 150, 2), device="cuda", generator=g).int())
    w, ones = rnd(g, D, std=0.1, mean=1.0), torch.ones(64, device="cuda")

    def run(i):
        r, idx = Rt.route_experts(i["logits"], 4, score="sigmoid", groups=8, top_groups=4)
        plan = Rt.expert_plan(idx, E)
        out = Rt.expert_combine(Rt.expert_dispatch(i["x"], plan), r, plan)
        x, h = Fz.sandwich_norm(i["a"], i["b"], i["gate"], w, w)
        q, k = Fz.rope_axes(h.unflatten(-1, (4, 64)), x.unflatten(-1, (4, 64)), i["pos"], (32, 32), q_w=ones, k_w=ones)
        return r, idx, plan.slot, plan.offsets, out, x, h, q, k
    state, other = make(), make()
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(state)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run(state)
        for name, t in other.items():
            state[name].copy_(t)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, run(other)))
