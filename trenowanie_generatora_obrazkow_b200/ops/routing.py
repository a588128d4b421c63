"""Routing of tokens to experts and the way of their rows there and back (csrc/route.cu, csrc/dispatch.cu).

    w, idx = route_experts(logits, k, score="sigmoid", bias=bias, groups=8, top_groups=4)
    plan   = expert_plan(idx, experts)                    # or capacity=C: static [experts * C] rows, overflow dropped
    xs     = expert_dispatch(x, plan)                     # [rows, D], experts' rows contiguous
    y      = ... the experts' products (ops/gemm.py: gemm_grouped(xs, w, plan.offsets), or a batched gemm) ...
    out    = expert_combine(y, w, plan)                   # [N, D]

Differentiable in the logits, x, y and w; nothing here synchronises with the host. CUDA tensors run the sm_100a
kernels, CPU tensors the fp32 definitions of ``reference.py`` under ordinary autograd.
"""
from typing import NamedTuple

import torch

from . import reference as R
from ._ext import ext

MAX_EXPERTS, MAX_CHOICES, MAX_GROUPS = 512, 32, 32


class ExpertPlan(NamedTuple):
    """Rows of the assignments in expert order: slot int32 [N, k] (-1: no row), offsets int32 [E + 1] (expert e owns rows
    offsets[e]..offsets[e + 1]), counts int32 [E] (assignments per expert, dropped ones included), capacity (0: packed)
    and the number of rows (N k packed, E capacity otherwise)."""
    slot: torch.Tensor
    offsets: torch.Tensor
    counts: torch.Tensor
    capacity: int
    rows: int


def route_experts(logits, k, score="softmax", bias=None, groups=1, top_groups=1, renorm=True, scale=1.0, valid=None):
    """Choose k experts for every token: logits [N, E] (fp32, bf16 or fp16) -> (w fp32 [N, k], idx int32 [N, k]).

    Scores are softmax(logits) or sigmoid(logits). The choice goes by the logits (softmax) or the scores (sigmoid), plus
    ``bias`` [E] fp32 (for balance: it moves the choice, not the weights), in descending order, ties to the lowest
    index. groups > 1: only the ``top_groups`` best of the ``groups`` equal runs of experts take part, a group's worth
    being its best expert (softmax) or the sum of its two best (sigmoid). renorm divides the weights by their sum
    (+ 1e-20); ``scale`` (a normal fp32 number) multiplies them. valid [N] bool: False rows get w 0 and idx -1. NaN logits
    are chosen last and count as -inf for their group; the weights of their row are unspecified. The gradient reaches the
    logits through the weights (once; forward-mode derivatives are refused)."""
    if score not in ("softmax", "sigmoid"):
        raise ValueError(f"route_experts: score is 'softmax' or 'sigmoid', not {score!r}")
    if logits.dim() != 2:
        raise ValueError("route_experts: logits [N, E] expected")
    E = logits.shape[1]
    if not (1 <= E <= MAX_EXPERTS and 1 <= groups <= MAX_GROUPS and E % groups == 0 and 1 <= top_groups <= groups
            and 1 <= k <= min(MAX_CHOICES, top_groups * (E // groups))):
        raise ValueError(f"route_experts: {E} experts, groups={groups}, top_groups={top_groups}, k={k} (at most "
                         f"{MAX_EXPERTS} experts in equal groups, k at most {MAX_CHOICES} and the kept groups' experts)")
    if not 2.0 ** -126 <= abs(scale) < 2.0 ** 128:
        raise ValueError(f"route_experts: scale is a normal fp32 number and not zero, not {scale}")
    if not logits.is_cuda:
        return R.route_experts(logits, k, score, bias, groups, top_groups, renorm, scale, valid)
    return ext().route_experts(logits, bias, valid, k, score == "sigmoid", groups, top_groups, renorm, scale)


def expert_plan(idx, experts, capacity=None):
    """Rows of the assignments idx int [N, k] (outside 0 .. experts - 1: none) in expert order, token order within an
    expert. capacity: every expert owns that many rows and later assignments are dropped (their slot is -1); None: packed
    without gaps."""
    if idx.dim() != 2 or not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"expert_plan: idx [N, k] and 1 to {MAX_EXPERTS} experts")
    if capacity is not None and capacity < 1:
        raise ValueError("expert_plan: capacity of at least 1 row")
    cap = int(capacity or 0)
    if not idx.is_cuda:
        slot, offsets, counts = R.expert_plan(idx, experts, cap)
    else:
        if idx.dtype is not torch.int32 or not idx.is_contiguous():
            if idx.dtype is torch.int64:  # what does not fit 32 bits is no expert
                idx = idx.clamp(-1, experts)
            idx = idx.to(torch.int32).contiguous()
        slot, offsets, counts = ext().expert_plan(idx, experts, cap)
    return ExpertPlan(slot, offsets, counts, cap, experts * cap if cap else idx.numel())


def expert_dispatch(x, plan):
    """x [N, D] -> [plan.rows, D]: the row of every assignment's token at its slot, zeros in unused rows."""
    if x.dim() != 2 or x.shape[0] != plan.slot.shape[0]:
        raise ValueError(f"expert_dispatch: x [{plan.slot.shape[0]}, D] expected, got {tuple(x.shape)}")
    if not x.is_cuda:
        return R.expert_dispatch(x, plan)
    return ext().dispatch_rows(x, *plan)


def expert_combine(y, w, plan):
    """y [plan.rows, D], w fp32 [N, k] -> [N, D]: the weighted sum of every token's rows (fp32 sum, one rounding);
    dropped assignments add nothing."""
    if y.dim() != 2 or y.shape[0] != plan.rows or w.shape != plan.slot.shape:
        raise ValueError(f"expert_combine: y [{plan.rows}, D] and w {tuple(plan.slot.shape)} expected, got "
                         f"{tuple(y.shape)} and {tuple(w.shape)}")
    if not y.is_cuda:
        return R.expert_combine(y, w, plan)
    return ext().combine_rows(y, w, *plan[:4])
