"""Edges of the routed block's operators that need no GPU: the CPU definitions at special values, and what the modules do on a
machine without the compiled extension."""
import math

import pytest
import torch

from trenowanie_generatora_obrazkow_b200.ops import routing as Rt


def test_sigmoid_scores_at_special_logits():
    """Scores of far negative logits stay apart; the gradient at 0 is 1/4 and at -inf and inf 0."""
    low = torch.tensor([[-103.0, -102.0, -101.5, -101.0, -104.0, -200.0, -math.inf, -103.5]])
    assert Rt.route_experts(low, 3, score="sigmoid")[1].tolist() == [[3, 2, 1]]
    x = torch.tensor([[0.0, -math.inf, math.inf, -100.0]], requires_grad=True)
    w, idx = Rt.route_experts(x, 4, score="sigmoid", renorm=False)
    w.sum().backward()
    assert idx.tolist() == [[2, 0, 3, 1]] and w[0, :2].tolist() == [1.0, 0.5] and 0 < w[0, 2] < 1e-43
    assert x.grad[0, :3].tolist() == [0.25, 0.0, 0.0] and 0 < x.grad[0, 3] < 1e-43
