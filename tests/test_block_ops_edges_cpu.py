"""Edges of the routed block's operators that need no GPU: the CPU definitions at special values, and what the modules do on a
machine without the compiled extension."""
import math
import sys
import types

import pytest
import torch

import trenowanie_generatora_obrazkow_b200 as package
from trenowanie_generatora_obrazkow_b200.ops import _ext
from trenowanie_generatora_obrazkow_b200.ops import fused as Fz
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


def test_grad_ready_hooks_do_not_load_the_extension(monkeypatch):
    """CPU training on a GPU machine without a built extension keeps its hooks; the extension hears of them when it is
    loaded, and of every change after that."""
    name = package.__name__ + "._C"
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(_ext, "_C", None)
    monkeypatch.delattr(package, "_C", raising=False)
    monkeypatch.setitem(sys.modules, name, None)  # importing it fails
    heard = []
    hook = Fz.add_grad_ready_hook(heard.append)
    try:
        with pytest.raises(ImportError, match="not built"):
            _ext.ext()
        told = []
        built = types.ModuleType(name)
        built.set_grad_ready = lambda on, notify: told.append((on, notify))
        monkeypatch.setitem(sys.modules, name, built)
        assert _ext.ext() is built and told[-1][0] is True
        p = torch.zeros(1)
        told[-1][1](p)
        assert heard == [p]
    finally:
        Fz.remove_grad_ready_hook(hook)
    assert told[-1][0] is False


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("scale", [0.0, 1e-50, -1e-39, 1e39, math.inf, math.nan])
def test_scale_that_fp32_does_not_hold_is_refused(device, scale):
    """The weights' gradient is divided by the scale in 32 bits."""
    logits = torch.randn(2, 8, device=device)
    with pytest.raises(ValueError, match="scale"):
        Rt.route_experts(logits, 2, scale=scale)
    assert Rt.route_experts(logits, 2, scale=-2.0 ** -126)[0].shape == (2, 2)
