"""Edges of the routed block's operators that need no GPU: the CPU definitions at special values, and what the modules do on a
machine without the compiled extension."""
import math
import os
import socket
import sys
import tempfile
import types

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

import trenowanie_generatora_obrazkow_b200 as package
from trenowanie_generatora_obrazkow_b200.models.routed import RoutedConfig, RoutedDenoiser, RoutedMLP
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


def _balance_model():
    torch.manual_seed(3)
    cfg = RoutedConfig(latent_channels=4, dim=32, depth=2, heads=2, kv_heads=2, axes=(4, 6, 6), text_dim=8, experts=8,
                       top_k=2, expert_hidden=16, groups=1, top_groups=1)
    return RoutedDenoiser(cfg), RoutedMLP(16, 8, experts=8, top_k=1)


def _balance_inputs():
    g = torch.Generator().manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=g)
    return rnd(4, 4, 2, 3, 5), torch.rand(4, generator=g), rnd(4, 3, 8), rnd(4, 50, 16) + 0.5


def _balance_steps(rows):
    model, mlp = _balance_model()
    z, t, text, h = (x[rows] for x in _balance_inputs())
    with torch.no_grad():
        for _ in range(5):
            model(z, t, text)
            mlp(h)
            model.update_balance(0.05)
            mlp.update_balance(0.05)
    return torch.stack([*(b.mlp.balance for b in model.blocks), mlp.balance])


def _balance_worker(rank, world, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    n = 4 // world
    torch.save(_balance_steps(slice(rank * n, rank * n + n)), os.path.join(out, f"{rank}.pt"))
    dist.destroy_process_group()


def test_balance_is_that_of_all_ranks():
    """Two ranks with half of the samples each move the balance bias as one process with all of them."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    with tempfile.TemporaryDirectory() as out:
        mp.spawn(_balance_worker, args=(2, port, out), nprocs=2, join=True)
        a, b = (torch.load(os.path.join(out, f"{r}.pt")) for r in range(2))
    want = _balance_steps(slice(None))
    assert want.abs().sum() > 0 and torch.equal(a, b) and torch.allclose(a, want, atol=1e-6)


both_devices = pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])


@both_devices
def test_empty_rows_of_any_stride(device):
    """Empty tensors that are expanded or transposed are taken like contiguous ones."""
    plan = Rt.expert_plan(torch.zeros(0, 2, device=device, dtype=torch.int32), 8, capacity=4)
    empty = torch.zeros(1, 1, device=device).expand(0, 64)
    pos = torch.zeros(2, 0, 1, device=device, dtype=torch.int32)
    for x in (empty, torch.zeros(64, 0, device=device).t()):
        assert Rt.route_experts(x, 2)[0].shape == (0, 2) and Rt.expert_dispatch(x, plan).shape == (32, 64)
        h = Fz.sandwich_norm(x.view(0, 3, 64), x.view(0, 3, 64), gate=x, w=torch.ones(64, device=device))[1]
        q = x.view(2, 0, 64).unflatten(-1, (4, 16)).transpose(0, 1).transpose(0, 1)
        assert h.shape == (0, 3, 64) and Fz.rope_axes(q, q, pos, (16,))[0].shape == (2, 0, 4, 16)


@both_devices
def test_experts_of_no_tokens(device):
    """Empty results and gradients, unfilled rows of 0."""
    idx = torch.zeros(0, 2, device=device, dtype=torch.int32)
    x, w = torch.zeros(0, 64, device=device, requires_grad=True), torch.zeros(0, 2, device=device, requires_grad=True)
    for cap, rows in ((4, 32), (None, 0)):
        plan = Rt.expert_plan(idx, 8, capacity=cap)
        xs = Rt.expert_dispatch(x, plan)
        out = Rt.expert_combine(xs, w, plan)
        assert xs.shape == (rows, 64) and (xs == 0).all() and (plan.counts == 0).all() and out.shape == (0, 64)
        out.sum().backward()
    assert x.grad.shape == x.shape and w.grad.shape == w.shape


@both_devices
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_routing_of_no_tokens(device, score):
    logits = torch.zeros(0, 8, device=device, requires_grad=True)
    w, idx = Rt.route_experts(logits, 2, score=score)
    w.sum().backward()
    assert w.shape == idx.shape == (0, 2) and logits.grad.shape == (0, 8)


no_tokens = pytest.mark.parametrize("B,T", [(2, 0), (0, 5)])


@both_devices
@no_tokens
@pytest.mark.parametrize("parts", ["all", "no modulation", "no h"])
def test_sandwich_norm_of_no_tokens(device, B, T, parts):
    """Empty results, gradients of 0 for the rows of a sample and for the weights."""
    x, y = (torch.zeros(B, T, 64, device=device, requires_grad=True) for _ in range(2))
    post_w, w = (torch.ones(64, device=device, requires_grad=True) for _ in range(2))
    mods = [torch.ones(B, 64, device=device, requires_grad=True) for _ in range(3)]
    if parts == "all":
        outs = Fz.sandwich_norm(x, y, mods[0], post_w, w, *mods[1:])
    elif parts == "no modulation":
        outs = Fz.sandwich_norm(x, y, None, post_w, w)
    else:
        outs = Fz.sandwich_norm(x, y, mods[0], post_w)[:1]
    torch.autograd.backward(outs, [torch.ones_like(o) for o in outs])
    assert all(o.shape == (B, T, 64) for o in outs) and x.grad.shape == y.grad.shape == x.shape
    assert all(t.grad is None or (t.grad == 0).all() for t in (post_w, w, *mods))


@both_devices
@no_tokens
def test_rope_axes_of_no_tokens(device, B, T):
    q, k = (torch.zeros(B, T, h, 64, device=device, requires_grad=True) for h in (4, 1))
    w = torch.ones(64, device=device, requires_grad=True)
    outs = Fz.rope_axes(q, k, torch.zeros(B, T, 1, device=device, dtype=torch.int32), (64,), q_w=w, k_w=w)
    torch.autograd.backward(outs, [torch.ones_like(o) for o in outs])
    assert outs[0].shape == q.grad.shape == q.shape and (w.grad == 0).all()


@both_devices
@no_tokens
def test_axes_attention_of_no_tokens(device, B, T):
    qkv = torch.zeros(B, T, 6 * 64, device=device, dtype=torch.bfloat16 if device == "cuda" else torch.float32,
                      requires_grad=True)
    pos = torch.zeros(B, T, 1, device=device, dtype=torch.int32)
    w = torch.ones(64, device=device, requires_grad=True)
    o = Fz.axes_attention_core(qkv, pos, (64,), 4, 1, 64, q_w=w, k_w=w)
    o.backward(torch.ones_like(o))
    assert o.shape == (B, T, 256) and qkv.grad.shape == qkv.shape and (w.grad is None or (w.grad == 0).all())


@pytest.mark.parametrize("name", ["w_in", "w_out", "router.weight"])
def test_routed_mlp_trains_each_weight_alone(name):
    """With every other weight frozen and an input without gradients, the one that is left gets the same gradient."""
    torch.manual_seed(5)
    mlp, h, up = RoutedMLP(16, 8, experts=4, top_k=2, capacity_factor=4.0), torch.randn(10, 16), torch.randn(10, 16)
    mlp(h).backward(up)
    want = dict(mlp.named_parameters())[name].grad
    mlp.zero_grad(set_to_none=True)
    for n, p in mlp.named_parameters():
        p.requires_grad_(n == name)
    mlp(h).backward(up)
    assert want.norm() > 0 and torch.allclose(dict(mlp.named_parameters())[name].grad, want, atol=1e-6)
