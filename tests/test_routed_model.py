"""The routed video DiT (models/routed.py) on the CPU: the routed MLP against every token through its experts, padding,
balance, and a short training run of the example."""
import pytest
import torch
import torch.nn.functional as F

import routed_video
from trenowanie_generatora_obrazkow_b200.models.routed import RoutedConfig, RoutedDenoiser, RoutedMLP


def dense(mlp, h):
    x = h.reshape(-1, mlp.dim)
    w, idx = mlp.route(x)
    out = torch.zeros_like(x)
    for e in range(mlp.E):
        a, b = (x @ mlp.w_in[e].T).chunk(2, -1)
        y = (F.silu(a) * b) @ mlp.w_out[e].T
        out = out + y * (w * (idx == e)).sum(1, keepdim=True)
    return out.view(h.shape)


@pytest.mark.parametrize("score,groups,top", [("softmax", 1, 1), ("sigmoid", 4, 2)])
def test_routed_mlp_matches_dense(score, groups, top):
    torch.manual_seed(0)
    mlp = RoutedMLP(24, 16, experts=8, top_k=3, score=score, groups=groups, top_groups=top, scale=1.5,
                    capacity_factor=8.0)
    h = torch.randn(2, 15, 24, requires_grad=True)
    out, want = mlp(h), dense(mlp, h)
    assert torch.allclose(out, want, atol=1e-5)
    g = torch.randn_like(out)
    params = [h, mlp.router.weight, mlp.w_in, mlp.w_out]
    for a, b in zip(torch.autograd.grad(out, params, g), torch.autograd.grad(want, params, g)):
        assert torch.allclose(a, b, atol=1e-4)
    with torch.no_grad():  # packed inference
        assert torch.allclose(mlp(h), want, atol=1e-5)
        assert torch.allclose(mlp(h[:1, :1]), want[:1, :1], atol=1e-5)  # one token
        valid = torch.ones(2, 15, dtype=torch.bool)
        valid[1, 9:] = False
        out = mlp(h, valid)
        assert torch.allclose(out[valid], want[valid], atol=1e-5) and (out[~valid] == 0).all()
        assert mlp.counts.sum() == valid.sum() * 3


def test_balance_moves_load():
    torch.manual_seed(1)
    mlp = RoutedMLP(16, 8, experts=8, top_k=1)
    h = torch.randn(400, 16) + 0.5
    with torch.no_grad():
        mlp(h)
        before = mlp.counts.float().max()
        for _ in range(200):
            mlp.update_balance(2e-3)
            mlp(h)
    assert mlp.counts.float().max() < before and mlp.balance.abs().sum() > 0


def test_example_trains_and_samples():
    losses, z = routed_video.main("--dim 64 --depth 2 --experts 4 --steps 30 --frames 2 --height 4 --width 4 --batch 2 "
                                  "--lr 3e-3 --device cpu".split())
    assert torch.isfinite(losses).all() and losses[-5:].mean() < losses[:5].mean()
    assert z.shape == (1, 16, 2, 4, 4) and torch.isfinite(z).all()


@pytest.mark.gpu
def test_routed_denoiser_gpu_matches_cpu():
    """Forward and parameter gradients in bf16 against the CPU's fp32; 2 % / 6 %: bf16 activations through two blocks."""
    torch.manual_seed(2)
    # one group, all experts chosen: rounding cannot move a token to another expert
    cfg = RoutedConfig(latent_channels=16, dim=256, depth=2, heads=4, kv_heads=2, axes=(16, 24, 24), text_dim=64,
                       experts=4, top_k=4, expert_hidden=128, groups=1, top_groups=1, capacity_factor=1.0, res_scale=0.7)
    cpu, gpu = RoutedDenoiser(cfg), RoutedDenoiser(cfg).cuda()
    with torch.no_grad():
        for b in cpu.blocks:
            b.mod_table.normal_(std=0.5)
    gpu.load_state_dict(cpu.state_dict())
    z, t, text = torch.randn(2, 16, 3, 5, 7), torch.rand(2), torch.randn(2, 6, 64)
    tl = torch.tensor([6, 3])
    g = torch.randn_like(z)
    rel = lambda a, b: ((a.float().cpu() - b).norm() / b.norm()).item()
    want = cpu(z, t, text, tl)
    want.backward(g)
    got = gpu(z.cuda(), t.cuda(), text.cuda(), tl.cuda())
    got.backward(g.cuda().to(got.dtype))
    assert rel(got, want.detach()) < 2e-2
    for (n, a), (_, b) in zip(gpu.named_parameters(), cpu.named_parameters()):
        if b.grad is not None and b.grad.norm() > 1e-6:
            assert a.grad is not None and rel(a.grad, b.grad) < 6e-2, n
    with torch.no_grad():
        assert rel(gpu(z.cuda(), t.cuda(), text.cuda(), tl.cuda()), want.detach()) < 2e-2


@pytest.mark.gpu
def test_example_and_recompute_on_the_gpu():
    """The example runs; selective recomputation gives the same gradients; grad-ready hooks see the norm weights."""
    from trenowanie_generatora_obrazkow_b200.ops import fused as Fz
    args = routed_video.parse("--steps 6 --frames 2 --height 6 --width 10 --dim 256 --depth 2".split())
    model = routed_video.make_model(args)
    losses = routed_video.train(model, args, log=lambda *_: None)
    z = routed_video.sample(model, args, 3)
    assert torch.isfinite(losses).all() and torch.isfinite(z).all()
    blk = model.blocks[0]
    x = torch.randn(2, 40, 256, device="cuda").bfloat16()
    t6, text = torch.randn(2, 6, 256, device="cuda").bfloat16() * 0.1, torch.randn(2, 8, 64, device="cuda").bfloat16()
    pos = model.positions(2, 2, 4, 5, "cuda")
    pending = (torch.randn_like(x), torch.randn(2, 256, device="cuda").bfloat16(), torch.ones(256, device="cuda"))
    seen, grads = [], []
    hook = Fz.add_grad_ready_hook(lambda p: seen.append(id(p)))
    try:
        for mode in (None, "selective"):
            model.zero_grad(set_to_none=True)
            xx = x.clone().requires_grad_()
            out, (branch, _, _) = Fz.run_block(blk, (xx, pending, t6, text, None, pos), mode)
            (out.float().square().sum() + branch.float().square().sum()).backward()
            grads.append([xx.grad] + [p.grad for p in blk.parameters()])
    finally:
        Fz.remove_grad_ready_hook(hook)
    for p in (blk.norm1.weight, blk.post1.weight, blk.norm3.weight, blk.q_norm.weight):
        assert seen.count(id(p)) == 2
    for a, b in zip(*grads):
        if a is not None:
            assert torch.allclose(a.float(), b.float(), rtol=2e-2, atol=2e-2 * a.float().abs().max().item())
