"""Models and commands on 8-bit products and with 8-bit activation checkpoints (CPU definitions)."""
import os
import socket
import subprocess
import sys

import pytest
import torch

from trenowanie_generatora_obrazkow_b200.models import DenoiserConfig, build_models
from trenowanie_generatora_obrazkow_b200.models.config import TE_SIZES
from trenowanie_generatora_obrazkow_b200.models.quant import BlockLinear, quantize, use_fp8
from trenowanie_generatora_obrazkow_b200.ops import blocks8 as B8
from trenowanie_generatora_obrazkow_b200.ops import fused as Fz

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _model():
    torch.manual_seed(0)
    te, den = build_models(DenoiserConfig(dim=128, depth=2, heads=2, mlp_hidden=384, text_dim=128, latent_size=4),
                           TE_SIZES["states-nano"], device="cpu")
    te.init_weights(), den.init_weights()
    with torch.no_grad():
        for p in list(te.parameters()) + list(den.parameters()):
            p.add_(0.05 * torch.randn_like(p))
    return te, den


def _step(te, den):
    g = torch.Generator().manual_seed(1)
    x, t, st = torch.randn(2, 128, 4, 4, generator=g), torch.rand(2, generator=g), torch.randn(2, 16, 64, generator=g)
    params = list(te.parameters()) + list(den.parameters())
    for p in params:
        p.grad = None
    text, valid = te(lm_states=st)
    out = den(x, t, text, valid)
    out.square().mean().backward()
    return out.detach(), [None if p.grad is None else p.grad.clone() for p in params]


def test_marked_blocks_run_on_8_bit_products():
    te, den = _model()
    plain, grads = _step(te, den)
    names = [n for n, _ in den.named_parameters()]
    use_fp8(te), use_fp8(den)
    assert den.blocks[0].mlp.in_proj.fp8 and "fp8" not in den.patch_in.__dict__
    assert [n for n, _ in den.named_parameters()] == names
    out, g8 = _step(te, den)
    # a value's error is at most 2^-4 of it; products of many add up like noise
    assert 0 < ((out - plain).norm() / plain.norm()).item() < 0.1
    assert [g is None for g in grads] == [g is None for g in g8]
    whole = torch.cat([g.flatten() for g in grads if g is not None]), torch.cat([g.flatten() for g in g8 if g is not None])
    assert ((whole[1] - whole[0]).norm() / whole[0].norm()).item() < 0.1
    with torch.no_grad():  # weights held in 8 bits: the same products
        text, valid = te(lm_states=torch.randn(2, 16, 64, generator=torch.Generator().manual_seed(2)))
        x = torch.randn(2, 128, 4, 4)
        first = den(x, torch.rand(2), text, valid)
        kept = den.blocks[0].attn.qkv.weight._tgo_fp8
        den(x, torch.rand(2), text, valid)
        assert den.blocks[0].attn.qkv.weight._tgo_fp8 is kept and torch.isfinite(first).all()
        den.blocks[0].attn.qkv.weight.mul_(2)
        den(x, torch.rand(2), text, valid)
        assert den.blocks[0].attn.qkv.weight._tgo_fp8 is not kept
    use_fp8(te, False), use_fp8(den, False)
    assert torch.equal(_step(*_model())[0], plain)


def test_marked_routed_blocks():
    from trenowanie_generatora_obrazkow_b200.models.routed import RoutedConfig, RoutedDenoiser
    torch.manual_seed(0)
    net = RoutedDenoiser(RoutedConfig(latent_channels=8, dim=128, depth=2, heads=2, kv_heads=2, axes=(16, 24, 24), text_dim=64,
                                      experts=8, top_k=2, expert_hidden=128, groups=2, top_groups=1, capacity_factor=8.0))
    z, t, text = torch.randn(2, 8, 2, 4, 4), torch.rand(2), torch.randn(2, 5, 64)

    def step():
        net.zero_grad()
        out = net(z, t, text)
        out.square().mean().backward()
        return out.detach(), torch.cat([p.grad.flatten() for p in net.parameters()])
    plain, grads = step()
    use_fp8(net)
    assert all(m.fp8 for b in net.blocks for m in (b.qkv, b.out, b.cross.q, b.cross.kv, b.cross.out))
    calls = []
    real, B8.linear_blocks = B8.linear_blocks, lambda *a: calls.append(a) or real(*a)
    try:
        out, g8 = step()
    finally:
        B8.linear_blocks = real
    assert len(calls) == 10
    # a value's error is at most 2^-4 of it; products of many add up like noise (a token at a border may take another expert)
    assert 0 < ((out - plain).norm() / plain.norm()).item() < 0.2
    assert g8.shape == grads.shape and g8.isfinite().all()


def test_held_weights_give_the_training_forward():
    lin = torch.nn.Linear(130, 48)
    lin.fp8 = True
    x = torch.randn(5, 130)
    y = Fz.linear(x, lin)
    with torch.no_grad():
        assert torch.equal(Fz.linear(x, lin), y)
    a, b = torch.nn.Linear(64, 256, bias=False), torch.nn.Linear(128, 32, bias=False)
    a.fp8 = b.fp8 = True
    x = torch.randn(5, 64)
    y = Fz.mlp_fp8(x, a, b)
    with torch.no_grad():
        assert torch.equal(Fz.mlp_fp8(x, a, b), y)


def test_checkpoint_mode_keeps_the_swiglu_in_8_bits():
    te, den = _model()
    plain, grads = _step(te, den)
    te.checkpoint_blocks = den.checkpoint_blocks = "fp8"
    out, g8 = _step(te, den)
    assert torch.equal(out, plain)  # the forward is the same
    for n, (a, b) in zip([n for n, _ in te.named_parameters()] + [n for n, _ in den.named_parameters()], zip(grads, g8)):
        if a is not None:
            assert ((a - b).norm() / a.norm().clamp_min(1e-12)).item() < 0.1, n
    assert Fz._PACK8_ACTIVE[0] == 0 and Fz._SAC_ACTIVE[0] == 0


def test_block_linear():
    m = torch.nn.Sequential(torch.nn.Linear(130, 64), torch.nn.GELU(), torch.nn.Linear(64, 8, bias=False))
    x = torch.randn(3, 7, 130)
    want = m(x)
    w = m[0].weight
    quantize(m, "fp8_block")
    assert isinstance(m[0], BlockLinear) and m[0].w.dtype == torch.float8_e4m3fn
    assert torch.equal(m[0](x), B8.linear_blocks(x, B8.quantize_blocks(w), m[0].bias.detach()))
    assert ((m(x) - want).norm() / want.norm()).item() < 0.1
    state = {k: v.clone() for k, v in m.state_dict().items()}
    m.load_state_dict(state)


def test_block_linear_refuses_an_input_that_wants_a_gradient():
    m = quantize(torch.nn.Sequential(torch.nn.Linear(130, 64)), "fp8_block")
    x = torch.randn(3, 130)
    leaf = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        m(leaf)
    with torch.no_grad():
        assert torch.equal(m(leaf), m(x))


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(), lambda m: m.type(torch.float32),
                                  lambda m: m.to("cpu", torch.float32), lambda m: m.to("meta").to_empty(device="cpu")])
def test_block_linear_keeps_its_codes_when_a_module_is_cast(cast):
    m = quantize(torch.nn.Sequential(torch.nn.Linear(130, 64)), "fp8_block")
    x, codes, scales = torch.randn(3, 130), m[0].w.clone(), m[0].s.clone()
    state = {k: v.clone() for k, v in m.state_dict().items()}
    assert cast(m) is m and m[0].w.dtype == torch.float8_e4m3fn and m[0].s.dtype == torch.uint8
    if not all(p.device.type == "cpu" and torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in ((m[0].w, codes), (m[0].s, scales))):
        m.load_state_dict(state)  # emptied on the way
    x, bias = x.to(m[0].bias.dtype if m[0].bias.dtype != torch.float64 else torch.float32), m[0].bias.detach()
    assert torch.equal(m[0](x), B8.linear_blocks(x, B8.Blocks8(codes, scales, 130), bias))


@pytest.mark.parametrize("kind", ["int8", "fp8", "w8a8", "fp8_block"])
@pytest.mark.parametrize("model", ["dit", "moe", "routed"])
def test_quantized_models(kind, model):
    """The framework's own models with every layer but the routers quantized."""
    from trenowanie_generatora_obrazkow_b200.models.moe import moe_denoiser
    from trenowanie_generatora_obrazkow_b200.models.routed import RoutedConfig, RoutedDenoiser
    g = torch.Generator().manual_seed(1)
    if model == "routed":
        torch.manual_seed(0)
        nets = [RoutedDenoiser(RoutedConfig(latent_channels=8, dim=128, depth=2, heads=2, kv_heads=2, axes=(16, 24, 24), text_dim=64,
                                            experts=8, top_k=2, expert_hidden=128, groups=2, top_groups=1))]
        z, t, text = torch.randn(2, 8, 2, 4, 4, generator=g), torch.rand(2, generator=g), torch.randn(2, 5, 64, generator=g)
        run = lambda: nets[0](z, t, text)  # noqa: E731
    else:
        nets = _model()
        if model == "moe":
            moe_denoiser(nets[1], 4, 2, 128)
        x, t, st = torch.randn(2, 128, 4, 4, generator=g), torch.rand(2, generator=g), torch.randn(2, 16, 64, generator=g)

        def run():
            text, valid = nets[0](lm_states=st)
            return nets[1](x, t, text, valid)
    with torch.no_grad():
        plain = run()
        for net in nets:
            quantize(net, kind)
            linears = [n for n, m in net.named_modules() if type(m) is torch.nn.Linear]
            assert all(n.endswith(".router") for n in linears) and (model == "dit" or net is not nets[-1] or linears)
        # a value's error is at most 2^-4 of it (less for the kinds of finer steps); products of many add up like noise
        assert 0 < ((run() - plain).norm() / plain.norm()).item() < 0.1


def test_quantized_blocks_are_the_marked_blocks():
    g = torch.Generator().manual_seed(1)
    x, t, text = torch.randn(2, 128, 4, 4, generator=g), torch.rand(2, generator=g), torch.randn(2, 9, 128, generator=g)
    marked, held = _model()[1], _model()[1]
    use_fp8(marked), quantize(held.blocks, "fp8_block")
    with torch.no_grad():
        assert torch.equal(marked(x, t, text), held(x, t, text))


@pytest.mark.parametrize("flags", [["--fp8"], ["--act-checkpoint", "fp8"], ["--fp8", "--act-checkpoint", "fp8"]])
def test_train_command(tmp_path, flags):
    r = subprocess.run([sys.executable, "train.py", "--synthetic", "16", "--out", str(tmp_path / "run"), "--size", "nano",
                        "--te-size", "13m", "--batch", "2", "--micro-batch", "2", "--steps", "1", "--eval-every", "0",
                        "--no-wandb", "--ckpt-every", "0"] + flags, cwd=ROOT, capture_output=True, text=True, timeout=600,
                       env=dict(os.environ, CUDA_VISIBLE_DEVICES=""))
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]


@pytest.mark.parametrize("opd", [False, True])
def test_pipeline_command(tmp_path, opd):
    with socket.socket() as sock:
        sock.bind(("127.0.0.1", 0))
        port = sock.getsockname()[1]
    mode = ["--dance-opd", "--teacher-size", "nano", "--batch", "2", "--micro-batch", "1", "--opd-rollout-steps", "2"] if opd \
        else ["--pp", "2", "--microbatches", "2", "--micro-batch", "1", "--act-checkpoint", "fp8"]
    r = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nnodes", "1", "--nproc-per-node", "1" if opd else "2",
                        "--master-addr", "127.0.0.1", "--master-port", str(port), "train_pp.py", "--out", str(tmp_path),
                        "--size", "nano", "--te-size", "states-nano", "--res", "128", "--steps", "1", "--log-every", "1",
                        "--fp8"] + mode, cwd=ROOT, capture_output=True, text=True, timeout=600,
                       env=dict(os.environ, CUDA_VISIBLE_DEVICES="", DIST_BACKEND="gloo"))
    assert r.returncode == 0 and "step 1/1" in r.stdout, r.stdout[-2000:] + r.stderr[-3000:]
