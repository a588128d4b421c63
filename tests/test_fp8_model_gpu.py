"""The DiT on 8-bit products and with 8-bit activation checkpoints on the GPU, and the operators in a run together."""
import io

import pytest
import torch

from trenowanie_generatora_obrazkow_b200.ops import blocks8 as B8
from trenowanie_generatora_obrazkow_b200.ops import fused as Fz
from trenowanie_generatora_obrazkow_b200.ops._ext import check_errors

pytestmark = pytest.mark.gpu


def _model():
    from trenowanie_generatora_obrazkow_b200.models import DenoiserConfig, LMEncoderConfig, build_models
    den_cfg = DenoiserConfig(dim=512, depth=2, heads=4, mlp_hidden=1408, text_dim=512, latent_size=16)
    te_cfg = LMEncoderConfig(repo="", tok_suffix="", lm_dim=256, skip_last=0, dim=512, depth=1, heads=8, kv_heads=2,
                             head_dim=64, mlp_hidden=1408, max_tokens=32, backend="states")
    torch.manual_seed(0)
    te, den = build_models(den_cfg, te_cfg, device="cuda")
    te.init_weights(), den.init_weights()
    with torch.no_grad():
        for p in list(te.parameters()) + list(den.parameters()):
            p.add_(0.02 * torch.randn_like(p))
    return te, den


def _step(te, den, mode=False):
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(4, 128, 16, 16, device="cuda", generator=g)
    t = torch.rand(4, device="cuda", generator=g)
    st = torch.randn(4, 32, 256, device="cuda", generator=g).bfloat16()
    te.checkpoint_blocks = den.checkpoint_blocks = mode
    params = list(te.parameters()) + list(den.parameters())
    for p in params:
        p.grad = None
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    text, valid = te(lm_states=st)
    out = den(x, t, text, valid)
    held = torch.cuda.memory_allocated() - base
    out.float().square().mean().backward()
    torch.cuda.synchronize()
    check_errors("cuda")
    return out.detach().float(), [None if p.grad is None else p.grad.clone() for p in params], held


def _apart(a, b):
    a, b = (torch.cat([g.flatten() for g in x if g is not None]) for x in (a, b))
    return ((a - b).norm() / b.norm()).item()


def test_dit_on_8_bit_products():
    from trenowanie_generatora_obrazkow_b200.models.quant import use_fp8
    te, den = _model()
    plain, grads, _ = _step(te, den)
    use_fp8(te), use_fp8(den)
    out, g8, _ = _step(te, den)
    # each value is off by at most 2^-4 of itself; sums of many add up like noise
    assert 0 < ((out - plain).norm() / plain.norm()).item() < 0.1
    assert [g is None for g in grads] == [g is None for g in g8]
    assert _apart(g8, grads) < 0.1
    again, g9, _ = _step(te, den)
    assert torch.equal(again, out)
    with torch.no_grad():
        g = torch.Generator(device="cuda").manual_seed(3)
        x = torch.randn(4, 128, 16, 16, device="cuda", generator=g)
        t = torch.rand(4, device="cuda", generator=g)
        st = torch.randn(4, 32, 256, device="cuda", generator=g).bfloat16()
        text, valid = te(lm_states=st)
        held = den(x, t, text, valid).float()
    assert ((held - out).norm() / out.norm()).item() < 0.02  # held weights: the same products without a graph


@pytest.mark.parametrize("fp8", [False, True])
def test_checkpoint_mode_fp8(fp8):
    from trenowanie_generatora_obrazkow_b200.models.quant import use_fp8
    te, den = _model()
    if fp8:
        use_fp8(te), use_fp8(den)
    plain, grads, held = _step(te, den)
    sel, _, held_sel = _step(te, den, "selective")
    out, g8, held8 = _step(te, den, "fp8")
    assert ((out - plain).norm() / plain.norm()).item() < 0.01  # the SwiGLU kernels differ by a rounding
    assert _apart(g8, grads) < 0.05
    if not fp8:
        assert held8 < held_sel < held, (held8, held_sel, held)


def test_trainer_step_and_optimizer_on_8_bit_products():
    from trenowanie_generatora_obrazkow_b200.models import DenoiserConfig, LMEncoderConfig
    from trenowanie_generatora_obrazkow_b200.train.trainer import TrainConfig, Trainer
    den = DenoiserConfig(dim=512, depth=2, heads=4, mlp_hidden=1408, text_dim=512, latent_size=16)
    te = LMEncoderConfig(repo="", tok_suffix="", lm_dim=256, skip_last=0, dim=512, depth=1, heads=8, kv_heads=2,
                         head_dim=64, mlp_hidden=1408, max_tokens=32, backend="states")
    device = torch.device("cuda", 0)
    tr = Trainer(den, te, TrainConfig(global_batch=4, micro_batch=2, steps=10, fp8=True), device)
    before = tr.den.blocks[0].mlp.in_proj.weight.detach().clone()
    layers = [tr.den.blocks[1].attn.qkv, tr.den.blocks[0].mlp.out_proj, tr.te.blocks[0].mlp.in_proj]
    held = [Fz.fp8_weight(m.weight) for m in layers]  # as an evaluation between steps leaves them
    batch = {"x0": torch.randn(4, 128, 16, 16, device=device),
             "lm_states": torch.randn(4, 32, 256, device=device, dtype=torch.bfloat16)}
    losses = [tr.step(batch) for _ in range(2)]
    torch.cuda.synchronize()
    check_errors(device)
    assert all(torch.isfinite(v).item() for v in losses)
    assert tr.den.blocks[0].mlp.in_proj.weight.grad.dtype == torch.float32
    assert not torch.equal(before, tr.den.blocks[0].mlp.in_proj.weight)
    for m, old in zip(layers, held):  # the optimizer's kernels write the weights past autograd's version counter
        now = Fz.fp8_weight(m.weight)
        assert now is not old and torch.equal(now.codes.view(torch.uint8), B8.quantize_blocks(m.weight).codes.view(torch.uint8))


def test_operators_in_a_run():
    """Packing, a layer, the MLP, a layer on held weights and the checkpointed activation, one after another."""
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s, std=1.0: torch.randn(*s, device="cuda", generator=g) * std  # noqa: E731
    x = r(3, 111, 256).bfloat16().requires_grad_()
    w0, w1, w2, w3 = r(320, 256, std=1 / 16), r(768, 320, std=1 / 18), r(320, 384, std=1 / 20), r(256, 320, std=1 / 18)
    ws = [w.requires_grad_() for w in (w0, w1, w2)]
    h = B8.linear_blocks(x, w0)
    y = h + B8.mlp_blocks(h, w1, w2)
    g0 = B8.swiglu_blocks(y)
    g0.backward(torch.ones_like(g0))
    # the same in fp32 torch operations without packing: noise of 8 bits apart
    xr = x.detach().float().requires_grad_()
    wr = [w.detach().clone().requires_grad_() for w in ws]
    hr = xr @ wr[0].t()
    a, b = (hr @ wr[1].t()).chunk(2, dim=-1)
    yr = hr + (torch.nn.functional.silu(a) * b) @ wr[2].t()
    p, q = yr.chunk(2, dim=-1)
    gr = torch.nn.functional.silu(p) * q
    gr.backward(torch.ones_like(gr))
    for got, want in [(g0, gr), (x.grad, xr.grad)] + [(w.grad, v.grad) for w, v in zip(ws, wr)]:
        assert ((got.float() - want).norm() / want.norm()).item() < 0.12
    with torch.no_grad():
        last = B8.linear_blocks(y, B8.quantize_blocks(w3))
        few = B8.linear_blocks(y[:1, :9], B8.quantize_blocks(w3))
        assert last.shape == (3, 111, 256)
        assert torch.allclose(few.float(), last[:1, :9].float(), rtol=2 ** -7, atol=1e-2)
    check_errors("cuda")


@pytest.mark.parametrize("M", [0, 1, 7, 16, 17, 200])
def test_mlp_on_held_weights(M):
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn(M, 200, device="cuda", generator=g)
    w1, w2 = torch.randn(512, 200, device="cuda", generator=g) / 14, torch.randn(72, 256, device="cuda", generator=g) / 16
    y = B8.mlp_blocks(x, B8.quantize_blocks(w1), B8.quantize_blocks(w2))
    want = B8.mlp_blocks(x, w1, w2)
    # few rows sum in another order: a value of g at a border may be packed to its neighbour, 2^-3 of it
    assert y.shape == want.shape and (M == 0 or ((y - want).norm() / want.norm()).item() < 0.01)
    with pytest.raises(RuntimeError, match="no gradient"):
        B8.mlp_blocks(x.clone().requires_grad_(), B8.quantize_blocks(w1), B8.quantize_blocks(w2))
    with pytest.raises(TypeError):
        B8.mlp_blocks(x, w1, B8.quantize_blocks(w2))


def test_block_linear_and_marked_layers():
    from trenowanie_generatora_obrazkow_b200.models.quant import quantize
    lin = torch.nn.Linear(300, 136, device="cuda")
    lin.fp8 = True
    x = torch.randn(2, 9, 300, device="cuda").bfloat16()
    with torch.no_grad():
        marked = Fz.linear(x, lin)
    m = torch.nn.Sequential(lin)
    assert torch.equal(quantize(m, "fp8_block")(x), marked)


@pytest.mark.parametrize("kind", ["int8", "fp8", "w8a8", "fp8_block"])
def test_quantized_dit(kind):
    from trenowanie_generatora_obrazkow_b200.models.quant import quantize, use_fp8
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(4, 128, 16, 16, device="cuda", generator=g)
    t = torch.rand(4, device="cuda", generator=g)
    st = torch.randn(4, 32, 256, device="cuda", generator=g).bfloat16()

    def run(te, den):
        text, valid = te(lm_states=st)
        return den(x, t, text, valid).float()
    with torch.no_grad():
        te, den = _model()
        plain = run(te, den)
        if kind == "fp8_block":
            use_fp8(te), use_fp8(den)
            marked = run(te, den)
            te, den = _model()
            quantize(te.blocks, kind), quantize(den.blocks, kind)
            # the same products but for g, which is rounded to bf16 before it is packed: one value in 2^-9 / 2^-4 = 2^5 takes its
            # neighbour, 2^-4 of it on average, 1.1 % of a branch's norm in each of two blocks
            assert ((run(te, den) - marked).norm() / marked.norm()).item() < 0.023
            te, den = _model()
        quantize(te, kind), quantize(den, kind)  # time_mlp and ada take the form of few rows
        assert 0 < ((run(te, den) - plain).norm() / plain.norm()).item() < 0.1
    check_errors("cuda")


def test_marked_routed_blocks():
    from trenowanie_generatora_obrazkow_b200.models.quant import use_fp8
    from trenowanie_generatora_obrazkow_b200.models.routed import RoutedConfig, RoutedDenoiser
    torch.manual_seed(0)
    net = RoutedDenoiser(RoutedConfig(latent_channels=8, dim=256, depth=2, heads=2, kv_heads=2, axes=(32, 48, 48), text_dim=64,
                                      experts=8, top_k=2, expert_hidden=128, groups=2, top_groups=1, capacity_factor=8.0)).cuda()
    z, t, text = torch.randn(2, 8, 3, 7, 9, device="cuda"), torch.rand(2, device="cuda"), torch.randn(2, 5, 64, device="cuda")

    def step():
        net.zero_grad()
        out = net(z, t, text)
        out.float().square().mean().backward()
        return out.detach().float(), [p.grad for p in net.parameters()]
    plain, _ = step()
    use_fp8(net)
    out, grads = step()
    # a value's error is at most 2^-4 of it; products of many add up like noise (a token at a border may take another expert)
    assert 0 < ((out - plain).norm() / plain.norm()).item() < 0.2
    assert all(g is not None and g.isfinite().all() for g in grads)
    with torch.no_grad():
        net(z, t, text)
        kept = [net.blocks[1].cross.kv.weight._tgo_fp8, net.blocks[0].qkv.weight._tgo_fp8]
        held = net(z, t, text).float()
    assert kept[0] is net.blocks[1].cross.kv.weight._tgo_fp8 and kept[1] is net.blocks[0].qkv.weight._tgo_fp8
    assert ((held - out).norm() / out.norm()).item() < 0.2
    check_errors("cuda")


@pytest.mark.parametrize("M", [3, 40])
def test_far_scales(M):
    """Large activations against small weights: the product is in range, and so is the result."""
    x, w = torch.full((M, 128), 2.0 ** 118, device="cuda"), torch.full((16, 128), 2.0 ** -60, device="cuda")
    got = B8.linear_blocks(x, B8.quantize_blocks(w))
    assert torch.equal(got, torch.full((M, 16), 2.0 ** 65, device="cuda"))


def test_captured_layer_packs_for_itself():
    """A graph of marked layers without gradients reads the weights as they are at each replay, and leaves nothing behind that
    an eager call would take for packed."""
    from trenowanie_generatora_obrazkow_b200.models.quant import use_fp8
    te, den = _model()
    use_fp8(den)
    mlp, qkv = den.blocks[0].mlp, den.blocks[0].attn.qkv
    x = torch.randn(300, 512, device="cuda", dtype=torch.bfloat16)

    def run():
        return Fz.mlp_fp8(x, mlp.in_proj, mlp.out_proj), Fz.linear(x, qkv)
    with torch.no_grad():
        other = torch.cuda.Stream()
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            B8.mlp_blocks(x, mlp.in_proj, mlp.out_proj)
        torch.cuda.current_stream().wait_stream(other)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run()
        first = run()  # before any replay
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, first))
        for lin in (mlp.in_proj, mlp.out_proj, qkv):
            lin.weight.mul_(1.25)
        graph.replay()
        want = run()
        assert all(torch.equal(a, b) and not torch.equal(a, c) for a, b, c in zip(got, want, first))


def test_packed_weight_on_another_stream():
    lin = torch.nn.Linear(2048, 8192, device="cuda", bias=False)
    lin.fp8 = True
    x = torch.randn(64, 2048, device="cuda", dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    with torch.no_grad():
        want = B8.linear_blocks(x, B8.quantize_blocks(lin.weight))
        torch.cuda.synchronize()
        for _ in range(20):
            lin.weight._tgo_fp8 = None
            first = Fz.linear(x, lin)  # packs here
            with torch.cuda.stream(side):
                second = Fz.linear(x, lin)
            torch.cuda.synchronize()
            assert torch.equal(first, want) and torch.equal(second, want)
        file = io.BytesIO()
        torch.save(lin, file)  # the copy and its stream stay behind
        again = torch.load(io.BytesIO(file.getvalue()), weights_only=False)
        assert again.weight._tgo_fp8 is None and torch.equal(Fz.linear(x, again), want)
