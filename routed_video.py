"""Train the routed video DiT (models/routed.py) on synthetic clips for a few steps and sample one clip from it:

  python routed_video.py [--frames 5 --height 12 --width 20] [--steps 20] [--device cuda]

Runs expert routing, expert dispatch / combine, the sandwich norms and the (time, row, column) rotary positions as a user
would: flow matching with AdamW, the balance bias moved after every step, then Euler sampling without gradients (where the
experts run packed, without a capacity). Prints the loss, the share of assignments that the capacity dropped and the
load of the busiest expert.
"""
import argparse

import torch

from trenowanie_generatora_obrazkow_b200.models.routed import RoutedConfig, RoutedDenoiser
from trenowanie_generatora_obrazkow_b200.optim.adamw import FusedAdamW
from trenowanie_generatora_obrazkow_b200.sampling.euler import time_grid


def make_model(args):
    torch.manual_seed(args.seed)
    cfg = RoutedConfig(latent_channels=16, dim=args.dim, depth=args.depth, heads=args.dim // 64, kv_heads=args.dim // 64,
                       axes=(16, 24, 24), text_dim=64, experts=args.experts, top_k=2, expert_hidden=args.dim,
                       groups=2, top_groups=1, res_scale=0.7)
    return RoutedDenoiser(cfg).to(args.device)


def train(model, args, log=print):
    g = torch.Generator(device=args.device).manual_seed(args.seed)
    rnd = lambda *s: torch.randn(*s, device=args.device, generator=g)
    shape = (args.batch, 16, args.frames, args.height, args.width)
    clips, text = rnd(*shape), rnd(args.batch, 8, 64)
    opt = FusedAdamW([dict(params=list(model.parameters()))], lr=args.lr)
    losses = []
    for step in range(args.steps):
        t = torch.sigmoid(rnd(args.batch))
        eps, tt = rnd(*shape), t.view(-1, 1, 1, 1, 1)
        v = model((1 - tt) * clips + tt * eps, t, text)
        loss = (v.float() - (eps - clips)).square().mean()
        loss.backward()
        opt.step()
        opt.zero_grad(set_to_none=True)
        model.update_balance(args.balance_rate)
        losses.append(loss.detach())
        if step % max(1, args.steps // 5) == 0 or step + 1 == args.steps:
            mlp = model.blocks[0].mlp
            tokens = args.batch * args.frames * args.height * args.width
            load = mlp.counts.float()
            dropped = (load - mlp.capacity(tokens)).clamp(min=0).sum() / load.sum()
            log(f"step {step}: loss {losses[-1].item():.4f}, dropped {100 * dropped.item():.1f} %, busiest expert "
                f"{(load.max() / load.mean()).item():.2f} x mean")
    return torch.stack(losses)


@torch.no_grad()
def sample(model, args, steps=8):
    z = torch.randn(1, 16, args.frames, args.height, args.width, device=args.device)
    text = torch.zeros(1, 8, 64, device=args.device)
    ts = time_grid(steps).tolist()
    for t0, t1 in zip(ts[:-1], ts[1:]):
        z = z + (t1 - t0) * model(z, torch.full((1,), t0, device=args.device), text).float()
    return z


def parse(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("frames", 5), ("height", 12), ("width", 20), ("batch", 2), ("dim", 512), ("depth", 4),
                          ("experts", 16), ("steps", 20), ("seed", 0)):
        p.add_argument(f"--{name}", type=int, default=default)
    p.add_argument("--lr", type=float, default=3e-4)
    p.add_argument("--balance-rate", type=float, default=1e-2)
    p.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    return p.parse_args(argv)


def main(argv=None):
    args = parse(argv)
    model = make_model(args)
    losses = train(model, args)
    z = sample(model, args)
    print(f"sampled clip {tuple(z.shape)}, std {z.std().item():.3f}, finite {bool(torch.isfinite(z).all())}")
    return losses, z


if __name__ == "__main__":
    main()
