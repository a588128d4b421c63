"""Routed diffusion transformer for images and video: the DiT block with rotary positions over time, height and width,
norms on both sides of every branch and an MLP of routed experts.

Per block, with (shift, scale, gate) x 2 from the shared modulation + the block's table, r = residual scale:

    h = rmsnorm(x) (1 + scale1) + shift1;   a = attention(q, k normalised and rotated by (t, row, column))
    x = x + r gate1 rmsnorm(a);             h = rmsnorm(x);                    c = cross-attention(h, text)
    x = x + r rmsnorm(c);                   h = rmsnorm(x) (1 + scale2) + shift2;   m = routed MLP(h)
    x = x + r gate2 rmsnorm(m)              (added by the next block's first norm)

Every "x = ...; h = ..." line is one ``sandwich_norm`` launch. The routed MLP scores each token against E experts (sigmoid
or softmax, group-limited top-k, a balance bias that is moved towards equal loads between steps instead of an auxiliary
loss), brings the rows into expert order and sums the chosen experts' outputs. Training gives every expert a static
capacity (fixed shapes, batched GEMMs forward and backward); inference packs the rows and runs grouped GEMMs whose
schedule comes from the offsets on the device, so one token costs one token's experts. Nothing synchronises with the
host. There is no such model in the reference; parameter naming follows models/dit.py.
"""
import math
from dataclasses import dataclass

import torch
import torch.distributed as dist
import torch.nn as nn

from ..ops import fused as Fz
from ..ops import reference as R
from ..ops import routing as Rt
from ..ops.gemm import gemm_grouped
from .dit import CrossAttention, RMSNorm
from .moe import batched_linear


@dataclass
class RoutedConfig:
    """axes: channels of a head that rotate with time, row and column (even, at most the head dim in all)."""
    latent_channels: int = 16
    dim: int = 1024
    depth: int = 12
    heads: int = 8
    kv_heads: int = 8
    axes: tuple = (16, 56, 56)
    theta: float = 10000.0
    text_dim: int = 1024
    experts: int = 64
    top_k: int = 8
    expert_hidden: int = 512
    score: str = "sigmoid"
    groups: int = 8
    top_groups: int = 4
    route_scale: float = 1.0
    capacity_factor: float = 1.25
    res_scale: float = 1.0


def _total_load(load, group):
    if dist.is_available() and dist.is_initialized() and dist.get_world_size(group) > 1:
        dist.all_reduce(load, group=group)
    return load


class RoutedMLP(nn.Module):
    """E SwiGLU experts of which each token uses k. ``capacity_factor`` applies while gradients are recorded (overflow is
    dropped); without gradients nothing is dropped. ``counts`` holds the last call's assignments per expert."""

    def __init__(self, dim, hidden, experts=64, top_k=8, score="sigmoid", groups=1, top_groups=1, scale=1.0,
                 capacity_factor=1.25):
        super().__init__()
        self.dim, self.E, self.k, self.cf = dim, experts, top_k, capacity_factor
        self.how = dict(score=score, groups=groups, top_groups=top_groups, scale=scale)
        self.router = nn.Linear(dim, experts, bias=False)
        self.w_in = nn.Parameter(torch.empty(experts, 2 * hidden, dim))
        self.w_out = nn.Parameter(torch.empty(experts, dim, hidden))
        self.register_buffer("balance", torch.zeros(experts))
        self.counts = None
        nn.init.normal_(self.router.weight, std=0.02)
        nn.init.normal_(self.w_in, std=dim ** -0.5)
        nn.init.normal_(self.w_out, std=hidden ** -0.5)

    def route(self, x2, valid=None):
        logits = torch.nn.functional.linear(x2.float(), self.router.weight.float())
        return Rt.route_experts(logits, self.k, bias=self.balance, valid=valid, **self.how)

    def capacity(self, n):
        return max(8, math.ceil(self.cf * n * self.k / self.E / 8) * 8)

    def forward(self, h, valid=None):
        """h [..., dim]; valid (bool, h's shape without dim): padding tokens take no expert and get zeros."""
        x2 = h.reshape(-1, self.dim)
        w, idx = self.route(x2, None if valid is None else valid.reshape(-1))
        training = torch.is_grad_enabled() and any(t.requires_grad for t in (x2, self.w_in, self.w_out))
        plan = Rt.expert_plan(idx, self.E, self.capacity(x2.shape[0]) if training else None)
        self.counts = plan.counts
        xs = Rt.expert_dispatch(x2, plan)
        if training:
            ab = batched_linear(xs.view(self.E, plan.capacity, self.dim), self.w_in)
            y = batched_linear(Fz.swiglu(ab), self.w_out).reshape(plan.rows, self.dim)
        else:
            up, down = (Fz.bf16_weight(p) if h.is_cuda else p.detach() for p in (self.w_in, self.w_out))
            y = gemm_grouped(Fz.swiglu(gemm_grouped(xs, up, plan.offsets)), down, plan.offsets)
        return Rt.expert_combine(y.to(h.dtype), w, plan).view(h.shape)

    @torch.no_grad()
    def update_balance(self, rate=1e-3, group=None):
        """Move the balance bias of overloaded experts down and of underloaded ones up (once per step). The load is that of
        all ranks of the process group (None: the default one, where there is one), so replicas keep one bias."""
        if self.counts is not None:
            self._move_balance(_total_load(self.counts.float(), group), rate)

    def _move_balance(self, load, rate):
        self.balance += rate * (load.mean() - load).sign()


class RoutedBlock(nn.Module):
    def __init__(self, c: RoutedConfig):
        super().__init__()
        self.c, self.head_dim = c, c.dim // c.heads
        self.norm1, self.norm2, self.norm3 = (RMSNorm(c.dim) for _ in range(3))
        self.post1, self.post2, self.post3 = (RMSNorm(c.dim) for _ in range(3))
        self.qkv = nn.Linear(c.dim, (c.heads + 2 * c.kv_heads) * self.head_dim, bias=False)
        self.out = nn.Linear(c.dim, c.dim, bias=False)
        self.q_norm, self.k_norm = RMSNorm(self.head_dim), RMSNorm(self.head_dim)
        self.cross = CrossAttention(c.dim, c.heads, c.text_dim)
        self.mlp = RoutedMLP(c.dim, c.expert_hidden, c.experts, c.top_k, c.score, c.groups, c.top_groups, c.route_scale,
                             c.capacity_factor)
        self.mod_table = nn.Parameter(torch.zeros(6, c.dim))

    def forward(self, x, pending, t6, text, text_len, pos):
        """pending: (branch, gate, post weight) of the block before, not yet added to x."""
        c = self.c
        shift1, scale1, gate1, shift2, scale2, gate2 = (t6 + self.mod_table[None]).to(x.dtype).unbind(1)
        if pending is None:
            x, h = Fz.adanorm(x, None, None, self.norm1.weight, shift1, scale1)
        else:
            x, h = Fz.sandwich_norm(x, *pending, self.norm1.weight, shift1, scale1, res_scale=c.res_scale)
        a = Fz.axes_attention_core(Fz.linear(h, self.qkv), pos, c.axes, c.heads, c.kv_heads, self.head_dim, c.theta,
                                   self.q_norm.weight, self.k_norm.weight)
        x, h = Fz.sandwich_norm(x, Fz.linear(a, self.out), gate1, self.post1.weight, self.norm2.weight,
                                res_scale=c.res_scale)
        x, h = Fz.sandwich_norm(x, self.cross(h, text, text_len), None, self.post2.weight, self.norm3.weight, shift2,
                                scale2, res_scale=c.res_scale)
        return x, (self.mlp(h), gate2, self.post3.weight)


class RoutedDenoiser(nn.Module):
    """Velocity of latent clips (B, C, F, H, W) (an image is a clip of one frame), one token per latent pixel."""

    def __init__(self, c: RoutedConfig = RoutedConfig()):
        super().__init__()
        self.config = c
        self.patch_in = nn.Linear(c.latent_channels, c.dim, bias=False)
        self.time_mlp = nn.Sequential(nn.Linear(256, c.dim), nn.SiLU(), nn.Linear(c.dim, c.dim))
        self.ada = nn.Linear(c.dim, 6 * c.dim)
        self.blocks = nn.ModuleList([RoutedBlock(c) for _ in range(c.depth)])
        self.norm = RMSNorm(c.dim)
        self.patch_out = nn.Linear(c.dim, c.latent_channels, bias=False)
        for m in (self.ada, self.time_mlp[0], self.time_mlp[2]):
            nn.init.normal_(m.weight, std=0.02)
            nn.init.zeros_(m.bias)
        nn.init.normal_(self.patch_out.weight, std=0.02)

    @staticmethod
    def positions(b, f, h, w, device=None):
        """(frame, row, column) of every token, int32 [B, F H W, 3]."""
        ax = [torch.arange(n, device=device, dtype=torch.int32) for n in (f, h, w)]
        return torch.stack(torch.meshgrid(*ax, indexing="ij"), -1).view(1, f * h * w, 3).expand(b, -1, -1).contiguous()

    def forward(self, z, t, text, text_len=None, pos=None):
        """z (B, C, F, H, W), t (B,), text (B, L, text_dim) -> velocity like z. pos overrides the grid positions (fp32
        for interpolated grids)."""
        b, c, f, h, w = z.shape
        pos = self.positions(b, f, h, w, z.device) if pos is None else pos
        tok = z.flatten(2).transpose(1, 2)
        if z.is_cuda:
            tok, text = tok.to(torch.bfloat16).contiguous(), text.to(torch.bfloat16)
        if text_len is not None:
            text_len = text_len.to(device=z.device, dtype=torch.int32)
        x = Fz.linear(tok, self.patch_in)
        te = Fz.linear(R.timestep_embedding(t, 256), self.time_mlp[0])
        te = Fz.linear(torch.nn.functional.silu(te), self.time_mlp[2])
        t6 = Fz.linear(torch.nn.functional.silu(te), self.ada).view(b, 6, -1)
        pending = None
        for blk in self.blocks:
            x, pending = blk(x, pending, t6, text, text_len, pos)
        _, hn = Fz.sandwich_norm(x, *pending, self.norm.weight, res_scale=self.config.res_scale)
        return Fz.linear(hn, self.patch_out).transpose(1, 2).reshape(b, c, f, h, w)

    @torch.no_grad()
    def update_balance(self, rate=1e-3, group=None):
        """RoutedMLP.update_balance of every block, with one sum over the ranks."""
        mlps = [blk.mlp for blk in self.blocks if blk.mlp.counts is not None]
        if mlps:
            for mlp, load in zip(mlps, _total_load(torch.stack([m.counts.float() for m in mlps]), group)):
                mlp._move_balance(load, rate)
