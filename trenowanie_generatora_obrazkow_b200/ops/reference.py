"""fp32 PyTorch oracles of every op the kernels implement (CPU path and numerics reference of the GPU tests).

The math is the reference's (aurora/model.py): RMSNorm :27-34, interleaved-pair RoPE :37-50 and :98-99, 2D RoPE
:53-72, RPE-2D coordinates :75-80, micro-conditioning :83-95, SwiGLU :102-110, attention :113-188, time embedding
:213-218. Layout differs: activations are [batch, token, head, head_dim] and RoPE tables are [token, head_dim]
(or [batch, token, head_dim] for per-sample coordinates).
"""
import math

import torch
import torch.nn.functional as F

EPS = 1e-6


def rmsnorm(x, w, eps=EPS):
    """x * rsqrt(mean(x^2) + eps) * w, the statistic in fp32 and the scale cast back to x's dtype."""
    return x * torch.rsqrt(x.float().pow(2).mean(dim=-1, keepdim=True) + eps).to(x.dtype) * w


def rotate_pairs(x):
    """(x0, x1, x2, x3, ...) -> (-x1, x0, -x3, x2, ...)."""
    ev, od = x[..., 0::2], x[..., 1::2]
    return torch.stack((-od, ev), dim=-1).flatten(-2)


def apply_rope(x, cos, sin):
    """x [B, T, H, d]; cos / sin [T, d] or [B, T, d] (already duplicated per pair)."""
    if cos.dim() == 2:
        cos, sin = cos[None, :, None], sin[None, :, None]
    else:
        cos, sin = cos[:, :, None], sin[:, :, None]
    return x * cos.to(x.dtype) + rotate_pairs(x) * sin.to(x.dtype)


def _dup(a):
    return a.repeat_interleave(2, dim=-1)


def rope_1d_table(n, d, device=None):
    """1D RoPE for positions 0..n-1: inv_freq = 10000^(-2i/d) -> cos, sin [n, d]."""
    inv = 1.0 / (10000 ** (torch.arange(0, d, 2, dtype=torch.float32, device=device) / d))
    ang = torch.arange(n, dtype=torch.float32, device=device)[:, None] * inv
    return _dup(ang.cos()), _dup(ang.sin())


def rope_2d_from_coords(rows, cols, d):
    """(B, h) row and (B, w) column positions -> cos, sin [B, h*w, d]: the first half of the head dim rotates with
    the row, the second half with the column; tokens are row-major."""
    b, h, w = rows.shape[0], rows.shape[1], cols.shape[1]
    inv = 1.0 / (10000 ** (torch.arange(0, d // 2, 2, dtype=torch.float32, device=rows.device) / (d // 2)))
    ar = (rows.float()[:, :, None] * inv)[:, :, None].expand(b, h, w, -1)
    ac = (cols.float()[:, :, None] * inv)[:, None].expand(b, h, w, -1)
    ang = torch.cat([ar, ac], dim=-1).reshape(b, h * w, -1)
    return _dup(ang.cos()), _dup(ang.sin())


def grid_coords(side, ref=0, device=None):
    """Positions of `side` tokens along one axis; ref > 0 spreads them over a ref-token field
    ((i + 0.5) * ref / side - 0.5, position interpolation)."""
    c = torch.arange(side, dtype=torch.float32, device=device)
    if ref and ref != side:
        c = (c + 0.5) * (ref / side) - 0.5
    return c


def rope_2d_table(h, w, d, ref=0, device=None):
    """2D RoPE of an h x w grid -> cos, sin [h*w, d]."""
    cos, sin = rope_2d_from_coords(grid_coords(h, ref, device)[None], grid_coords(w, ref, device)[None], d)
    return cos[0], sin[0]


def random_rope_coords(b, side, field, device=None, generator=None):
    """RPE-2D (arXiv:2503.18719): per sample and axis `side` sorted distinct integer positions of 0..field-1."""
    def axis():
        r = torch.rand(b, field, device=device, generator=generator)
        return r.topk(side, dim=1).indices.sort(dim=1).values
    return axis(), axis()


def timestep_embedding(t, dim=256):
    """t * 1000 -> [sin, cos] with freqs exp(-ln(1e4) i / (half - 1))."""
    t = t.float() * 1000.0
    half = dim // 2
    freqs = torch.exp(-math.log(10000) * torch.arange(half, device=t.device).float() / max(half - 1, 1))
    ang = t[:, None] * freqs[None]
    return torch.cat([ang.sin(), ang.cos()], dim=-1)


def micro_cond_embedding(cond, dim=256):
    """(B, 8) micro-conditions in pixels -> (B, 8 * dim) sinusoids with freqs exp(-ln(1e4) i / half)."""
    half = dim // 2
    freqs = torch.exp(-math.log(10000) * torch.arange(half, device=cond.device).float() / half)
    ang = cond.float()[:, :, None] * freqs
    return torch.cat([ang.sin(), ang.cos()], dim=-1).flatten(1)


def default_micro_cond(base, res, b, device=None):
    """Micro-conditions of a whole uncropped image: [orig_h, orig_w, top, left, bottom, right, tgt_h, tgt_w]."""
    o = max(base, res)
    return torch.tensor([o, o, 0, 0, o, o, res, res], dtype=torch.float32, device=device).expand(b, 8)


def attention(q, k, v, kv_len=None, scale=None):
    """q [B, Tq, Hq, d], k / v [B, Tk, Hkv, d] (Hq % Hkv == 0), keys >= kv_len[b] masked -> [B, Tq, Hq, d]."""
    B, Tq, Hq, d = q.shape
    Hkv = k.shape[2]
    rep = Hq // Hkv
    qh = q.transpose(1, 2)
    kh = k.transpose(1, 2).repeat_interleave(rep, dim=1)
    vh = v.transpose(1, 2).repeat_interleave(rep, dim=1)
    mask = None
    if kv_len is not None:
        mask = (torch.arange(k.shape[1], device=q.device)[None] < kv_len.to(q.device)[:, None])[:, None, None, :]
    o = F.scaled_dot_product_attention(qh, kh, vh, attn_mask=mask, scale=scale)
    return o.transpose(1, 2)


def varlen_attention(q, k, v, cu_seqlens, causal=True, scale=None):
    """Packed sequences: q [T, Hq, d], k / v [T, Hkv, d], cu_seqlens [n + 1] token offsets; attention stays inside
    each sequence (causal: key <= query position) -> [T, Hq, d]."""
    out = torch.empty_like(q)
    cu = [int(c) for c in cu_seqlens.tolist()]
    for a, b in zip(cu[:-1], cu[1:]):
        if b <= a:
            continue
        qh, kh, vh = (x[a:b].transpose(0, 1) for x in (q, k, v))
        rep = qh.shape[0] // kh.shape[0]
        kh, vh = kh.repeat_interleave(rep, 0), vh.repeat_interleave(rep, 0)
        out[a:b] = F.scaled_dot_product_attention(qh, kh, vh, is_causal=causal, scale=scale).transpose(0, 1)
    return out


def swiglu(ab):
    a, b = ab.chunk(2, dim=-1)
    return F.silu(a) * b


def valid_to_len(valid):
    """Boolean key mask [B, L] (a prefix per row, captions are right-padded) -> int32 lengths [B]."""
    return valid.sum(dim=1).to(torch.int32)


def route_experts(logits, k, score="softmax", bias=None, groups=1, top_groups=1, renorm=True, scale=1.0, valid=None):
    """Expert choice and weights (see ops/routing.py); NaN scores come last."""
    l = logits.float() if logits.dtype in (torch.bfloat16, torch.float16) else logits
    n, e = l.shape
    if score == "softmax":
        p = torch.softmax(torch.where((l == -math.inf).all(-1, keepdim=True), torch.zeros_like(l), l), -1)
        p = torch.where((l == -math.inf), torch.zeros_like(p), p)
        key = l.detach()
    else:
        ex = torch.exp(torch.where(l >= 0, -l, l))  # torch's own sigmoid is 0 below -88 in 32 bits: ties of what differs
        p = torch.where(l >= 0, torch.ones_like(ex), ex) / (1 + ex)
        key = p.detach()
    if bias is not None:
        key = key + bias
    live = torch.ones_like(key, dtype=torch.bool)
    nan = key.isnan()
    key = key.masked_fill(nan, -math.inf)
    if groups > 1:
        by = key.view(n, groups, -1).sort(dim=-1, descending=True).values
        worth = by[..., 0] if score == "softmax" or by.shape[-1] == 1 else by[..., 0] + by[..., 1]
        worth = worth.masked_fill(worth.isnan(), -math.inf)
        kept = worth.sort(dim=-1, descending=True, stable=True).indices[:, :top_groups]
        on = torch.zeros(n, groups, device=l.device, dtype=torch.bool).scatter_(1, kept, True)
        live = on.repeat_interleave(e // groups, 1)
    order = key.sort(dim=-1, descending=True, stable=True).indices
    late = 2 * (~live).to(torch.int8) + nan.to(torch.int8)  # kept numbers, kept NaNs, then dropped groups
    idx = order.gather(1, late.gather(1, order).sort(dim=-1, stable=True).indices)[:, :k]
    w = p.gather(1, idx)
    if renorm:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    w, idx = w * scale, idx.to(torch.int32)
    if valid is not None:
        w, idx = w * valid[:, None], idx.masked_fill(~valid[:, None], -1)
    return w, idx


def expert_plan(idx, experts, capacity=0):
    """(slot [N, k], offsets [E + 1], counts [E]), int32: a stable counting sort of the assignments by expert."""
    flat = idx.reshape(-1).long()
    flat = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, -1))
    hit = flat[:, None] == torch.arange(experts, device=flat.device)
    rank = (hit.cumsum(0) - 1).gather(1, flat.clamp(min=0)[:, None])[:, 0]
    counts = hit.sum(0)
    if capacity:
        offsets = torch.arange(experts + 1, device=flat.device) * capacity
        ok = (flat >= 0) & (rank < capacity)
    else:
        offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
        ok = flat >= 0
    slot = torch.where(ok, offsets[flat.clamp(min=0)] + rank, torch.full_like(flat, -1))
    i32 = torch.int32
    return slot.view(idx.shape).to(i32), offsets.to(i32), counts.to(i32)


def expert_dispatch(x, plan):
    """x [N, D] -> [rows, D] (unused rows zero)."""
    k = plan.slot.shape[1]
    slot = plan.slot.reshape(-1).long()
    at = torch.where(slot >= 0, slot, torch.full_like(slot, plan.rows))
    return x.new_zeros(plan.rows + 1, x.shape[1]).index_copy(0, at, x.repeat_interleave(k, 0))[:plan.rows]


def expert_combine(y, w, plan):
    """y [rows, D], w [N, k] -> [N, D]."""
    n, k = plan.slot.shape
    slot = plan.slot.reshape(-1).long()
    rows = torch.cat([y, y.new_zeros(1, y.shape[1])])[torch.where(slot >= 0, slot, torch.full_like(slot, plan.rows))]
    keep = (slot >= 0).view(n, k, 1)
    wide = torch.promote_types(y.dtype, torch.float32)
    rows = rows.view(n, k, y.shape[1]).to(wide) * w[..., None].to(wide)
    return torch.where(keep, rows, torch.zeros((), dtype=wide)).sum(1).to(y.dtype)


def sandwich_norm(x, y, gate=None, post_w=None, w=None, shift=None, scale=None, res_scale=1.0, eps=EPS):
    """x_new = x + res_scale gate rmsnorm(y) post_w; h = rmsnorm(x_new) w (1 + scale) + shift (see ops/fused.py)."""
    wide = torch.promote_types(x.dtype, torch.float32)
    norm = lambda a: a * torch.rsqrt(a.square().mean(-1, keepdim=True) + eps)
    u = y.to(wide)
    if post_w is not None:
        u = norm(u) * post_w
    if gate is not None:
        u = u * gate.to(wide)[:, None]
    x_new = x.to(wide) + res_scale * u
    if w is None:
        return x_new.to(x.dtype), None
    h = norm(x_new) * w
    if scale is not None:
        h = h * (1 + scale.to(wide)[:, None]) + shift.to(wide)[:, None]
    return x_new.to(x.dtype), h.to(x.dtype)


def axes_frequencies(axes, theta=10000.0):
    """Angle per position of every rotated pair (fp64 [sum(axes) / 2]) and its position axis: axis a turns the pairs
    m < axes[a] / 2 by theta_a^(-2 m / axes[a])."""
    thetas = [theta] * len(axes) if isinstance(theta, (int, float)) else list(theta)
    freq = torch.cat([float(th) ** (-torch.arange(0, d, 2, dtype=torch.float64) / d) for d, th in zip(axes, thetas)])
    return freq, torch.cat([torch.full((d // 2,), a, dtype=torch.int32) for a, d in enumerate(axes)])


def rope_axes(q, k, pos, axes, theta=10000.0, q_w=None, k_w=None, interleaved=True, eps=EPS):
    """q [B, T, Hq, d], k [B, T, Hkv, d], pos [B, T, len(axes)] -> rotated (and normalised) q, k (see ops/fused.py)."""
    freq, axis = axes_frequencies(axes, theta)
    wide = torch.promote_types(q.dtype, torch.float32)
    ang = (pos.double()[..., axis.long()] * freq.to(pos.device))[:, :, None]
    cos, sin = ang.cos().to(wide), ang.sin().to(wide)
    half = freq.numel()

    def turn(x, w):
        x = x.to(wide)
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
        rot, rest = x[..., :2 * half], x[..., 2 * half:]
        if interleaved:
            rot = torch.stack((rot[..., 0::2] * cos - rot[..., 1::2] * sin,
                               rot[..., 1::2] * cos + rot[..., 0::2] * sin), dim=-1).flatten(-2)
        else:
            a, b = rot[..., :half], rot[..., half:]
            rot = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
        return torch.cat((rot, rest), dim=-1)
    return turn(q, q_w).to(q.dtype), turn(k, k_w).to(k.dtype)


# ----------------------------------------------------------------------------------------------------------------
# 8-bit blocks: e4m3 with a power-of-two scale for each 128 values of a row
# ----------------------------------------------------------------------------------------------------------------
def quantize_blocks(x):
    """x [M, K] -> (codes e4m3 [M, Kp], scales uint8 [ceil(M / 128), ceil(Kp / 512), 32, 4, 4]): see ops/blocks8.py."""
    M, K = x.shape
    nb, rt = -(-K // 128), -(-M // 128)
    quads = -(-nb // 4)
    f = torch.nn.functional.pad(x.detach().float(), (0, nb * 128 - K)).view(M, nb, 128)
    finite = f.isfinite()
    top = torch.where(finite, f.abs(), 0.0).amax(-1)
    m, e = torch.frexp(top)  # top = m 2^e, 1/2 <= m < 1; 448 = 7/8 2^9
    e = torch.where(top > 0, torch.where(m <= 0.875, e - 9, e - 8).clamp_min(-127), -127)
    q = torch.where(finite, torch.ldexp(f, -e[..., None]), math.nan).to(torch.float8_e4m3fn)
    scales = torch.zeros(rt * 128, quads * 4, dtype=torch.uint8, device=x.device)
    scales[:M, :nb] = (e + 127).to(torch.uint8)
    return q.view(M, nb * 128), scales.view(rt, 4, 32, quads, 4).permute(0, 3, 2, 1, 4).contiguous()


def dequantize_blocks(codes, scales, cols):
    """The values of quantize_blocks' output, fp32 [M, cols]."""
    M, width = codes.shape
    rt, quads = scales.shape[:2]
    e = scales.permute(0, 3, 2, 1, 4).reshape(rt * 128, quads * 4)[:M, :width // 128].int() - 127
    return torch.ldexp(codes.float().view(M, width // 128, 128), e[..., None]).view(M, width)[:, :cols]


def in_blocks(x):
    """The values that 8 bits hold of x [M, K], blocks along the rows (fp32)."""
    return dequantize_blocks(*quantize_blocks(x), x.shape[1])


class LinearBlocks(torch.autograd.Function):
    """y = Q(x) Q(W)^T + b; dx = Q(dy) Q'(W); dW = Q'(dy)^T Q'(x) (Q: blocks along the rows, Q': along the columns)."""

    @staticmethod
    def forward(ctx, x, w, bias):
        ctx.xt, ctx.wt = in_blocks(x.t()), in_blocks(w.t())
        ctx.types = w.dtype, None if bias is None else bias.dtype
        y = in_blocks(x) @ in_blocks(w).t()
        return (y if bias is None else y + bias.float()).to(x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        dx = (in_blocks(dy) @ ctx.wt.t()).to(dy.dtype)
        dw = (in_blocks(dy.t()) @ ctx.xt.t()).to(ctx.types[0])
        return dx, dw, None if ctx.types[1] is None else dy.float().sum(0).to(ctx.types[1])


def _far(a):
    """Where a sigmoid leaves fp32's range or nears that (a < -64: it is exp(a) there), and exp(a / 2): a factor for each side of
    a product, which may be far inside."""
    return a < -64, torch.exp(a.clamp(max=0) / 2)


def swiglu_f32(ab):
    a, b = ab.float().chunk(2, dim=-1)
    far, h = _far(a)
    return torch.where(far, (a * h) * (b * h), torch.nn.functional.silu(a) * b)


def swiglu_grad_f32(ab, dg):
    a, b = ab.float().chunk(2, dim=-1)
    dg, s = dg.float(), torch.sigmoid(a)
    far, h = _far(a)
    da = torch.where(far, (dg * h) * (b * h) * (1 + a), dg * b * s * (1 + a * (1 - s)))
    return torch.cat([da, torch.where(far, (dg * h) * (a * h), dg * a * s)], dim=-1)


class SwigluBlocks(torch.autograd.Function):
    """silu(a) b; the backward reads a and b in 8-bit blocks (each from its own first column)."""

    @staticmethod
    def forward(ctx, ab):
        ctx.ab = torch.cat([in_blocks(v) for v in ab.chunk(2, dim=-1)], dim=-1)
        return swiglu_f32(ab).to(ab.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dg):
        return swiglu_grad_f32(ctx.ab, dg).to(dg.dtype)


class MlpBlocks(torch.autograd.Function):
    """[a | b] = Q(x) Q(W1)^T in x's type, g = silu(a) b, y = Q(g) Q(W2)^T; the backward reads x, g, a and b in 8 bits."""

    @staticmethod
    def forward(ctx, x, w1, w2):
        ab = (in_blocks(x) @ in_blocks(w1).t()).to(x.dtype)
        g = swiglu_f32(ab)
        ctx.xt, ctx.w1t, ctx.w2t, ctx.gt = (in_blocks(v.t()) for v in (x, w1, w2, g))
        ctx.ab = in_blocks(ab)
        ctx.types = w1.dtype, w2.dtype
        return (in_blocks(g) @ in_blocks(w2).t()).to(x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        dg = (in_blocks(dy) @ ctx.w2t.t()).to(dy.dtype)
        dab = swiglu_grad_f32(ctx.ab, dg)
        return ((in_blocks(dab) @ ctx.w1t.t()).to(dy.dtype), (in_blocks(dab.t()) @ ctx.xt.t()).to(ctx.types[0]),
                (in_blocks(dy.t()) @ ctx.gt.t()).to(ctx.types[1]))
