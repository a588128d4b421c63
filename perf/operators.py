"""The operators of a routed diffusion-transformer block as single passes over real sizes: their plain forms in 32-bit
torch operations, the framework's own calls (``own = True``) and their definitions in 64 bits.

Four operators, each forward and (where training uses it) backward:

* route     scores of N tokens for E experts -> the k chosen experts and their weights
* dispatch  token rows into expert order, and the experts' rows back into token order, weighted
* sandwich  x_new = x + r gate rmsnorm(y) w_post;  h = rmsnorm(x_new) w (1 + scale) + shift
* rope      q/k RMSNorm and rotary positions with several axes (time, height, width)
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6


# ----------------------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of an autoregressive caption model through a 64-expert router (decoding: latency counts)
        dict(name="route decode 1x64", op="route", train=False, n=1, e=64, k=8, score="sigmoid", bias=True, groups=8,
             top_groups=4, renorm=True, scale=2.5, masked=0.0, dtype="float32"),
        # one micro-batch of 32 images of 1024 tokens through the 8-expert router of the MoE DiT
        dict(name="route train 32768x8", op="route", train=True, n=32768, e=8, k=2, score="softmax", bias=False,
             groups=1, top_groups=1, renorm=True, scale=1.0, masked=0.0, dtype="float32"),
        # a fine-grained router (many small experts) with group limits and a balance bias, some experts switched off
        dict(name="route train 65536x256", op="route", train=True, n=65536, e=256, k=8, score="sigmoid", bias=True,
             groups=8, top_groups=4, renorm=True, scale=2.5, masked=0.02, dtype="float32"),
        # decoding: the two experts' rows of one token
        dict(name="dispatch decode 1x2048", op="dispatch", train=False, n=1, d=2048, e=8, k=2, cap=0.0, pad=0.0,
             dtype="bfloat16"),
        # the MoE DiT's micro-batch with a fixed capacity per expert (factor 1.25)
        dict(name="dispatch train 32768x2048", op="dispatch", train=True, n=32768, d=2048, e=8, k=2, cap=1.25, pad=0.0,
             dtype="bfloat16"),
        # an odd number of right-padded caption tokens, many experts, no capacity limit
        dict(name="dispatch train 8191x1280", op="dispatch", train=True, n=8191, d=1280, e=64, k=8, cap=0.0, pad=0.1,
             dtype="bfloat16"),
        # sampling two 256-token images with the 576-wide test model: latency counts
        dict(name="sandwich infer 2x256x576", op="sandwich", train=False, b=2, t=256, d=576, post=True, gate=True,
             mod=True, pre=True, res=1.0, dtype="bfloat16"),
        # one micro-batch of the 2048-wide model
        dict(name="sandwich train 32x1024x2048", op="sandwich", train=True, b=32, t=1024, d=2048, post=True, gate=True,
             mod=True, pre=True, res=0.5, dtype="bfloat16"),
        # the 2560-wide model on odd image sizes, ungated branch without modulation
        dict(name="sandwich train 7x333x2560", op="sandwich", train=True, b=7, t=333, d=2560, post=True, gate=False,
             mod=False, pre=True, res=0.7, dtype="bfloat16"),
        # one new token of each of eight captions, one axis, heads of 64 (decoding: latency counts)
        dict(name="rope decode 8x1x12x64", op="rope", train=False, b=8, t=1, hq=12, hkv=4, hd=64, axes="64",
             norm=True, interleaved=False, dtype="bfloat16"),
        # 32 images of 32 x 32 tokens, two axes, the 2048-wide model's heads
        dict(name="rope train 32x1024x16x128", op="rope", train=True, b=32, t=1024, hq=16, hkv=16, hd=128,
             axes="64,64", norm=True, interleaved=True, dtype="bfloat16"),
        # one clip of 13 frames of 30 x 43 tokens, three axes, shared key heads
        dict(name="rope train 1x16770x20x128", op="rope", train=True, b=1, t=16770, hq=20, hkv=4, hd=128,
             axes="16,56,56", norm=True, interleaved=False, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "dispatch", "sandwich", "rope"])
    if op == "route":
        score = rng.choice(["softmax", "sigmoid"])
        groups = rng.choice([1, 1, 2, 4, 8])
        e = groups * _log(rng, 4, 256 // groups)
        top_groups = rng.randint(max(1, groups // 2), groups)
        k = rng.randint(1, min(8, top_groups * (e // groups)))
        return dict(op=op, train=rng.random() < 0.75, n=_log(rng, 1, 65536), e=e, k=k, score=score,
                    bias=rng.random() < 0.5, groups=groups, top_groups=top_groups, renorm=rng.random() < 0.7,
                    scale=rng.choice([1.0, 2.5]), masked=rng.choice([0.0, 0.0, 0.02]),
                    dtype=rng.choice(["float32", "float32", "bfloat16"]))
    if op == "dispatch":
        d = 8 * _log(rng, 8, 320)
        e = _log(rng, 2, 128)
        k = rng.randint(1, min(8, e))
        n = min(_log(rng, 1, 32768), (32768 * 2048 * 2) // (d * k))
        return dict(op=op, train=rng.random() < 0.75, n=max(1, n), d=d, e=e, k=k, cap=rng.choice([0.0, 1.0, 1.25]),
                    pad=rng.choice([0.0, 0.1]) if n >= 64 else 0.0, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]))
    if op == "sandwich":
        d = 8 * _log(rng, 16, 320)
        t = _log(rng, 1, 4096)
        b = max(1, min(_log(rng, 1, 64), (32768 * 2048) // (d * t)))
        gate, mod = rng.random() < 0.7, rng.random() < 0.7
        return dict(op=op, train=rng.random() < 0.75, b=b, t=t, d=d, post=rng.random() < 0.8, gate=gate, mod=mod,
                    pre=True, res=rng.choice([1.0, 0.5]), dtype=rng.choice(["bfloat16", "bfloat16", "float32"]))
    hd = rng.choice([64, 96, 128])
    hkv = rng.randint(1, 8)
    hq = hkv * rng.randint(1, 3)
    third = 2 * (hd // 6)
    axes = rng.choice([[hd], [hd // 2, hd // 2], [hd - 2 * third, third, third], [hd // 2]])
    t = _log(rng, 1, 16384)
    b = max(1, min(_log(rng, 1, 32), (32768 * 32 * 128) // (t * (hq + hkv) * hd)))
    return dict(op="rope", train=rng.random() < 0.75, b=b, t=t, hq=hq, hkv=hkv, hd=hd, axes=",".join(map(str, axes)),
                norm=rng.random() < 0.7, interleaved=rng.random() < 0.5,
                dtype=rng.choice(["bfloat16", "bfloat16", "float32"]))


def _axes(c):
    return [int(d) for d in c["axes"].split(",")]


def _capacity(c):
    return 0 if not c["cap"] else max(8, int(math.ceil(c["cap"] * c["n"] * c["k"] / c["e"] / 8)) * 8)


def _rows(c):
    return c["e"] * _capacity(c) if c["cap"] else c["n"] * c["k"]


# ----------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = getattr(torch, c["dtype"])
    s = {"case": c}

    def r(*shape, std=1.0, mean=0.0, dtype=None):
        return (torch.randn(*shape, device=DEV, generator=g) * std + mean).to(dtype or dt)

    leaf = c["train"]

    def p(t):
        return t.requires_grad_(leaf)

    if c["op"] == "route":
        logits = r(c["n"], c["e"], std=2.0, dtype=torch.float32)
        if c["masked"]:  # experts switched off for a token
            logits.masked_fill_(torch.rand(c["n"], c["e"], device=DEV, generator=g) < c["masked"], -math.inf)
        s["logits"] = p(logits.to(dt))
        s["bias"] = r(c["e"], std=0.05, dtype=torch.float32) if c["bias"] else None
        s["dw"] = r(c["n"], c["k"], dtype=torch.float32)
    elif c["op"] == "dispatch":
        n, e, k, d = c["n"], c["e"], c["k"], c["d"]
        # uneven popularity of the experts; k distinct experts of each token
        pop = torch.randn(e, device=DEV, generator=g) * 0.5
        noise = -torch.log(-torch.log(torch.rand(n, e, device=DEV, generator=g).clamp(1e-7, 1 - 1e-7)))
        idx = (pop + noise).topk(k, dim=1).indices.to(torch.int32)
        if c["pad"]:  # padding tokens have no expert
            idx.masked_fill_((torch.rand(n, device=DEV, generator=g) < c["pad"])[:, None], -1)
        s["idx"] = idx
        s["w"] = p(torch.rand(n, k, device=DEV, generator=g) * (idx >= 0))
        s["x"], s["y"] = p(r(n, d)), p(r(_rows(c), d))
        s["dxs"], s["dout"] = r(_rows(c), d), r(n, d)
    elif c["op"] == "sandwich":
        b, t, d = c["b"], c["t"], c["d"]
        s["x"], s["y"] = p(r(b, t, d, std=1.5)), p(r(b, t, d, std=0.7))
        mods = r(b, 6, d, std=0.3)  # shift / scale / gate rows of one modulation tensor, as the block splits it
        s["post_w"] = p(r(d, std=0.1, mean=1.0, dtype=torch.float32)) if c["post"] else None
        s["gate"] = p(mods[:, 2]) if c["gate"] else None
        s["w"] = p(r(d, std=0.1, mean=1.0, dtype=torch.float32))
        s["shift"], s["scale"] = (p(mods[:, 0]), p(mods[:, 1])) if c["mod"] else (None, None)
        s["dx_new"], s["dh"] = r(b, t, d), r(b, t, d)
    else:
        b, t, hq, hkv, hd = c["b"], c["t"], c["hq"], c["hkv"], c["hd"]
        qkv = r(b, t, (hq + 2 * hkv) * hd)  # q and k are read in place from the fused projection's rows
        s["q"] = p(qkv[..., :hq * hd].unflatten(-1, (hq, hd)))
        s["k"] = p(qkv[..., hq * hd:(hq + hkv) * hd].unflatten(-1, (hkv, hd)))
        s["axes"] = _axes(c)
        ends = (1024,) if len(s["axes"]) == 1 else (13, 128, 128)[-len(s["axes"]):]
        s["pos"] = torch.stack([torch.randint(0, m, (b, t), device=DEV, generator=g) for m in ends],
                               -1).to(torch.int32)
        s["q_w"] = p(r(hd, std=0.1, mean=1.0, dtype=torch.float32)) if c["norm"] else None
        s["k_w"] = p(r(hd, std=0.1, mean=1.0, dtype=torch.float32)) if c["norm"] else None
        s["dq"], s["dk"] = r(b, t, hq, hd), r(b, t, hkv, hd)
    s["leaves"] = {n: v for n, v in s.items() if isinstance(v, torch.Tensor) and v.requires_grad}
    return s


# ----------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------
def run(state):
    if not state["case"]["train"]:
        with torch.no_grad():
            return _forward(state)
    for v in state["leaves"].values():
        v.grad = None
    out = _forward(state)
    c = state["case"]
    pairs = {"route": (("w", "dw"),), "dispatch": (("xs", "dxs"), ("out", "dout")),
             "sandwich": (("x_new", "dx_new"), ("h", "dh")), "rope": (("q", "dq"), ("k", "dk"))}[c["op"]]
    torch.autograd.backward([out[a] for a, _ in pairs], [state[b] for _, b in pairs])
    out = {n: v.detach() for n, v in out.items()}
    out.update({"grad_" + n: v.grad for n, v in state["leaves"].items()})
    return out


def _forward(s):
    c = s["case"]
    if own:
        from trenowanie_generatora_obrazkow_b200.ops import fused as Fz
        from trenowanie_generatora_obrazkow_b200.ops import routing as Rt
        if c["op"] == "route":
            w, idx = Rt.route_experts(s["logits"], c["k"], score=c["score"], bias=s["bias"], groups=c["groups"],
                                      top_groups=c["top_groups"], renorm=c["renorm"], scale=c["scale"])
            return {"w": w, "idx": idx}
        if c["op"] == "dispatch":
            plan = Rt.expert_plan(s["idx"], c["e"], capacity=_capacity(c) or None)
            return {"slot": plan.slot, "offsets": plan.offsets, "counts": plan.counts,
                    "xs": Rt.expert_dispatch(s["x"], plan), "out": Rt.expert_combine(s["y"], s["w"], plan)}
        if c["op"] == "sandwich":
            x_new, h = Fz.sandwich_norm(s["x"], s["y"], s["gate"], s["post_w"], s["w"], s["shift"], s["scale"],
                                        res_scale=c["res"], eps=EPS)
            return {"x_new": x_new, "h": h}
        q, k = Fz.rope_axes(s["q"], s["k"], s["pos"], s["axes"], theta=10000.0, q_w=s["q_w"], k_w=s["k_w"],
                            interleaved=c["interleaved"], eps=EPS)
        return {"q": q, "k": k}
    return {"route": _plain_route, "dispatch": _plain_dispatch, "sandwich": _plain_sandwich,
            "rope": _plain_rope}[c["op"]](s, c)


def _plain_route(s, c):
    l = s["logits"].float()
    n, e = l.shape
    if c["score"] == "softmax":
        # a token with every expert switched off has no probabilities: zero weights
        ex = torch.exp(l - l.detach().amax(-1, keepdim=True).clamp(min=-3e38))
        p, key = ex / ex.sum(-1, keepdim=True).clamp(min=1e-20), l.detach()
    else:
        ex = torch.exp(torch.where(l >= 0, -l, l))  # at most 1: no overflow, and a gradient of 0 at -inf
        p = torch.where(l >= 0, torch.ones_like(ex), ex) / (1 + ex)
        key = p.detach()
    if s["bias"] is not None:
        key = key + s["bias"]
    if c["groups"] > 1:  # groups by their best score (softmax) or the sum of their two best (sigmoid)
        by = key.view(n, c["groups"], -1).sort(dim=-1, descending=True).values
        gs = by[..., 0] if c["score"] == "softmax" or by.shape[-1] == 1 else by[..., 0] + by[..., 1]
        kept = gs.sort(dim=-1, descending=True, stable=True).indices[:, :c["top_groups"]]
        on = torch.zeros(n, c["groups"], device=l.device, dtype=torch.bool).scatter_(1, kept, True)
        # experts of dropped groups come after every expert of a kept one, whatever their scores
        rank = key.sort(dim=-1, descending=True, stable=True).indices
        late = ~on.gather(1, rank // (e // c["groups"]))
        idx = rank.gather(1, late.to(torch.uint8).sort(dim=-1, stable=True).indices)[:, :c["k"]]
    else:
        idx = key.sort(dim=-1, descending=True, stable=True).indices[:, :c["k"]]
    w = p.gather(1, idx)
    if c["renorm"]:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    return {"w": w * c["scale"], "idx": idx.to(torch.int32)}


def _plain_dispatch(s, c):
    n, k, e, cap = c["n"], c["k"], c["e"], _capacity(c)
    flat = s["idx"].reshape(-1).long()
    rows = _rows(c)
    hit = flat[:, None] == torch.arange(e, device=flat.device)
    rank = (hit.cumsum(0) - 1).gather(1, flat.clamp(min=0)[:, None])[:, 0]
    counts = hit.sum(0)
    if cap:
        offsets = torch.arange(e + 1, device=flat.device) * cap
        slot = torch.where((flat >= 0) & (rank < cap), flat * cap + rank, -1)
    else:
        offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
        slot = torch.where(flat >= 0, offsets[flat.clamp(min=0)] + rank, -1)
    keep = slot >= 0
    at = torch.where(keep, slot, rows)  # dropped assignments share one row past the end
    x = s["x"].float()
    xs = x.new_zeros(rows + 1, c["d"]).index_copy(0, at, x.repeat_interleave(k, 0))[:rows]
    y = torch.cat([s["y"].float(), x.new_zeros(1, c["d"])])[at].view(n, k, -1)
    out = (y * s["w"][..., None] * keep.view(n, k, 1)).sum(1)
    i32 = torch.int32
    return {"slot": slot.view(n, k).to(i32), "offsets": offsets.to(i32), "counts": counts.to(i32),
            "xs": xs.to(s["x"].dtype), "out": out.to(s["y"].dtype)}


def _norm(x):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _plain_sandwich(s, c):
    x, u = s["x"].float(), s["y"].float()
    if s["post_w"] is not None:
        u = _norm(u) * s["post_w"]
    if s["gate"] is not None:
        u = u * s["gate"].float()[:, None]
    x_new = x + c["res"] * u
    h = _norm(x_new) * s["w"]
    if s["scale"] is not None:
        h = h * (1 + s["scale"].float()[:, None]) + s["shift"].float()[:, None]
    return {"x_new": x_new.to(s["x"].dtype), "h": h.to(s["x"].dtype)}


def _angles(pos, axes, dtype):
    """Angles of every rotated pair [B, T, sum(axes) / 2]: axis a rotates pair m of its axes[a] / 2 pairs by
    pos_a theta^(-2m / axes[a])."""
    parts = [pos[..., a:a + 1].to(dtype) / 10000.0 ** (torch.arange(0, d, 2, device=pos.device, dtype=dtype) / d)
             for a, d in enumerate(axes)]
    return torch.cat(parts, -1)


def _plain_rope(s, c):
    ang = _angles(s["pos"], s["axes"], torch.float32)[:, :, None]
    cos, sin = ang.cos(), ang.sin()
    half = sum(s["axes"]) // 2

    def turn(x, w):
        x = x.float()
        if w is not None:
            x = _norm(x) * w
        rot, rest = x[..., :2 * half], x[..., 2 * half:]
        if c["interleaved"]:
            a, b = rot[..., 0::2], rot[..., 1::2]
            rot = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = rot[..., :half], rot[..., half:]
            rot = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([rot, rest], -1)
    return {"q": turn(s["q"], s["q_w"]).to(s["q"].dtype), "k": turn(s["k"], s["k_w"]).to(s["k"].dtype)}


# ----------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    es = 2 if c["dtype"] == "bfloat16" else 4
    if c["op"] == "route":
        n, e, k = c["n"], c["e"], c["k"]
        b = n * e * es + n * k * 8 + (4 * e if c["bias"] else 0)
        if c["train"]:
            b += n * k * 4 + n * e * es
        return {"bytes": b, "flops": n * e * (8 if not c["train"] else 12)}
    if c["op"] == "dispatch":
        n, k, d, r = c["n"], c["k"], c["d"], _rows(c)
        # x, w, idx in; xs, out, slot, offsets, counts out; the expert rows that are used (all at most) in
        used = min(r, n * k)
        b = n * d * es + n * k * 8 + r * d * es + n * d * es + n * k * 4 + c["e"] * 8 + used * d * es
        f = 2 * n * k * d
        if c["train"]:  # dxs, dout in; dx, dy, dw out
            b += used * d * es + n * d * es + n * d * es + r * d * es + n * k * 4
            f *= 4
        return {"bytes": b, "flops": f}
    if c["op"] == "sandwich":
        m = c["b"] * c["t"] * c["d"]
        rows = c["b"] * c["d"] * es * ((1 if c["gate"] else 0) + (2 if c["mod"] else 0))
        w = 4 * c["d"] * (1 + (1 if c["post"] else 0))
        b, f = 4 * m * es + rows + w, 16 * m
        if c["train"]:
            b, f = b + 4 * m * es + rows + w, f + 32 * m
        return {"bytes": b, "flops": f}
    m = c["b"] * c["t"] * (c["hq"] + c["hkv"]) * c["hd"]
    b, f = 2 * m * es + c["b"] * c["t"] * len(_axes(c)) * 4, 8 * m
    if c["train"]:
        b, f = b + 2 * m * es, 24 * m
    return {"bytes": b, "flops": f}


# ----------------------------------------------------------------------------------------------------------------
# definitions in 64 bits, gradients from their formulas
# ----------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"route": _exact_route, "dispatch": _exact_dispatch, "sandwich": _exact_sandwich,
                "rope": _exact_rope}[case["op"]](s, case)


def _exact_route(s, c):
    # the choice is made on 32-bit scores, so the experts are those of the 32-bit scores here too
    idx = _plain_route({**s, "logits": s["logits"].detach()}, c)["idx"].long()
    l = s["logits"].detach().double()
    on = torch.zeros_like(l, dtype=torch.bool).scatter_(1, idx, True)
    p = torch.softmax(l, -1).nan_to_num(0.0) if c["score"] == "softmax" else torch.sigmoid(l)
    z = torch.ones_like(p[:, :1])
    if c["renorm"]:
        z = torch.where(on, p, torch.zeros_like(p)).sum(-1, keepdim=True) + 1e-20
    w = c["scale"] * p / z
    out = {"w": w.gather(1, idx), "idx": None}
    if c["train"]:
        up = torch.zeros_like(l).scatter_(1, idx, s["dw"].double())
        mean = (up * w).sum(-1, keepdim=True) / c["scale"]  # sum of weight times gradient over the chosen
        if c["renorm"]:
            dp = torch.where(on, c["scale"] * (up - mean) / z, torch.zeros_like(p))
        else:
            dp = c["scale"] * up
        if c["score"] == "softmax":
            out["grad_logits"] = p * (dp - (dp * p).sum(-1, keepdim=True))
        else:
            out["grad_logits"] = dp * p * torch.sigmoid(-l)
    return out


def _exact_dispatch(s, c):
    n, k = c["n"], c["k"]
    slot = _plain_dispatch({**s, "x": s["x"].detach(), "y": s["y"].detach(), "w": s["w"].detach()}, c)["slot"].long()
    x, y, w = s["x"].detach().double(), s["y"].detach().double(), s["w"].detach().double()
    keep = (slot >= 0).double()
    xs, out = torch.zeros_like(y), torch.zeros_like(x)
    dx, dy, dw = torch.zeros_like(x), torch.zeros_like(y), torch.zeros_like(w)
    dxs, dout = s["dxs"].double(), s["dout"].double()
    for j in range(k):
        t, at = keep[:, j].nonzero()[:, 0], slot[:, j][slot[:, j] >= 0]
        xs[at] = x[t]
        out[t] += w[t, j, None] * y[at]
        dx[t] += dxs[at]
        dy[at] = w[t, j, None] * dout[t]
        dw[t, j] = (dout[t] * y[at]).sum(-1)
    r = {"slot": None, "offsets": None, "counts": None, "xs": xs, "out": out}
    if c["train"]:
        r.update(grad_w=dw, grad_x=dx, grad_y=dy)
    return r


def _rms_back(g, n, r):
    """Gradient of the input of n = x r(x) from the gradient g of n."""
    return r * (g - n * (g * n).mean(-1, keepdim=True))


def _exact_sandwich(s, c):
    d = {n: v.detach().double() for n, v in s.items() if isinstance(v, torch.Tensor)}
    one = torch.ones((), device=DEV, dtype=torch.float64)
    gate = d["gate"][:, None] if "gate" in d else one
    sc = 1 + d["scale"][:, None] if "scale" in d else one
    sh = d["shift"][:, None] if "shift" in d else 0 * one
    ry = (d["y"].square().mean(-1, keepdim=True) + EPS) ** -0.5 if "post_w" in d else one
    pw = d.get("post_w", one)
    u = d["y"] * ry
    x_new = d["x"] + c["res"] * gate * pw * u
    rx = (x_new.square().mean(-1, keepdim=True) + EPS) ** -0.5
    n = x_new * rx
    out = {"x_new": x_new, "h": n * d["w"] * sc + sh}
    if c["train"]:
        dx = d["dx_new"] + _rms_back(d["dh"] * d["w"] * sc, n, rx)
        du = c["res"] * gate * pw * dx
        out["grad_x"] = dx
        out["grad_y"] = _rms_back(du, u, ry) if "post_w" in d else du
        if "post_w" in d:
            out["grad_post_w"] = (c["res"] * gate * dx * u).sum((0, 1))
        if "gate" in d:
            out["grad_gate"] = (c["res"] * pw * u * dx).sum(1)
        out["grad_w"] = (d["dh"] * n * sc).sum((0, 1))
        if "scale" in d:
            out["grad_shift"], out["grad_scale"] = d["dh"].sum(1), (d["dh"] * n * d["w"]).sum(1)
    return out


def _exact_rope(s, c):
    ang = _angles(s["pos"], s["axes"], torch.float64)[:, :, None]
    z = torch.polar(torch.ones_like(ang), ang)
    m = 2 * ang.shape[-1]

    def turn(x, z):
        rot = x[..., :m]
        if c["interleaved"]:
            v = torch.view_as_real(torch.view_as_complex(rot.unflatten(-1, (-1, 2)).contiguous()) * z).flatten(-2)
        else:
            v = torch.complex(rot[..., :m // 2], rot[..., m // 2:]) * z
            v = torch.cat([v.real, v.imag], -1)
        return torch.cat([v, x[..., m:]], -1)

    out, grads = {}, {}
    for name, wn in (("q", "q_w"), ("k", "k_w")):
        x = s[name].detach().double()
        w = s[wn].detach().double() if s[wn] is not None else None
        r = (x.square().mean(-1, keepdim=True) + EPS) ** -0.5 if w is not None else 1.0
        n = x * r
        out[name] = turn(n if w is None else n * w, z)
        if c["train"]:
            g = turn(s["d" + name].double(), z.conj())
            grads["grad_" + name] = g if w is None else _rms_back(g * w, n, r)
            if w is not None:
                grads["grad_" + wn] = (g * n).sum((0, 1, 2))
    return {**out, **grads}
