"""Matrix products of 8-bit floating point with a scale for each block of 128, and activations kept in 8 bits for the
backward pass, as single passes over real sizes: their plain forms in 32-bit torch operations, the framework's own calls
(``own = True``) and their definitions in 64 bits.

The 8-bit form of a row is cut into blocks of 128 numbers along the axis that a product sums over. A block with the largest
finite magnitude A has the scale 2^e, e the smallest whole number >= -127 with A <= 448 2^e, and holds x / 2^e rounded to
e4m3 (to nearest, ties to even; what is not finite is held as NaN). Q(x) are the values that the codes stand for with blocks
along the rows of x, Q'(x) with blocks along its columns. Five operators:

* pack    x -> Q(x) (a checkpoint kept in 8 bits and read again), or Q(x) and Q'(x)
* serve   y = Q(x) W^T + b with W held in 8 bits
* linear  y = Q(x) Q(W)^T + b;  dx = Q(dy) Q'(W);  dW = Q'(dy)^T Q'(x);  db = the column sums of dy
* mlp     [a | b] = Q(x) Q(W1)^T rounded to x's type;  g = silu(a) b;  y = Q(g) Q(W2)^T;  the backward reads x, g, [a | b]
          in 8 bits: dg = Q(dy) Q'(W2) rounded;  [da | db] = dsilu of Q([a | b]);  dx = Q(dab) Q'(W1);
          dW1 = Q'(dab)^T Q'(x);  dW2 = Q'(dy)^T Q'(g)
* swiglu  g = silu(a) b;  [da | db] from dg and Q(a), Q(b), whose blocks start at their own first columns
"""
import math

import torch

own = False

DEV = "cuda"


# ----------------------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the checkpoint of one small image's tokens in the 640-wide model: latency counts
        dict(name="pack 256x640 rows", op="pack", m=256, k=640, side="rows", dtype="float16"),
        # one micro-batch of 32 images of 1024 tokens: the operand of the forward and of the weight gradient in one pass
        dict(name="pack 32768x2048 both", op="pack", m=32768, k=2048, side="both", dtype="bfloat16"),
        # one token through the qkv projection of a model held in 8 bits: reading the weight counts
        dict(name="serve 1x2048->6144", op="serve", m=1, k=2048, n=6144, bias=False, dtype="bfloat16"),
        # a few tokens of a 1280-wide refiner, a layer with a bias
        dict(name="serve 7x1280->3456", op="serve", m=7, k=1280, n=3456, bias=True, dtype="float16"),
        # sampling one 1024 px image: 4096 tokens through the MLP's up projection
        dict(name="serve 4096x2048->11008", op="serve", m=4096, k=2048, n=11008, bias=False, dtype="bfloat16"),
        # training: the micro-batch's qkv projection, fp32 master weights
        dict(name="linear 32768x2048->6144", op="linear", m=32768, k=2048, n=6144, bias=False, dtype="bfloat16"),
        # text tokens of 15 captions of 77, fp32 states, a layer with a bias
        dict(name="linear 1155x1280->3840", op="linear", m=1155, k=1280, n=3840, bias=True, dtype="float32"),
        # widths that end inside a block and inside a vector
        dict(name="linear 2047x1000->777", op="linear", m=2047, k=1000, n=777, bias=False, dtype="bfloat16"),
        # the SwiGLU MLP of the 2048-wide model over one micro-batch, bf16 weights
        dict(name="mlp 32768x2048x5504", op="mlp", m=32768, k=2048, h=5504, dtype="bfloat16"),
        # the MLP of the 512-wide text encoder over an odd number of tokens
        dict(name="mlp 333x512x1408", op="mlp", m=333, k=512, h=1408, dtype="bfloat16"),
        # the activation alone, its input kept in 8 bits
        dict(name="swiglu 32768x5504", op="swiglu", m=32768, h=5504, dtype="bfloat16"),
        # the text refiner's activation over one caption
        dict(name="swiglu 77x1408", op="swiglu", m=77, h=1408, dtype="float16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pack", "serve", "linear", "mlp", "swiglu"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])

    def width(lo, hi):  # mostly whole vectors, some odd
        w = _log(rng, lo, hi)
        return w if rng.random() < 0.25 else max(8, w // 8 * 8)

    if op == "pack":
        k = width(64, 5504)
        return dict(op=op, m=max(1, min(_log(rng, 1, 32768), 32768 * 2048 // k)), k=k,
                    side=rng.choice(["rows", "cols", "both"]), dtype=dtype)
    if op == "serve":
        k, n = width(64, 5504), width(64, 11008)
        m = rng.choice([_log(rng, 1, 16), _log(rng, 1, 4096)])
        return dict(op=op, m=max(1, min(m, 4096 * 2048 * 11008 // (k * n))), k=k, n=n, bias=rng.random() < 0.4, dtype=dtype)
    if op == "linear":
        k, n = width(64, 2560), width(64, 6912)
        return dict(op=op, m=max(1, min(_log(rng, 1, 32768), 32768 * 2048 * 6144 // (k * n))), k=k, n=n,
                    bias=rng.random() < 0.4, dtype=dtype)
    h = 128 * _log(rng, 3, 43)
    if op == "mlp":
        k = 64 * _log(rng, 2, 32)
        return dict(op=op, m=_log(rng, 1, 32768), k=k, h=h, dtype=rng.choice(["bfloat16", "bfloat16", "float16"]))
    return dict(op=op, m=max(1, min(_log(rng, 1, 32768), 32768 * 5504 // h)), h=h if rng.random() < 0.7 else width(64, 5504),
                dtype=dtype)


# ----------------------------------------------------------------------------------------------------------------
# inputs
# ----------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = getattr(torch, c["dtype"])
    s = {"case": c}

    def r(*shape, std=1.0, spread=0.0, dtype=None):
        t = torch.randn(*shape, device=DEV, generator=g) * std
        if spread:  # channels of unequal size, as behind a norm's weight
            t *= torch.exp(torch.randn(shape[-1], device=DEV, generator=g) * spread)
        return t.to(dtype or dt)

    if c["op"] == "pack":
        s["x"] = r(c["m"], c["k"], spread=0.5)
    elif c["op"] == "serve":
        s["x"] = r(c["m"], c["k"], spread=0.5)
        # the weight as the program holds it: codes [N, K padded to 128], a byte per block of 128 (see _unpack)
        s["w"] = _lay_out(r(c["n"], c["k"], std=c["k"] ** -0.5, dtype=torch.float32))
        s["bias"] = r(c["n"], std=0.1, dtype=torch.float32) if c["bias"] else None
    elif c["op"] == "linear":
        s["x"] = r(c["m"], c["k"], spread=0.5).requires_grad_()
        s["w"] = r(c["n"], c["k"], std=c["k"] ** -0.5, dtype=torch.float32).requires_grad_()
        s["bias"] = r(c["n"], std=0.1, dtype=torch.float32).requires_grad_() if c["bias"] else None
        s["dy"] = r(c["m"], c["n"], std=0.01, spread=0.5)
    elif c["op"] == "mlp":
        s["x"] = r(c["m"], c["k"], spread=0.5).requires_grad_()
        s["w1"] = r(2 * c["h"], c["k"], std=c["k"] ** -0.5).requires_grad_()
        s["w2"] = r(c["k"], c["h"], std=c["h"] ** -0.5).requires_grad_()
        s["dy"] = r(c["m"], c["k"], std=0.1, spread=0.5)
    else:
        s["x"] = r(c["m"], 2 * c["h"], spread=0.3).requires_grad_()
        s["dy"] = r(c["m"], c["h"], std=0.1)
    return s


def _lay_out(w):
    """(codes [N, Kp] e4m3, bytes [ceil(N / 128), ceil(Kp / 512), 32, 4, 4]): the scale 2^(byte - 127) of row
    128 i + 32 c + r and block 4 j + b stands at [i, j, r, c, b]."""
    v, e = _blocks(w)
    n, nb = e.shape
    codes = torch.ldexp(v, -e[..., None]).to(torch.float8_e4m3fn).reshape(n, nb * 128)
    rt, kq = -(-n // 128), -(-nb // 4)
    full = torch.zeros(rt * 128, kq * 4, dtype=torch.uint8, device=w.device)
    full[:n, :nb] = (e + 127).to(torch.uint8)
    return codes, full.view(rt, 4, 32, kq, 4).permute(0, 3, 2, 1, 4).contiguous()


def _unpack(codes, scales, k):
    rt, kq = scales.shape[:2]
    n, kp = codes.shape
    e = scales.permute(0, 3, 2, 1, 4).reshape(rt * 128, kq * 4)[:n, :kp // 128].int() - 127
    return torch.ldexp(codes.float().view(n, kp // 128, 128), e[..., None]).view(n, kp)[:, :k]


# ----------------------------------------------------------------------------------------------------------------
# plain forms
# ----------------------------------------------------------------------------------------------------------------
def _blocks(x):
    """(the values of x in 8 bits as blocks [M, ceil(K / 128), 128] in 32 bits, the scales' exponents [M, ceil(K / 128)])"""
    m, k = x.shape
    f = torch.nn.functional.pad(x.detach().float(), (0, -k % 128)).view(m, -1, 128)
    top = torch.where(f.isfinite(), f.abs(), 0.0).amax(-1)
    frac, e = torch.frexp(top)  # top = frac 2^e, 1/2 <= frac < 1; 448 = 7/8 2^9
    e = torch.where(frac <= 0.875, e - 9, e - 8).clamp_min(-127)
    e = torch.where(top == 0, -127, e)
    q = torch.ldexp(f, -e[..., None])
    q = torch.where(q.isfinite(), q, math.nan).to(torch.float8_e4m3fn).float()
    return torch.ldexp(q, e[..., None]), e


def _q(x):
    """Q(x)"""
    return _blocks(x)[0].view(x.shape[0], -1)[:, :x.shape[1]]


def _qt(x):
    """Q'(x)"""
    return _q(x.t()).t()


def _plain(s):
    c, dt = s["case"], getattr(torch, s["case"]["dtype"])
    x = s["x"].detach()
    if c["op"] == "pack":
        return [_q(x).to(dt)] * (c["side"] != "cols") + [_qt(x).to(dt)] * (c["side"] != "rows")
    if c["op"] == "serve":
        y = _q(x) @ _unpack(*s["w"], c["k"]).t()
        return [(y if s["bias"] is None else y + s["bias"]).to(dt)]
    dy = s["dy"]
    if c["op"] == "linear":
        w, b = s["w"].detach(), s["bias"]
        y = _q(x) @ _q(w).t()
        out = [(y if b is None else y + b.detach()).to(dt), (_q(dy) @ _qt(w)).to(dt), _qt(dy).t() @ _qt(x)]
        return out if b is None else out + [dy.float().sum(0)]
    if c["op"] == "mlp":
        w1, w2 = s["w1"].detach(), s["w2"].detach()
        ab = (_q(x) @ _q(w1).t()).to(dt)
        g = _silu_mul(ab)
        y = (_q(g) @ _q(w2).t()).to(dt)
        dg = (_q(dy) @ _qt(w2)).to(dt)
        dab = _silu_mul_grad(_q(ab), dg)
        return [y, (_q(dab) @ _qt(w1)).to(dt), (_qt(dab).t() @ _qt(x)).to(dt), (_qt(dy).t() @ _qt(g)).to(dt)]
    return [_silu_mul(x).to(dt), _silu_mul_grad(torch.cat([_q(v) for v in x.chunk(2, dim=1)], dim=1), dy).to(dt)]


def _silu_mul(ab):
    a, b = ab.float().chunk(2, dim=1)
    return a / (1 + torch.exp(-a)) * b


def _silu_mul_grad(ab, dg):
    a, b = ab.float().chunk(2, dim=1)
    dg, s = dg.float(), 1 / (1 + torch.exp(-a))
    return torch.cat([dg * b * s * (1 + a * (1 - s)), dg * a * s], dim=1)


def _own(s):
    from trenowanie_generatora_obrazkow_b200.ops import blocks8 as B8
    c, dt = s["case"], getattr(torch, s["case"]["dtype"])
    if c["op"] == "pack":
        got = B8.quantize_blocks(s["x"], c["side"])
        if c["side"] == "rows":
            return [B8.dequantize_blocks(got, dt)]
        if c["side"] == "cols":
            return [B8.dequantize_blocks(got, dt).t()]
        return [B8.dequantize_blocks(got[0], dt), B8.dequantize_blocks(got[1], dt).t()]
    if c["op"] == "serve":
        return [B8.linear_blocks(s["x"], B8.Blocks8(*s["w"], c["k"]), s["bias"])]
    leaves = [s[name] for name in ("x", "w", "w1", "w2", "bias") if s.get(name) is not None]
    for t in leaves:
        t.grad = None
    if c["op"] == "linear":
        y = B8.linear_blocks(s["x"], s["w"], s["bias"])
    elif c["op"] == "mlp":
        y = B8.mlp_blocks(s["x"], s["w1"], s["w2"])
    else:
        y = B8.swiglu_blocks(s["x"])
    y.backward(s["dy"])
    return [y.detach()] + [t.grad for t in leaves]


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ----------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    size = 4 if c["dtype"] == "float32" else 2
    m = c["m"]
    if c["op"] == "pack":  # x in, the values of each side out
        return {"bytes": m * c["k"] * size * (1 + (2 if c["side"] == "both" else 1)), "flops": 0}
    if c["op"] == "serve":  # x and 8-bit weights in, y out
        k, n = c["k"], c["n"]
        return {"bytes": (m * k + m * n) * size + n * k * (1 + 1 / 128), "flops": 2 * m * n * k}
    if c["op"] == "linear":  # x, dy, W in; y, dx, dW out
        k, n = c["k"], c["n"]
        return {"bytes": 2 * (m * k + m * n) * size + 8 * n * k, "flops": 6 * m * n * k}
    if c["op"] == "mlp":  # x, dy, W1, W2 in; y, dx, dW1, dW2 out
        k, h = c["k"], c["h"]
        return {"bytes": 4 * m * k * size + 2 * 3 * h * k * size, "flops": 6 * m * 3 * h * k}
    return {"bytes": m * c["h"] * size * (2 + 1 + 1 + 2), "flops": 0}  # ab, dg in; g, dab out


# ----------------------------------------------------------------------------------------------------------------
# definitions in 64 bits
# ----------------------------------------------------------------------------------------------------------------
def _grid(x, dim):
    """The values that 8 bits hold of x [M, K] with blocks of 128 along dim, in 64 bits."""
    x = x.detach().double()
    if dim == 0:
        return _grid(x.t(), 1).t()
    m, k = x.shape
    out = torch.empty_like(x)
    for lo in range(0, k, 128):
        v = x[:, lo:lo + 128]
        top = v.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2((top / 448).clamp_min(2.0 ** -200)))
        # the logarithm's rounding: the smallest whole e with top <= 448 2^e
        e = torch.where(top <= 448 * torch.exp2(e - 1), e - 1, e)
        e = torch.where(top > 448 * torch.exp2(e), e + 1, e).clamp_min(-127)
        scale = torch.exp2(e)
        u = v / scale
        # e4m3: steps of 2^-3 of the power of two below, of 2^-9 under 2^-6
        p = torch.frexp(u.abs().clamp_min(2.0 ** -6))[1] - 1
        step = torch.exp2((p - 3).double())
        out[:, lo:lo + 128] = torch.round(u / step) * step * scale  # torch.round: ties to even
    return out


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    dt = getattr(torch, c["dtype"])
    x = s["x"].detach()
    if c["op"] == "pack":
        return [_grid(x, 1)] * (c["side"] != "cols") + [_grid(x, 0)] * (c["side"] != "rows")
    if c["op"] == "serve":
        y = _grid(x, 1) @ _unpack(*s["w"], c["k"]).double().t()
        return [y if s["bias"] is None else y + s["bias"].double()]
    dy = s["dy"]
    if c["op"] == "linear":
        w = s["w"].detach()
        y = _grid(x, 1) @ _grid(w, 1).t()
        out = [y if s["bias"] is None else y + s["bias"].detach().double(), _grid(dy, 1) @ _grid(w, 0),
               _grid(dy, 0).t() @ _grid(x, 0)]
        return out if s["bias"] is None else out + [dy.double().sum(0)]
    if c["op"] == "mlp":
        w1, w2 = s["w1"].detach(), s["w2"].detach()
        ab = (_grid(x, 1) @ _grid(w1, 1).t()).to(dt).double()
        h = c["h"]
        g = ab[:, :h] * torch.sigmoid(ab[:, :h]) * ab[:, h:]
        dg = (_grid(dy, 1) @ _grid(w2, 0)).to(dt).double()
        dab = _dswiglu64(_grid(ab, 1), dg)
        y = _grid(g, 1) @ _grid(w2, 1).t()
        return [y, _grid(dab, 1) @ _grid(w1, 0), _grid(dab, 0).t() @ _grid(x, 0), _grid(dy, 0).t() @ _grid(g, 0)]
    h = c["h"]
    x64 = x.double()
    kept = torch.cat([_grid(x[:, :h], 1), _grid(x[:, h:], 1)], dim=1)
    return [x64[:, :h] * torch.sigmoid(x64[:, :h]) * x64[:, h:], _dswiglu64(kept, dy.double())]


def _dswiglu64(ab, dg):
    h = dg.shape[1]
    a, b = ab[:, :h], ab[:, h:]
    s = torch.sigmoid(a)
    return torch.cat([dg * b * (s + a * s * (1 - s)), dg * a * s], dim=1)
