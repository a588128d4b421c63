"""Matrix products of 8-bit floating point with a scale for each block of 128, and activations kept in 8 bits for the
backward pass (csrc/blocks8.cu, csrc/gemm8.cu).

    w8 = quantize_blocks(layer.weight)            # a weight held in 8 bits
    y  = linear_blocks(x, w8, bias)               # serving; one launch for up to 16 rows
    y  = linear_blocks(x, layer)                  # training: forward and both gradients on 8-bit products
    y  = mlp_blocks(x, in_proj, out_proj)         # SwiGLU MLP, activations packed by the kernel that makes them
    g  = swiglu_blocks(ab)                        # silu(a) b, its input kept in 8 bits for the backward

A row is cut into blocks of 128 along the axis that a product sums over. A block whose largest finite magnitude is A has the
scale 2^e, e the smallest whole number >= -127 with A <= 448 2^e, and holds x / 2^e rounded to e4m3; infinities and NaN are
held as NaN. With Q(x) the values held of x with blocks along its rows and Q'(x) with blocks along its columns:

    y = Q(x) Q(W)^T + b        dx = Q(dy) Q'(W)        dW = Q'(dy)^T Q'(x)        db = column sums of dy

Q' is written by the pass that packs Q. A backward keeps no activation in its own type: the checkpoint of x is Q'(x), the
operand of the weight's gradient, one byte a value. Sums are fp32; the gradients pass Q straight through.

Differentiable once. The gradients of fp32 leaves (weights, biases) are accumulated in place into their ``.grad`` like those
of ``fused.linear`` (``torch.autograd.grad`` does not return them, tensor hooks on them do not run); other weights get theirs
from autograd in their own type. A weight or bias that requires no gradient in the forward gets none, nor does one that is
frozen by the time of the backward. CUDA tensors run the sm_100a kernels, CPU tensors the definitions of ``reference.py``.
"""
from typing import NamedTuple

import torch

from . import reference as R
from ._ext import err_buf, ext, _ERR


class Blocks8(NamedTuple):
    """A matrix in 8-bit blocks along its rows: codes float8_e4m3fn [rows, width] (width: cols rounded up to 128, zeros past
    cols), scales uint8 [ceil(rows / 128), ceil(width / 512), 32, 4, 4] (the scale 2^(byte - 127) of row 128 i + 32 c + r and
    block 4 j + b stands at [i, j, r, c, b]) and the number of columns."""
    codes: torch.Tensor
    scales: torch.Tensor
    cols: int

    @property
    def shape(self):
        return torch.Size((self.codes.shape[0], self.cols))


def _err_word(t):
    buf = _ERR.get(t.get_device())
    return buf if buf is not None else err_buf(t.device)


def quantize_blocks(x, side="rows"):
    """x [M, K] (bf16, fp16 or fp32) -> Blocks8 of x (side "rows": blocks along the rows), of x^T ("cols": blocks along the
    columns, the rows of the result) or both as a pair, written by one pass over x. No gradient passes."""
    if side not in ("rows", "cols", "both"):
        raise ValueError(f"quantize_blocks: side is 'rows', 'cols' or 'both', not {side!r}")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"quantize_blocks: a matrix of at least one column expected, got {tuple(x.shape)}")
    M, K = x.shape
    if x.is_cuda:
        t = ext().pack8(x, side != "cols", side != "rows")
    else:
        t = (R.quantize_blocks(x) if side != "cols" else ()) + (R.quantize_blocks(x.t()) if side != "rows" else ())
    if side == "both":
        return Blocks8(t[0], t[1], K), Blocks8(t[2], t[3], M)
    return Blocks8(t[0], t[1], K if side == "rows" else M)


def dequantize_blocks(b, dtype=torch.bfloat16):
    """The values that a Blocks8 holds, [rows, cols] in dtype (exact in bf16 and fp32 down to 2^-126; fp16 rounds)."""
    if not b.codes.is_cuda:
        return R.dequantize_blocks(*b).to(dtype)
    return ext().unpack8(b.codes, b.scales, b.cols, dtype)


def gemm_blocks(a, b, out=None, bias=None, dtype=torch.bfloat16, accumulate=False):
    """C = a b^T (+ bias) of two Blocks8 [M, K] and [N, K] -> [M, N] in ``dtype`` (bf16, fp16 or fp32), or into ``out``
    (rows of any stride; fp32 ``out`` with accumulate: added to it). fp32 results are joined from parts of 4096 along K."""
    if a.cols != b.cols:
        raise ValueError(f"gemm_blocks: sums over {a.cols} and {b.cols}")
    if accumulate and (out is None or out.dtype != torch.float32 or bias is not None):
        raise ValueError("gemm_blocks: accumulate takes an fp32 out and no bias")
    if not a.codes.is_cuda:
        c = R.dequantize_blocks(*a) @ R.dequantize_blocks(*b).t()
        c = c if bias is None else c + bias.float()
        if out is None:
            return c.to(dtype)
        return out.add_(c) if accumulate else out.copy_(c)
    return ext().gemm8(a.codes, a.scales, b.codes, b.scales, a.cols, dtype, out, bias, accumulate, _err_word(a.codes))


def _weight_of(layer, what):
    if isinstance(layer, torch.nn.Linear):
        return layer.weight, layer.bias
    if isinstance(layer, (torch.Tensor, Blocks8)):
        return layer, None
    raise TypeError(f"{what}: an nn.Linear, a weight tensor or a Blocks8 expected, got {type(layer).__name__}")


def _no_graph(*ts):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise RuntimeError("a weight held in 8 bits passes no gradient on (use torch.no_grad() or detach x)")


def linear_blocks(x, layer_or_weight, bias=None):
    """y = Q(x) Q(W)^T + b: x [..., K] (bf16, fp16 or fp32) -> [..., N] in x's type. W: an ``nn.Linear``, a weight tensor
    [N, K] (packed in the call) or a Blocks8 (held in 8 bits; passes no gradient on). bias [N] fp32 or a 16-bit type. Rows of
    any stride are read in place, other layouts copied."""
    if type(layer_or_weight) is Blocks8 and x.is_cuda and x.dim() == 2 and x.shape[1] == layer_or_weight[2]:
        return ext().linear8_frozen(x, *layer_or_weight, bias, _err_word(x))  # a single token's cost is the host's
    w, own_bias = _weight_of(layer_or_weight, "linear_blocks")
    if own_bias is not None:
        if bias is not None:
            raise ValueError("linear_blocks: the layer has a bias of its own")
        bias = own_bias
    N, K = w.shape
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"linear_blocks: x [..., {K}] expected, got {tuple(x.shape)}")
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    if not x.is_cuda:
        if isinstance(w, Blocks8):
            _no_graph(x, bias)
            y = R.in_blocks(x2) @ R.dequantize_blocks(*w).t()
            y = (y if bias is None else y + bias.float()).to(x.dtype)
        else:
            y = R.LinearBlocks.apply(x2, w, bias)
    elif isinstance(w, Blocks8):
        y = ext().linear8_frozen(x2, w.codes, w.scales, K, bias, _err_word(x))
    else:
        y = ext().linear8(x2, w, bias, _err_word(x))
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)


def swiglu_blocks(ab):
    """silu(a) b for ab [..., 2 H] = [a | b] (bf16, fp16 or fp32) -> [..., H]; the backward reads a and b from 8-bit blocks
    (half the bytes of 16-bit ones; each half's blocks start at its first column)."""
    if ab.dim() < 1 or ab.shape[-1] < 2 or ab.shape[-1] % 2:
        raise ValueError(f"swiglu_blocks: [..., 2 H] expected, got {tuple(ab.shape)}")
    ab2 = ab if ab.dim() == 2 else ab.reshape(-1, ab.shape[-1])
    g = ext().swiglu8(ab2) if ab.is_cuda else R.SwigluBlocks.apply(ab2)
    return g if ab.dim() == 2 else g.view(*ab.shape[:-1], ab.shape[-1] // 2)


def mlp_blocks(x, in_proj, out_proj):
    """SwiGLU MLP on 8-bit products: [a | b] = Q(x) Q(W1)^T rounded to x's type, g = silu(a) b, y = Q(g) Q(W2)^T; x [..., K],
    in_proj [2 H, K], out_proj [N, H] (``nn.Linear`` without bias, weight tensors, or both Blocks8: held in 8 bits, no gradient)
    -> [..., N]. With H a multiple of 128, g, [a | b] and their gradient are written in 8 bits only (of 16-bit types by the first
    product itself; [a | b] where the backward wants it); other widths run ``linear_blocks``, ``swiglu_blocks`` and
    ``linear_blocks`` (g is then rounded to x's type before it is packed)."""
    w1, b1 = _weight_of(in_proj, "mlp_blocks")
    w2, b2 = _weight_of(out_proj, "mlp_blocks")
    if b1 is not None or b2 is not None:
        raise ValueError("mlp_blocks: projections without bias expected")
    held = isinstance(w1, Blocks8)
    if held != isinstance(w2, Blocks8):
        raise TypeError("mlp_blocks: both weights held in 8 bits, or neither")
    if len(w1.shape) != 2 or len(w2.shape) != 2 or w1.shape[0] != 2 * w2.shape[1] or x.dim() < 1 or x.shape[-1] != w1.shape[1]:
        raise ValueError(f"mlp_blocks: x [..., K], in_proj [2 H, K] and out_proj [N, H] expected, got {tuple(x.shape)}, "
                         f"{tuple(w1.shape)} and {tuple(w2.shape)}")
    if w2.shape[1] % 128:
        return linear_blocks(swiglu_blocks(linear_blocks(x, w1)), w2)
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if x.is_cuda:
        if held:
            y = ext().mlp8_frozen(x2, w1.codes, w1.scales, w2.codes, w2.scales, w1.cols, w2.cols, _err_word(x))
        else:
            y = ext().mlp8(x2, w1, w2, _err_word(x))
    elif held:
        _no_graph(x2)
        g = R.swiglu_f32((R.in_blocks(x2) @ R.dequantize_blocks(*w1).t()).to(x.dtype))
        y = (R.in_blocks(g) @ R.dequantize_blocks(*w2).t()).to(x.dtype)
    else:
        y = R.MlpBlocks.apply(x2, w1, w2)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], w2.shape[0])
