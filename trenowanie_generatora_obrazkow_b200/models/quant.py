"""Frozen quantized projections for teacher models (reference aurora/klein.py:45-107), and 8-bit products for this
framework's own blocks.

* ``QLinear``: 8-bit weights with one scale per group of ``group`` consecutive inputs of an output row, symmetric
  int8 (max |w| / 127) or fp8 e4m3 (max |w| / 448, e4m3's largest normal value); dequantised to the activation dtype
  and multiplied with the framework's GEMM (``ops.fused.linear``: the tcgen05 kernel on CUDA). Halves the weight
  memory of a frozen teacher; the arithmetic stays bf16.
* ``W8A8Linear``: per-output-channel int8 weights, dynamic per-token int8 activations, int32 accumulation. On CUDA
  the activations are quantised by one kernel and multiplied by the tcgen05 ``kind::i8`` GEMM with both scales
  applied in its epilogue (``ext().quantize_rows_i8``, ``ext().gemm_i8``); elsewhere ``torch._int_mm``. Used for
  frozen teachers only.
* ``BlockLinear``: e4m3 weights with a power-of-two scale for each 128 inputs, activations packed the same way in the call
  (``ops.blocks8``): one launch for up to 16 rows, the block-scaled tcgen05 product above. No gradient: an input that wants
  one is refused.
* ``quantize(module, kind)``: replaces every ``nn.Linear`` below ``module`` in place (kind "int8", "fp8", "fp8_block" or
  "w8a8"; w8a8 only where both feature counts are multiples of 8, as the int8 GEMM requires) but the routers of experts,
  whose scores are computed from their weights in fp32. Plain modules, and this framework's own models for inference.
* ``use_fp8(module)``: the linear layers of every DiT, routed and text block below ``module`` (not the routed experts, nor
  the routers, whose scores stay fp32) run on 8-bit products, in training forward and backward (fp32 master weights and
  gradients, ``ops.blocks8.linear_blocks`` / ``mlp_blocks``), without gradients with weights packed once per version.
  Parameters and checkpoints keep their names and types.
"""
import torch
import torch.nn as nn

from ..ops import blocks8 as B8
from ..ops import fused as Fz


class QLinear(nn.Module):
    def __init__(self, lin: nn.Linear, kind: str = "int8", group: int = 128):
        super().__init__()
        assert kind in ("int8", "fp8"), kind
        w = lin.weight.detach().float()
        out, inp = w.shape
        g = group if inp % group == 0 else inp
        wg = w.view(out, inp // g, g)
        top = 127.0 if kind == "int8" else 448.0
        scale = wg.abs().amax(-1, keepdim=True).clamp_min(1e-12) / top
        if kind == "int8":
            q = torch.round(wg / scale).clamp_(-127, 127).to(torch.int8)
        else:
            q = (wg / scale).to(torch.float8_e4m3fn)
        self.register_buffer("w", q)
        self.register_buffer("s", scale.to(torch.bfloat16))
        self.bias = lin.bias
        self.kind, self.shape = kind, (out, inp)

    def dequantized(self, dtype):
        return (self.w.to(dtype) * self.s.to(dtype)).view(self.shape)

    def forward(self, x):
        w = self.dequantized(x.dtype if x.is_floating_point() else torch.bfloat16)
        y = Fz.linear(x, w) if x.is_cuda else torch.nn.functional.linear(x, w)
        return y + self.bias if self.bias is not None else y


class W8A8Linear(nn.Module):
    def __init__(self, lin: nn.Linear):
        super().__init__()
        w = lin.weight.detach().float()
        scale = w.abs().amax(1).clamp_min(1e-12) / 127
        self.register_buffer("scale", scale)
        # [in, out] view of the row-major [out, in] int8 matrix (the layout the int8 GEMM takes for its B operand)
        self.register_buffer("weight_t", torch.round(w / scale[:, None]).clamp_(-127, 127).to(torch.int8).contiguous().T)
        self.bias = lin.bias

    def forward(self, x):
        k, n = self.weight_t.shape
        if x.is_cuda and k % 16 == 0 and n % 8 == 0:
            from ..ops._ext import err_buf, ext
            rows = x.reshape(-1, k).to(torch.bfloat16).contiguous()
            q, a_scale = ext().quantize_rows_i8(rows)
            out = torch.empty(rows.shape[0], n, device=x.device, dtype=torch.bfloat16)
            ext().gemm_i8(q, self.weight_t.T, out, a_scale, self.scale, err_buf(x.device))
            if self.bias is not None:
                out = out + self.bias.to(out.dtype)
            return out.to(x.dtype).reshape(*x.shape[:-1], n)
        rows = x.reshape(-1, x.shape[-1]).float()
        a_scale = rows.abs().amax(1, keepdim=True).clamp_min(1e-12) / 127
        q = torch.round(rows / a_scale).clamp_(-127, 127).to(torch.int8)
        pad = max(24, -(-q.shape[0] // 8) * 8) - q.shape[0]  # the int8 GEMM wants > 16 rows, a multiple of 8
        if pad:
            q = torch.nn.functional.pad(q, (0, 0, 0, pad))
        acc = torch._int_mm(q, self.weight_t)[:rows.shape[0]]
        out = acc.float() * a_scale * self.scale
        if self.bias is not None:
            out = out + self.bias.float()
        return out.to(x.dtype).reshape(*x.shape[:-1], -1)


class BlockLinear(nn.Module):
    def __init__(self, lin: nn.Linear):
        super().__init__()
        w = B8.quantize_blocks(lin.weight.detach())
        self.register_buffer("w", w.codes)
        self.register_buffer("s", w.scales)
        self.bias = lin.bias
        self.in_features, self.out_features = lin.in_features, lin.out_features

    def _apply(self, fn, recurse=True):
        """Codes and scale bytes move, but are no numbers to convert (``module.to(torch.bfloat16)``)."""
        held = self.w, self.s
        super()._apply(fn, recurse)
        self.w, self.s = (new if new.dtype == old.dtype else old.to(new.device) for new, old in zip((self.w, self.s), held))
        return self

    def forward(self, x):
        if x.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("BlockLinear: a weight held in 8 bits passes no gradient on (use torch.no_grad() or detach x)")
        return self._forward(x)

    @torch.no_grad()
    def _forward(self, x):
        return B8.linear_blocks(x, B8.Blocks8(self.w, self.s, self.in_features), self.bias)


def use_fp8(module: nn.Module, on: bool = True) -> nn.Module:
    from .dit import DenoiserBlock
    from .routed import RoutedBlock
    from .text import TextBlock
    for block in module.modules():
        if isinstance(block, (DenoiserBlock, RoutedBlock, TextBlock)):
            for lin in block.modules():
                if isinstance(lin, nn.Linear):
                    lin.fp8 = on
    return module


def quantize(module: nn.Module, kind: str) -> nn.Module:
    from .moe import MoEMLP
    from .routed import RoutedMLP
    for name, child in list(module.named_children()):
        if isinstance(child, nn.Linear):
            if name == "router" and isinstance(module, (MoEMLP, RoutedMLP)):
                continue
            if kind == "fp8_block":
                setattr(module, name, BlockLinear(child))
            elif kind == "w8a8":
                if child.in_features % 8 == 0 and child.out_features % 8 == 0:
                    setattr(module, name, W8A8Linear(child))
            else:
                setattr(module, name, QLinear(child, kind))
        else:
            quantize(child, kind)
    return module
