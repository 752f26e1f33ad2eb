"""Fused LayerNorm / RMSNorm modules backed by the gfx950 kernels.

GPU path: hand-written HIP kernels (ops/hip/norms.hip) — bf16 in/out,
fp32 statistics, one fused pass each direction.  CPU path (tests): the
same math via plain fp32 torch ops under autograd.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from ._ext import get_ext


class _NormFn(torch.autograd.Function):
    """Fused norm with optional residual-add: y = norm(x + res).
    Returns (y, summed): ``summed`` is x+res (the residual stream) when
    a residual is given, else x."""

    @staticmethod
    def forward(ctx, x, res, weight, bias, eps, rms):
        ext = get_ext(required=True)
        ctx.set_materialize_grads(False)
        x = x.contiguous()
        y, summed, mean, rstd = ext.norm_fwd(x, res, weight, bias, eps,
                                             rms)
        has_res = res is not None
        ctx.save_for_backward(summed, weight, mean, rstd)
        ctx.rms = rms
        ctx.has_res = has_res
        # second output: the residual stream (x+res); dummy when no res
        return y, (summed if has_res else x.new_empty(0))

    @staticmethod
    def backward(ctx, dy, dsum):
        ext = get_ext(required=True)
        summed, weight, mean, rstd = ctx.saved_tensors
        if dy is None:
            dy = torch.zeros_like(summed)
        # downstream residual-stream grad (dsum) is added into dx
        # INSIDE the bwd kernel — no separate elementwise add pass
        dx, dw, db = ext.norm_bwd(dy.contiguous(), summed,
                                  None if ctx.rms else mean, rstd,
                                  weight, ctx.rms,
                                  dsum.contiguous()
                                  if dsum is not None else None)
        dres = dx if ctx.has_res else None
        return dx, dres, dw, (None if ctx.rms else db), None, None


def _cpu_layernorm(x, w, b, eps):
    xf = x.float()
    y = torch.nn.functional.layer_norm(xf, (x.shape[-1],), w.float(),
                                       b.float(), eps)
    return y.to(x.dtype)


def _cpu_rmsnorm(x, w, eps):
    xf = x.float()
    y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return (y * w.float()).to(x.dtype)


class FusedLayerNorm(nn.Module):
    def __init__(self, dim: int, eps: float = 1e-5):
        super().__init__()
        self.dim, self.eps = dim, eps
        self.weight = nn.Parameter(torch.ones(dim))
        self.bias = nn.Parameter(torch.zeros(dim))

    def forward(self, x, residual=None, return_sum=False):
        if x.is_cuda:
            y, summed = _NormFn.apply(
                x, residual.contiguous() if residual is not None
                else None, self.weight, self.bias, self.eps, False)
            return (y, summed) if return_sum else y
        y = _cpu_layernorm(x + residual if residual is not None else x,
                           self.weight, self.bias, self.eps)
        if return_sum:
            return y, (x + residual if residual is not None else x)
        return y

    def extra_repr(self):
        return f"{self.dim}, eps={self.eps}"


class FusedRMSNorm(nn.Module):
    def __init__(self, dim: int, eps: float = 1e-6):
        super().__init__()
        self.dim, self.eps = dim, eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x, residual=None, return_sum=False):
        if x.is_cuda:
            y, summed = _NormFn.apply(
                x, residual.contiguous() if residual is not None
                else None, self.weight, None, self.eps, True)
            return (y, summed) if return_sum else y
        xs = x + residual if residual is not None else x
        y = _cpu_rmsnorm(xs, self.weight, self.eps)
        return (y, xs) if return_sum else y

    def extra_repr(self):
        return f"{self.dim}, eps={self.eps}"


def fused_block_norm(h: torch.Tensor, x: torch.Tensor,
                     post_weight: torch.Tensor, pre_weight: torch.Tensor,
                     gate: Optional[torch.Tensor] = None,
                     residual_scale: float = 1.0, eps: float = 1e-6):
    """What stands between two residual blocks, in one pass each way:

        s = residual_scale * x + gate * rmsnorm(h) * post_weight
        n = rmsnorm(s) * pre_weight

    ``h`` [..., D] is a block's output, ``x`` [..., D] the residual
    stream before it.  Returns ``(n, s)``: the next block's input and
    the stream behind the sum (``FusedRMSNorm``'s ``return_sum`` order).

    ``gate``: ``[D]`` for all rows, ``[h.shape[0], D]`` for one gate row
    for each index of h's first dimension (a sequence of a batch), or
    h's own shape; None is 1.  All tensors share one type (bf16, fp16 or
    fp32) and device; D is at most 16384.  Statistics and sums are fp32,
    ``n`` is computed from the sum before that is rounded.  Inputs that
    are not contiguous are copied."""
    D = h.shape[-1] if h.dim() else 0
    if x.shape != h.shape:
        raise ValueError(f"fused_block_norm: x is {tuple(x.shape)}, "
                         f"h is {tuple(h.shape)}")
    for name, w in (("post_weight", post_weight),
                    ("pre_weight", pre_weight)):
        if w.shape != (D,):
            raise ValueError(f"fused_block_norm: {name} must be [{D}], "
                             f"got {tuple(w.shape)}")
    for t in (x, post_weight, pre_weight, gate):
        if t is not None and (t.dtype != h.dtype or t.device != h.device):
            raise ValueError("fused_block_norm: all tensors must have h's "
                             "type and device")
    if not 1 <= D <= 16384:
        raise ValueError(f"fused_block_norm: D must be 1 to 16384, got {D}")
    if h.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"fused_block_norm: bf16, fp16 or fp32 only, "
                         f"got {h.dtype}")
    if gate is not None and gate.shape != (D,) and gate.shape != h.shape \
            and (h.dim() < 2 or gate.shape != (h.shape[0], D)):
        raise ValueError(f"fused_block_norm: gate {tuple(gate.shape)} is "
                         f"none of [D], [h.shape[0], D] and h's shape")
    if not h.is_cuda:
        g = 1.0
        if gate is not None:
            g = gate.float()
            if gate.shape != h.shape and gate.dim() == 2:
                g = g.view(h.shape[0], *[1] * (h.dim() - 2), D)
        hf, xf = h.float(), x.float()
        z = hf * torch.rsqrt(hf.pow(2).mean(-1, keepdim=True) + eps)
        s = residual_scale * xf + g * (z * post_weight.float())
        n = s * torch.rsqrt(s.pow(2).mean(-1, keepdim=True) + eps)
        return (n * pre_weight.float()).to(h.dtype), s.to(h.dtype)
    return tuple(get_ext(required=True).block_norm(
        h, x, post_weight, pre_weight, gate, residual_scale, eps))


class FusedBlockNorm(nn.Module):
    """:func:`fused_block_norm` with its weights.  ``gated=True`` adds a
    learned gate [D] that begins at ``gate_init``; a gate given to
    ``forward`` takes its place."""

    def __init__(self, dim: int, residual_scale: float = 1.0,
                 gated: bool = False, gate_init: float = 1.0,
                 eps: float = 1e-6):
        super().__init__()
        self.dim, self.eps = dim, eps
        self.residual_scale = residual_scale
        self.post_weight = nn.Parameter(torch.ones(dim))
        self.pre_weight = nn.Parameter(torch.ones(dim))
        self.gate = (nn.Parameter(torch.full((dim,), float(gate_init)))
                     if gated else None)

    def forward(self, h, x, gate=None):
        return fused_block_norm(h, x, self.post_weight, self.pre_weight,
                                self.gate if gate is None else gate,
                                self.residual_scale, self.eps)

    def extra_repr(self):
        return (f"{self.dim}, residual_scale={self.residual_scale}, "
                f"gated={self.gate is not None}, eps={self.eps}")
