"""Fused RoPE and SwiGLU-gate wrappers (ops/hip/elementwise.hip)."""
from __future__ import annotations

from typing import Sequence

import torch
from torch.autograd import forward_ad

from ._ext import get_ext


class _RopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, cosb, sinb):
        ext = get_ext(required=True)
        ctx.save_for_backward(cosb, sinb)
        return ext.rope_apply(x, cosb, sinb, False)

    @staticmethod
    def backward(ctx, dy):
        ext = get_ext(required=True)
        cosb, sinb = ctx.saved_tensors
        return ext.rope_apply(dy.contiguous(), cosb, sinb, True), \
            None, None


def fused_rope(x: torch.Tensor, cosb: torch.Tensor,
               sinb: torch.Tensor) -> torch.Tensor:
    """Rotate-half RoPE on [B, H, S, D] bf16 with fp32 [S, D/2] tables."""
    if x.is_cuda and x.dtype == torch.bfloat16:
        return _RopeFn.apply(x, cosb, sinb)
    S = x.shape[-2]
    c = cosb[:S].to(x.dtype)[None, None]
    s = sinb[:S].to(x.dtype)[None, None]
    x1, x2 = x.chunk(2, dim=-1)
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1)


def fused_rope_axes(q: torch.Tensor, k: torch.Tensor,
                    positions: torch.Tensor, cosb: torch.Tensor,
                    sinb: torch.Tensor, sections: Sequence[int]):
    """Rotate-half RoPE by token positions on one or several axes.

    ``q`` [T, H, D], ``k`` [T, HK, D]: packed tokens (slices of a fused
    projection are read in place).  ``positions`` [axes, T], int32 or
    int64: each token's position on each axis, e.g. time, height and
    width; the positions of packed sequences restart at will.  ``cosb``,
    ``sinb`` [P, R/2] fp32: row p holds the angles of position p.
    ``sections``: how many of the R/2 frequencies, in order, go by each
    axis (``[R/2]`` for one axis).  Values from R on (R <= D) pass
    through.  1 to 4 axes; q and k both bf16, fp16 or fp32.

    Returns new contiguous ``(q, k)``.  A position outside of the tables
    makes that token's values on that axis NaN.  The tables get no
    gradient, and may carry no forward-mode tangent."""
    sections = [int(n) for n in sections]
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] \
            or q.shape[2] != k.shape[2]:
        raise ValueError(f"fused_rope_axes: q [T, H, D] and k [T, HK, D] "
                         f"wanted, got {tuple(q.shape)}, {tuple(k.shape)}")
    if q.dtype != k.dtype or q.dtype not in (torch.bfloat16, torch.float16,
                                             torch.float32):
        raise ValueError(f"fused_rope_axes: q and k must both be bf16, fp16 "
                         f"or fp32, got {q.dtype}, {k.dtype}")
    if cosb.dim() != 2 or cosb.shape != sinb.shape \
            or cosb.dtype != torch.float32 or sinb.dtype != torch.float32:
        raise ValueError("fused_rope_axes: cosb and sinb must be fp32 "
                         "[places, R/2]")
    half = cosb.shape[1]
    if not 1 <= len(sections) <= 4 or min(sections) < 1 \
            or sum(sections) != half or 2 * half > q.shape[2]:
        raise ValueError(f"fused_rope_axes: sections {sections} must be 1 to "
                         f"4 positive counts that add up to {half}, at most "
                         f"half of D = {q.shape[2]}")
    if positions.shape != (len(sections), q.shape[0]) \
            or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"fused_rope_axes: positions must be int32 or int64 "
                         f"[{len(sections)}, {q.shape[0]}], got "
                         f"{positions.dtype} {tuple(positions.shape)}")
    for t in (k, positions, cosb, sinb):
        if t.device != q.device:
            raise ValueError("fused_rope_axes: all tensors must be on one "
                             "device")
    if q.is_cuda:
        return tuple(get_ext(required=True).rope_axes(
            q, k, positions, cosb, sinb, sections))
    if any(forward_ad.unpack_dual(t).tangent is not None
           for t in (cosb, sinb)):
        raise RuntimeError("fused_rope_axes: tables with a forward-mode "
                           "tangent are not supported")
    cosb, sinb = cosb.detach(), sinb.detach()
    axis = torch.repeat_interleave(torch.arange(len(sections)),
                                   torch.tensor(sections))
    at = positions[axis].t().long()                        # [T, R/2]
    ok = (at >= 0) & (at < cosb.shape[0])
    nan = torch.full((), float("nan"))
    if cosb.shape[0]:
        at = at.clamp(0, cosb.shape[0] - 1)
        place = torch.arange(half)
        c, s = (torch.where(ok, b[at, place], nan)[:, None]
                for b in (cosb, sinb))
    else:
        c = s = nan.expand(q.shape[0], 1, half)

    def turn(x):
        a, b = x[..., :half].float(), x[..., half:2 * half].float()
        return torch.cat([(a * c - b * s).to(x.dtype),
                          (b * c + a * s).to(x.dtype),
                          x[..., 2 * half:]], dim=-1)

    return turn(q), turn(k)


class _SiluMulFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, g, u):
        ext = get_ext(required=True)
        ctx.save_for_backward(g, u)
        return ext.silu_mul_fwd(g, u)

    @staticmethod
    def backward(ctx, dy):
        ext = get_ext(required=True)
        g, u = ctx.saved_tensors
        dg, du = ext.silu_mul_bwd(dy.contiguous(), g, u)
        return dg, du


def silu_mul(g: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    if g.is_cuda and g.dtype == torch.bfloat16:
        return _SiluMulFn.apply(g.contiguous(), u.contiguous())
    return torch.nn.functional.silu(g) * u


class _GeluFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        ext = get_ext(required=True)
        ctx.save_for_backward(x)
        return ext.gelu_fwd(x)

    @staticmethod
    def backward(ctx, dy):
        ext = get_ext(required=True)
        (x,) = ctx.saved_tensors
        return ext.gelu_bwd(dy.contiguous(), x)


def fused_gelu(x: torch.Tensor) -> torch.Tensor:
    """tanh-approximate GELU: one fused bf16 pass each way on GPU
    (torch's Gelu + GeluBackward elementwise pair otherwise); fp32
    torch reference on CPU."""
    if x.is_cuda and x.dtype == torch.bfloat16:
        return _GeluFn.apply(x.contiguous())
    return torch.nn.functional.gelu(x, approximate="tanh")


class _SwigluPackedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gu):
        ext = get_ext(required=True)
        ctx.save_for_backward(gu)
        return ext.swiglu_fwd(gu)

    @staticmethod
    def backward(ctx, dy):
        ext = get_ext(required=True)
        (gu,) = ctx.saved_tensors
        return ext.swiglu_bwd(dy.contiguous(), gu)


def swiglu_packed(gu: torch.Tensor) -> torch.Tensor:
    """SwiGLU on the PACKED [.., 2F] gate_up projection: the kernels
    read both halves through the row stride and the backward writes one
    packed grad buffer — no contiguous() copies of the halves and no
    chunk-backward cat.  CPU: fp32 torch reference."""
    if gu.is_cuda and gu.dtype == torch.bfloat16:
        return _SwigluPackedFn.apply(gu.contiguous())
    g, u = gu.chunk(2, dim=-1)
    return torch.nn.functional.silu(g) * u
