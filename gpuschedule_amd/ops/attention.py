"""Attention dispatch: hand-written flash kernels on GPU.

``flash_attention(q, k, v, causal)`` takes [B, H, S, D] bf16 tensors
(k/v may have fewer heads: GQA).  ``flash_attention_qkv(qkv, causal)``
takes the packed [B, S, 3, H, D] view of a fused self-attention
projection and runs the zero-copy strided path.  GPU forward runs the
gfx950 flash kernel (ops/hip/attention.hip, online-softmax MFMA);
backward runs the FA2-style two-kernel HIP backward (dK/dV then dQ —
no S x S activation is ever materialized).  CPU path: fp32 reference
composite (tests).
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from ._ext import get_ext


def _ref_attention(q, k, v, causal: bool):
    # fp32 reference composite; used on CPU and as the numerics oracle.
    scale = 1.0 / math.sqrt(q.shape[-1])
    s = torch.matmul(q.float(), k.float().transpose(-1, -2)) * scale
    if causal:
        S = q.shape[-2]
        mask = torch.ones(S, S, dtype=torch.bool, device=q.device).triu(1)
        s = s.masked_fill(mask, float("-inf"))
    p = torch.softmax(s, dim=-1)
    return torch.matmul(p, v.float()).to(q.dtype)


class _FlashAttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal):
        ext = get_ext(required=True)
        o, lse = ext.attn_fwd(q, k, v, causal)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.causal = causal
        return o

    @staticmethod
    def backward(ctx, do):
        # hand-written FA2-style backward (ops/hip/attention.hip):
        # no S x S activation ever materialized.
        ext = get_ext(required=True)
        q, k, v, o, lse = ctx.saved_tensors
        dq, dk, dv = ext.attn_bwd(q, k, v, o, do.contiguous(), lse,
                                  ctx.causal)
        return dq, dk, dv, None


class _FlashAttnQKVFn(torch.autograd.Function):
    """Packed-QKV self-attention: takes the [B,S,3,H,D] view of one
    fused projection.  The kernels read the q/k/v slices through their
    strides and write the three grads into ONE [B,S,3,H,D] buffer, so
    the whole attention block adds ZERO layout copies (no per-slice
    contiguous(), no select-backward zero+copy, no output re-pack)."""

    @staticmethod
    def forward(ctx, qkv, causal):
        ext = get_ext(required=True)
        q = qkv[:, :, 0].transpose(1, 2)  # [B,H,S,D] strided views
        k = qkv[:, :, 1].transpose(1, 2)
        v = qkv[:, :, 2].transpose(1, 2)
        o, lse = ext.attn_fwd(q, k, v, causal)
        ctx.save_for_backward(qkv, o, lse)
        ctx.causal = causal
        return o

    @staticmethod
    def backward(ctx, do):
        ext = get_ext(required=True)
        qkv, o, lse = ctx.saved_tensors
        q = qkv[:, :, 0].transpose(1, 2)
        k = qkv[:, :, 1].transpose(1, 2)
        v = qkv[:, :, 2].transpose(1, 2)
        if do.stride() != o.stride():  # usually a free view already
            do = do.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        out = ext.attn_bwd(q, k, v, o, do, lse, ctx.causal)
        return out[3], None  # the packed [B,S,3,H,D] grad


def flash_attention_qkv(qkv: torch.Tensor,
                        causal: bool = False) -> torch.Tensor:
    """qkv: [B, S, 3, H, D] (contiguous, e.g. a fused-projection view).
    Returns O as logical [B, H, S, D]; ``o.transpose(1, 2)`` is a free
    view for the head-merge reshape."""
    if qkv.is_cuda:
        return _FlashAttnQKVFn.apply(qkv.contiguous(), causal)
    q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    return _ref_attention(q, k, v, causal)


def flash_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    causal: bool = False) -> torch.Tensor:
    """q,k,v: [B, H, S, D] bf16 (k/v may have fewer heads: GQA)."""
    if q.is_cuda:
        ext = get_ext(required=True)
        if hasattr(ext, "attn_fwd"):
            # GQA is kernel-native: k/v keep their (fewer) heads; the
            # kernels read kv head h/(H/HK) directly and the backward
            # group-accumulates dK/dV over each head's query group.
            return _FlashAttnFn.apply(q.contiguous(), k.contiguous(),
                                      v.contiguous(), causal)
        raise RuntimeError("attn_fwd missing from HIP extension")
    if k.shape[1] != q.shape[1]:
        rep = q.shape[1] // k.shape[1]
        k = k.repeat_interleave(rep, dim=1)
        v = v.repeat_interleave(rep, dim=1)
    return _ref_attention(q, k, v, causal)


def _ref_attention_packed(q, k, v, cu_seqlens, lengths, causal, window,
                          scale):
    # fp32 composite; used on CPU
    T, H, D = q.shape
    rep = H // k.shape[1]
    o = torch.zeros(T, H, D, dtype=torch.float32, device=q.device)
    cu = [min(max(int(c), 0), T) for c in cu_seqlens.tolist()]
    lens = (lengths.tolist() if lengths is not None
            else [T] * (len(cu) - 1))
    parts, at = [], 0
    for b, e, n in zip(cu[:-1], cu[1:], lens):
        n = min(max(int(n), 0), max(e - b, 0))
        if n == 0:
            continue
        qs, ks, vs = (x[b:b + n].float().transpose(0, 1) for x in (q, k, v))
        ks, vs = (x.repeat_interleave(rep, dim=0) for x in (ks, vs))
        s = torch.matmul(qs, ks.transpose(-1, -2)) * scale
        far = torch.arange(n)[:, None] - torch.arange(n)
        if causal:
            s = s.masked_fill(far < 0, float("-inf"))
        if window:
            s = s.masked_fill(far >= window, float("-inf"))
        out = torch.matmul(torch.softmax(s, dim=-1), vs).transpose(0, 1)
        parts += [o[at:b], out]
        at = b + n
    return torch.cat(parts + [o[at:]]).to(q.dtype)


def flash_attention_packed(q: torch.Tensor, k: torch.Tensor,
                           v: torch.Tensor, cu_seqlens: torch.Tensor,
                           lengths: Optional[torch.Tensor] = None,
                           causal: bool = False,
                           window: Optional[int] = None,
                           scale: Optional[float] = None) -> torch.Tensor:
    """Self-attention within each of several packed sequences.

    ``q`` [T, H, D], ``k``, ``v`` [T, HK, D] (HK divides H), bf16 or
    fp16, D a multiple of 8 up to 128; slices of a fused projection are
    read in place.  ``cu_seqlens`` int32 [sequences + 1], on q's device:
    sequence i is rows ``cu_seqlens[i]`` to ``cu_seqlens[i + 1]``; it
    does not fall, and rows in front of its first value (0, if all are
    used) or behind its last belong to no sequence.  ``lengths`` int32 [sequences]: only the
    first ``lengths[i]`` rows of sequence i are tokens, the rest is
    padding (a padded batch [B, S] is ``cu_seqlens = [0, S, 2S, ...]``).

    ``causal``: a row sees its own and earlier rows; ``window`` (causal
    only): of those the last ``window``, its own among them.  ``scale``
    (positive) defaults to 1/sqrt(D).

    Returns o [T, H, D], contiguous.  Rows that are no tokens get zeros,
    in o and in the gradients, whatever they hold.  An infinity or NaN
    stays in its own sequence.  Where cu_seqlens falls or leaves [0, T]
    the result is undefined, but nothing outside the tensors is
    touched.  Nothing here waits for the GPU; a call can be captured.
    (T / 128 + sequences) * H has to stay under 2^24."""
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape \
            or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError(f"flash_attention_packed: q [T, H, D], k and v "
                         f"[T, HK, D] wanted, got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    T, H, D = q.shape
    if k.shape[1] < 1 or H < 1 or H % k.shape[1]:
        raise ValueError(f"flash_attention_packed: {k.shape[1]} kv heads do "
                         f"not divide {H} heads")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"flash_attention_packed: D must be a multiple of "
                         f"8, at most 128, got {D}")
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 \
            or cu_seqlens.dtype != torch.int32:
        raise ValueError("flash_attention_packed: cu_seqlens must be int32 "
                         "[sequences + 1]")
    if lengths is not None and (lengths.dtype != torch.int32 or
                                lengths.shape != (cu_seqlens.numel() - 1,)):
        raise ValueError("flash_attention_packed: lengths must be int32 "
                         "[sequences]")
    for t in (k, v, cu_seqlens, lengths):
        if t is not None and t.device != q.device:
            raise ValueError("flash_attention_packed: all tensors must be "
                             "on one device")
    if window is not None and (not causal or window < 1):
        raise ValueError("flash_attention_packed: window must be at least "
                         "1, and needs causal")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 1e-30 < scale < 1e30:
        raise ValueError(f"flash_attention_packed: scale must be positive, "
                         f"got {scale}")
    if q.is_cuda:
        if q.dtype not in (torch.bfloat16, torch.float16) \
                or k.dtype != q.dtype or v.dtype != q.dtype:
            raise ValueError(f"flash_attention_packed: q, k and v must all "
                             f"be bf16 or fp16, got {q.dtype}, {k.dtype}, "
                             f"{v.dtype}")
        return get_ext(required=True).attn_packed(
            q, k, v, cu_seqlens, lengths, causal, window or 0, scale)
    return _ref_attention_packed(q, k, v, cu_seqlens, lengths, causal,
                                 window, scale)
