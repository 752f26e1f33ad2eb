"""Global gradient norm and clipping over many tensors (ops/hip/clip.hip).

``clip_grad_norm_(parameters, max_norm)`` stands between ``backward()``
(and a gang's ``GradReducer.finalize()``) and the fused optimizers'
``step()``.  It never waits for the GPU: the norm comes back as a device
scalar, and a captured step replays it.  CPU path: plain torch (tests).
"""
from __future__ import annotations

import math
from typing import Iterable, List, Union

import torch

from ._ext import get_ext


def _grads_of(parameters) -> List[torch.Tensor]:
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    seen, grads = set(), []
    for p in parameters:
        if p.grad is None or id(p) in seen:  # a tied weight counts once
            continue
        seen.add(id(p))
        grads.append(p.grad.detach())
    return grads


def _cpu_norm(grads) -> torch.Tensor:
    total = sum(g.double().square().sum() for g in grads)
    return torch.as_tensor(total).sqrt()


def grad_norm(parameters: Union[torch.Tensor, Iterable[torch.Tensor]]
              ) -> torch.Tensor:
    """The 2-norm of all gradients of ``parameters`` taken together, as
    an fp32 scalar tensor on their device (0 if there are none).

    Gradients may mix bf16, fp16 and fp32.  They must be on one device,
    dense in memory (any order of dimensions), and must not share
    memory.  Squares are summed in 64 bits."""
    grads = _grads_of(parameters)
    if not grads:
        return torch.zeros(())
    if grads[0].is_cuda:
        return get_ext(required=True).grad_norm_clip(grads, -1.0)
    return _cpu_norm(grads).float()


@torch.no_grad()
def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]],
                    max_norm: float) -> torch.Tensor:
    """Scales the gradients of ``parameters`` in place by
    ``min(1, max_norm / (norm + 1e-6))`` and returns their norm before
    that, as :func:`grad_norm` does (same requirements).

    Where the norm is infinite or NaN no scale is right: finite
    gradients become 0 or NaN.  Check the returned norm to skip such a
    step."""
    max_norm = float(max_norm)
    if math.isnan(max_norm) or max_norm < 0:
        raise ValueError(f"clip_grad_norm_: max_norm must be >= 0, "
                         f"got {max_norm}")
    grads = _grads_of(parameters)
    if not grads:
        return torch.zeros(())
    if grads[0].is_cuda:
        norm = get_ext(required=True).grad_norm_clip(grads, max_norm)
        torch.autograd.graph.increment_version(grads)
        return norm
    norm = _cpu_norm(grads)
    ratio = max_norm / (norm + 1e-6)
    if not ratio >= 1.0:
        for g in grads:
            g.copy_(g.double() * ratio)
    return norm.float()
