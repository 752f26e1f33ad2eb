"""Global gradient norm and clipping over many tensors (ops/hip/clip.hip).

``clip_grad_norm_(parameters, max_norm)`` stands between ``backward()``
(and a gang's ``GradReducer.finalize()``) and the fused optimizers'
``step()``.  It never waits for the GPU: the norm comes back as a device
scalar, and a captured step replays it.  CPU path: plain torch (tests).
"""
from __future__ import annotations

from typing import Iterable, List, Union

import torch
from torch.autograd import forward_ad

from ._ext import get_ext


def _with_grad(parameters):
    """The parameters as a list, and the first gradient among them."""
    params = ([parameters] if isinstance(parameters, torch.Tensor)
              else list(parameters))
    for p in params:
        if p.grad is not None:
            return params, p.grad
    return params, None


def _nothing(params) -> torch.Tensor:
    return torch.zeros((), dtype=torch.float32,
                       device=params[0].device if params else "cpu")


def _cpu_grads(params) -> List[torch.Tensor]:
    # a tied weight counts once
    grads = [p.grad for p in dict.fromkeys(params) if p.grad is not None]
    if any(g.device.type != "cpu" for g in grads):
        raise RuntimeError("grad_norm: all gradients must be on one device")
    if any(forward_ad.unpack_dual(g).tangent is not None for g in grads):
        raise RuntimeError("grad_norm: gradients with a forward-mode "
                           "tangent are not supported")
    return grads


def _cpu_norm(grads) -> torch.Tensor:
    return sum(g.detach().double().square().sum() for g in grads).sqrt()


def grad_norm(parameters: Union[torch.Tensor, Iterable[torch.Tensor]]
              ) -> torch.Tensor:
    """The 2-norm of all gradients of ``parameters`` taken together, as
    an fp32 scalar tensor on their device (0, on the parameters' device,
    if there are none).

    Gradients may mix bf16, fp16 and fp32.  They must be on one device,
    dense in memory (any order of dimensions), and must not share
    memory; a parameter that is named twice counts once.  Squares are
    summed in 64 bits."""
    params, any_grad = _with_grad(parameters)
    if any_grad is None:
        return _nothing(params)
    if any_grad.is_cuda:
        return get_ext(required=True).grad_norm_clip(params, -1.0)
    return _cpu_norm(_cpu_grads(params)).float()


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
    if not max_norm >= 0:
        raise ValueError(f"clip_grad_norm_: max_norm must be >= 0, "
                         f"got {max_norm}")
    params, any_grad = _with_grad(parameters)
    if any_grad is None:
        return _nothing(params)
    if any_grad.is_cuda:
        return get_ext(required=True).grad_norm_clip(params, max_norm)
    grads = _cpu_grads(params)
    norm = _cpu_norm(grads)
    ratio = max_norm / (norm + 1e-6)
    if not ratio >= 1.0:
        for g in grads:
            g.copy_(g.double() * ratio)
    return norm.float()
