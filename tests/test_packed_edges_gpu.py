"""Packed-sequence operators where they are easily wrong: tangents, the range
of 16 bits, narrow windows, rows in front of the first sequence."""
import math

import pytest
import torch
from torch.autograd import forward_ad

from gpuschedule_amd.ops import (clip_grad_norm_, flash_attention_packed,
                                 fused_block_norm, fused_rope_axes,
                                 grad_norm)

pytestmark = pytest.mark.gpu

BF, FH, FP = torch.bfloat16, torch.float16, torch.float32


def normal(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def cu_of(*bounds):
    return torch.tensor(bounds, dtype=torch.int32, device="cuda")


# ---- forward mode ----------------------------------------------------------

def calls_of(q, w):
    cos, sin = torch.ones(2, 4, device="cuda"), torch.zeros(2, 4,
                                                            device="cuda")
    pos = torch.zeros(1, q.shape[0], dtype=torch.int64, device="cuda")
    plain = q.detach()
    return [
        lambda: flash_attention_packed(q, plain, plain, cu_of(0, 6)),
        lambda: flash_attention_packed(plain, q, plain, cu_of(0, 6)),
        lambda: flash_attention_packed(plain, plain, q, cu_of(0, 6)),
        lambda: fused_rope_axes(q, plain, pos, cos, sin, [4]),
        lambda: fused_rope_axes(plain, q, pos, cos, sin, [4]),
        lambda: fused_block_norm(q, plain, w.detach(), w.detach()),
        lambda: fused_block_norm(plain, q, w.detach(), w.detach()),
        lambda: fused_block_norm(plain, plain, w, w.detach()),
        lambda: fused_block_norm(plain, plain, w.detach(), w),
        lambda: fused_block_norm(plain, plain, w.detach(), w.detach(), w),
    ]


@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(grad):
    """A derivative in forward mode is refused, never dropped."""
    x, w = normal((6, 2, 8), BF, 0), normal((8,), BF, 1)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dual = [forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, w)]
        for i, call in enumerate(calls_of(*dual)):
            with pytest.raises((RuntimeError, NotImplementedError),
                               match="jvp"):
                call()
                pytest.fail(f"call {i} dropped its tangent")
        p = torch.nn.Parameter(torch.zeros(6, 2, 8, device="cuda", dtype=BF))
        p.grad = dual[0]
        for call in (grad_norm, lambda q: clip_grad_norm_(q, 0.1)):
            with pytest.raises(RuntimeError, match="tangent"):
                call([p])
        # without tangents the same calls run inside of a dual level
        for call in calls_of(x, w):
            call()
