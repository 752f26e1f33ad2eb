"""Packed-sequence operators where they are easily wrong, on the CPU."""
import pytest
import torch
from torch.autograd import forward_ad

from gpuschedule_amd.ops import clip_grad_norm_, grad_norm


def test_clip_refuses_tangents():
    p = torch.nn.Parameter(torch.zeros(3))
    with forward_ad.dual_level():
        p.grad = forward_ad.make_dual(torch.ones(3), torch.ones(3))
        for call in (grad_norm, lambda q: clip_grad_norm_(q, 0.1)):
            with pytest.raises(RuntimeError, match="tangent"):
                call([p])
        assert (p.grad == 1).all()
