"""Packed-sequence operators where they are easily wrong, on the CPU."""
import pytest
import torch
from torch.autograd import forward_ad

from gpuschedule_amd.ops import (clip_grad_norm_, flash_attention_packed,
                                 fused_rope_axes, grad_norm)


def test_clip_refuses_tangents():
    p = torch.nn.Parameter(torch.zeros(3))
    with forward_ad.dual_level():
        p.grad = forward_ad.make_dual(torch.ones(3), torch.ones(3))
        for call in (grad_norm, lambda q: clip_grad_norm_(q, 0.1)):
            with pytest.raises(RuntimeError, match="tangent"):
                call([p])
        assert (p.grad == 1).all()


def test_rope_refuses_tangents_of_tables():
    q, pos = torch.randn(3, 1, 8), torch.zeros(1, 3, dtype=torch.int64)
    c = torch.ones(2, 4)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(c, torch.ones(2, 4))
        for tables in ((d, c), (c, d)):
            with pytest.raises(RuntimeError, match="tangent"):
                fused_rope_axes(q, q, pos, *tables, [4])
        y, _ = fused_rope_axes(forward_ad.make_dual(q, q), q, pos, c, c, [4])
        assert forward_ad.unpack_dual(y).tangent is not None


def test_attention_rows_in_front():
    q, k, v = (torch.randn(9, n, 8, requires_grad=True) for n in (2, 1, 1))
    cu = torch.tensor([3, 7, 8], dtype=torch.int32)
    o = flash_attention_packed(q, k, v, cu, causal=True)
    grads = torch.autograd.grad(o.sum(), (q, k, v))
    part = flash_attention_packed(q[3:], k[3:], v[3:], cu - 3, causal=True)
    assert torch.equal(o[3:], part)
    for t in (o,) + grads:
        assert (t[:3] == 0).all() and (t[8:] == 0).all()


@pytest.mark.parametrize("T,B", [(0, 1), (1, 1), (5, 3), (300, 1), (300, 4),
                                 (1024, 7), (1000, 40)])
def test_attention_slots_cover_all_rows(T, B):
    """The blocks' search for their rows, on the host: every row is some
    slot's, once, for any rising bounds and none leaves [0, T] for others."""
    R, gen = 128, torch.Generator().manual_seed(T + B)

    def tiles(cu):
        def bound(i):
            return 0 if i == 0 else T if i > B + 1 else \
                min(max(cu[i - 1], 0), T)

        for slot in range(T // R + B + 2):
            lo, hi = 0, B + 1
            while lo < hi:
                mid = (lo + hi + 1) // 2
                if bound(mid) // R + mid <= slot:
                    lo = mid
                else:
                    hi = mid - 1
            begin = bound(lo)
            rows = max(bound(lo + 1) - begin, 0)
            row0 = (slot - (begin // R + lo)) * R
            if 0 <= row0 < rows:
                yield begin + row0, begin + min(row0 + R, rows)

    for _ in range(50):
        cu = torch.randint(0, T + 1, (B + 1,), generator=gen)
        seen = torch.zeros(T, dtype=torch.int32)
        for b, e in tiles(cu.sort().values.tolist()):
            seen[b:e] += 1
        assert (seen == 1).all()
        wild = torch.randint(-T - 9, 2 * T + 9, (B + 1,), generator=gen)
        for b, e in tiles(wild.tolist()):
            assert 0 <= b <= e <= T


def test_no_gradients_at_all():
    """0 as any other norm comes: fp32, on the parameters' device."""
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.float64)
    try:
        for device in ("cpu", "meta"):
            p = torch.nn.Parameter(torch.empty(3, device=device))
            for n in (grad_norm([p]), clip_grad_norm_(iter([p, p]), 1.0)):
                assert n.dtype == torch.float32 and n.device.type == device
                assert n.shape == ()
        assert grad_norm([]).dtype == torch.float32 and grad_norm([]) == 0
    finally:
        torch.set_default_dtype(before)
