"""Packed attention, rotary on axes, block norm and clipping on the CPU:
the plain paths against 64 bits, and what every path refuses."""
import math

import pytest
import torch

from gpuschedule_amd.ops import (FusedBlockNorm, clip_grad_norm_,
                                 flash_attention_packed, fused_block_norm,
                                 fused_rope_axes, grad_norm)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("causal,window", [(False, None), (True, None),
                                           (True, 3)])
def test_attention(causal, window):
    torch.manual_seed(0)
    T, H, HK, D = 20, 4, 2, 8
    q, k, v = (torch.randn(T, n, D, requires_grad=True)
               for n in (H, HK, HK))
    o = flash_attention_packed(q, k, v, i32(0, 5, 5, 17), i32(5, 0, 9),
                               causal, window)
    seq = torch.tensor([0] * 5 + [2] * 9 + [-1] * 6)
    i = torch.arange(T)
    seen = (seq[:, None] == seq) & (seq >= 0)
    if causal:
        seen &= i <= i[:, None]
    if window:
        seen &= i > i[:, None] - window
    kd, vd = (t.double().repeat_interleave(2, 1) for t in (k, v))
    s = torch.einsum("qhd,khd->hqk", q.double(), kd) / math.sqrt(D)
    s = s.masked_fill(~seen, -1e300)
    want = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1) * seen, vd)
    assert torch.allclose(o.double(), want, atol=1e-5)
    do = torch.randn(T, H, D)
    got = torch.autograd.grad(o, (q, k, v), do)
    ref = torch.autograd.grad(want, (q, k, v), do.double())
    for a, b in zip(got, ref):
        assert torch.allclose(a, b, atol=1e-5)
    assert (o[14:] == 0).all()


def test_attention_refuses():
    q = torch.zeros(6, 4, 16)
    k = torch.zeros(6, 2, 16)
    cu = i32(0, 6)
    for args, kw in (
            ((q, k, k[:5], cu), {}), ((q, k[:5], k[:5], cu), {}),
            ((q[0], k, k, cu), {}),
            ((q, torch.zeros(6, 3, 16), torch.zeros(6, 3, 16), cu), {}),
            ((q[:, :0], k, k, cu), {}),
            ((q[..., :12], k[..., :12], k[..., :12], cu), {}),
            ((torch.zeros(6, 4, 136),) * 3 + (cu,), {}),
            ((q, k, k, cu.long()), {}), ((q, k, k, cu[:1]), {}),
            ((q, k, k, cu), {"lengths": i32(1, 2)}),
            ((q, k, k, cu), {"lengths": torch.tensor([6])}),
            ((q, k, k, cu), {"window": 4}),
            ((q, k, k, cu), {"window": 0, "causal": True}),
            ((q, k, k, cu), {"scale": math.inf}),
            ((q, k, k, cu), {"scale": 0.0}),
            ((q, k, k, cu), {"scale": -0.1}),
            ((q, k, k, cu), {"scale": math.nan})):
        with pytest.raises(ValueError, match="flash_attention_packed"):
            flash_attention_packed(*args, **kw)


def test_rope_axes():
    torch.manual_seed(1)
    T, D, sections = 11, 20, [3, 5]
    q, k = torch.randn(T, 3, D), torch.randn(T, 1, D)
    ang = torch.outer(torch.arange(9.), 0.7 ** torch.arange(8.))
    pos = torch.randint(0, 9, (2, T))
    y, z = fused_rope_axes(q, k, pos, ang.cos(), ang.sin(), sections)
    for x, got in ((q, y), (k, z)):
        w = x.clone()
        for t in range(T):
            for j in range(8):
                a = ang[pos[0 if j < 3 else 1, t], j]
                w[t, :, j] = x[t, :, j] * a.cos() - x[t, :, j + 8] * a.sin()
                w[t, :, j + 8] = (x[t, :, j + 8] * a.cos()
                                  + x[t, :, j] * a.sin())
        assert torch.allclose(got, w, atol=1e-6)
    pos[1, 4] = 9
    y, _ = fused_rope_axes(q, k, pos, ang.cos(), ang.sin(), sections)
    assert y[4, :, 3:8].isnan().all() and not y[4, :, :3].isnan().any()


def test_rope_refuses():
    q, k = torch.zeros(5, 4, 16), torch.zeros(5, 2, 16)
    c = torch.zeros(7, 8)
    p = torch.zeros(1, 5, dtype=torch.int64)
    for args in ((q, k[:4], p, c, c, [8]), (q, k.half(), p, c, c, [8]),
                 (q, k[..., :8], p, c, c, [8]), (q, k, p[0], c, c, [8]),
                 (q, k, p.float(), c, c, [8]), (q, k, p, c, c, [4, 4]),
                 (q, k, p, c, c, [7]), (q, k, p, c, c, []),
                 (q, k, p.expand(2, 5), c, c, [8, 0]),
                 (q, k, p.expand(5, 5), c, c, [1, 1, 1, 1, 4]),
                 (q, k, p, c.double(), c.double(), [8]),
                 (q, k, p, c, c[:6], [8]),
                 (q, k, p, torch.zeros(7, 9), torch.zeros(7, 9), [9]),
                 (q.double(), k.double(), p, c, c, [8])):
        with pytest.raises(ValueError, match="fused_rope_axes"):
            fused_rope_axes(*args)


@pytest.mark.parametrize("gate", [None, (12,), (2, 12), (2, 3, 12)])
def test_block_norm(gate):
    torch.manual_seed(2)
    h, x = torch.randn(2, 3, 12), torch.randn(2, 3, 12)
    a, b = torch.rand(12) + 0.5, torch.rand(12) + 0.5
    g = None if gate is None else torch.randn(gate)
    n, s = fused_block_norm(h, x, a, b, g, 0.7)
    gd = 1.0 if g is None else g.double()
    if gate == (2, 12):
        gd = gd[:, None]

    def norm(t, w):
        t = t.double()
        return t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w

    want = 0.7 * x.double() + gd * norm(h, a)
    assert torch.allclose(s.double(), want, atol=1e-5)
    assert torch.allclose(n.double(), norm(want, b), atol=1e-5)


def test_block_norm_module():
    m = FusedBlockNorm(8, residual_scale=0.5, gated=True, gate_init=0.25)
    h, x = torch.randn(4, 8), torch.randn(4, 8)
    want = fused_block_norm(h, x, torch.ones(8), torch.ones(8),
                            torch.full((8,), 0.25), 0.5)
    assert all(torch.equal(a, b) for a, b in zip(m(h, x), want))
    assert sorted(dict(m.named_parameters())) == ["gate", "post_weight",
                                                  "pre_weight"]
    given = m(h, x, torch.zeros(8))[1]
    assert torch.equal(given, 0.5 * x)
    assert FusedBlockNorm(8).gate is None


def test_block_norm_refuses():
    h, w = torch.zeros(4, 6, 8), torch.ones(8)
    for args in ((h, h[:3], w, w), (h, h, w[:7], w), (h, h, w, w[None]),
                 (h, h, w.half(), w), (h, h, w, w, torch.ones(6, 8)),
                 (h, h, w, w, torch.ones(4, 1, 8)),
                 (h, h, w, w, torch.ones(8).half()),
                 (h.double(), h.double(), w.double(), w.double()),
                 (torch.zeros(()), torch.zeros(()), w, w),
                 (torch.zeros(1, 16385),) * 2 + (torch.ones(16385),) * 2):
        with pytest.raises(ValueError, match="fused_block_norm"):
            fused_block_norm(*args)


def test_clip():
    torch.manual_seed(3)
    ps = [torch.nn.Parameter(torch.zeros(s)) for s in ((3, 4), (5,), (2,))]
    for p in ps[:2]:
        p.grad = torch.randn_like(p)
    before = [p.grad.clone() for p in ps[:2]]
    total = torch.cat([g.flatten() for g in before]).norm()
    assert torch.allclose(grad_norm(ps), total)
    assert torch.allclose(clip_grad_norm_(ps + ps, 1.0), total)
    for p, g in zip(ps, before):
        assert torch.allclose(p.grad, g / total, rtol=1e-5)
    assert clip_grad_norm_(ps, 5.0) <= 1.0 and ps[2].grad is None
    assert grad_norm(ps[2]) == 0 and grad_norm([]) == 0
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_(ps, bad)
