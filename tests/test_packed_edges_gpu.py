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
        cos = torch.ones(2, 4, device="cuda")
        pos = torch.zeros(1, 6, dtype=torch.int64, device="cuda")
        table = forward_ad.make_dual(cos, torch.ones_like(cos))
        for tables in ((table, cos), (cos, table)):
            with pytest.raises(RuntimeError, match="tangent"):
                fused_rope_axes(x, x, pos, *tables, [4])
        # without tangents the same calls run inside of a dual level
        for call in calls_of(x, w):
            call()


# ---- the range of 16 bits --------------------------------------------------

def leaf(t):
    return t.detach().requires_grad_()


def spread(q, k, v, do, causal, scale, window=None, exact_d=False):
    """64-bit o, dq, dk, dv of one sequence, and how far each is off as a
    whole, as the root of a sum of squares: every rounding to the type's
    relative half step u is off by u / sqrt(3) at most in the mean, and
    roundings of different values are independent.  What is rounded: p and
    dS on their way into a product, o (which D = dO.o takes up, unless it is
    exact) and the results; nothing but a result may fall under the type's
    range."""
    u = torch.finfo(q.dtype).eps / 2
    step = torch.finfo(q.dtype).smallest_normal * 2 * u
    rep = q.shape[1] // k.shape[1]
    q, k, v, do = (t.detach().double().transpose(0, 1)
                   for t in (q, k, v, do))
    kr, vr = (t.repeat_interleave(rep, 0) for t in (k, v))
    s = (q @ kr.mT) * scale
    if causal:
        n = torch.arange(s.shape[-1], device=s.device)
        far = n[:, None] - n
        s = s.masked_fill((far < 0) | (far >= (window or len(n))), -math.inf)
    p = s.softmax(-1)
    o = p @ vr
    off_o = p.square() @ vr.square() + o.square()
    off_d = (do.square() * off_o).sum(-1, keepdim=True) * (not exact_d)
    ds = p * (do @ vr.mT - (do * o).sum(-1, keepdim=True))
    dq, dk, dv = scale * (ds @ kr), scale * (ds.mT @ q), p.mT @ do
    off_q = scale ** 2 * (ds.square() @ kr.square()
                          + off_d * (p @ kr).square()) + dq.square()
    off_k = scale ** 2 * (ds.square().mT @ q.square()
                          + p.square().mT @ (off_d * q.square()))
    off_v = p.square().mT @ do.square()

    def group(t):
        return t.unflatten(0, (-1, rep)).sum(1)

    dk, dv = group(dk), group(dv)
    off_k, off_v = group(off_k) + dk.square(), group(off_v) + dv.square()
    return [(w.transpose(0, 1),
             ((u * u * off.sum() + (step / 2) ** 2 * w.numel()) / 3).sqrt())
            for w, off in ((o, off_o), (dq, off_q), (dk, off_k),
                           (dv, off_v))]


@pytest.mark.parametrize("dtype", [FH, BF])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-4])
def test_attention_small_gradients(size, D, causal, dtype):
    """Gradients of dO far below 1 keep the precision of their type.  Twice
    the mean error is allowed: of so many values it hardly strays."""
    T, H = 2048, 2
    q, k, v = (leaf(normal((T, n, D), dtype, i))
               for i, n in enumerate((H, 1, 1)))
    do = normal((T, H, D), dtype, 3, size)
    o = flash_attention_packed(q, k, v, cu_of(0, T), causal=causal)
    got = (o,) + torch.autograd.grad(o, (q, k, v), do)
    for g, (w, off), name in zip(got, spread(q, k, v, do, causal, D ** -0.5),
                                 ("o", "dq", "dk", "dv")):
        err = (g.double() - w).norm()
        assert err <= 2 * off, f"{name}: {err / off:.3g} of the mean error"


def test_attention_large_gradients():
    """dS over the largest fp16 number, while no result is."""
    n, T = 3, 300
    q, k, v, do = (normal((T, 1, 64), FH, i, size) for i, size in
                   enumerate((1e-3, 1e-3, 100.0, 3000.0)))
    q, k, v = leaf(q), leaf(k), leaf(v)
    o = flash_attention_packed(q, k, v, cu_of(*range(0, T + 1, n)))
    got = (o,) + torch.autograd.grad(o, (q, k, v), do)
    parts = [spread(*(t[i:i + n] for t in (q, k, v, do)), False, 1 / 8)
             for i in range(0, T, n)]
    for g, part, name in zip(got, zip(*parts), ("o", "dq", "dk", "dv")):
        w = torch.cat([w for w, _ in part])
        off = torch.stack([e for _, e in part]).norm()
        assert torch.isfinite(g).all(), name
        err = (g.double() - w).norm()
        assert err <= 2 * off, f"{name}: {err / off:.3g} of the mean error"


@pytest.mark.parametrize("dtype", [FH, BF])
@pytest.mark.parametrize("T", [200, 2048])
def test_attention_many_small_probabilities(T, dtype):
    """One key takes nearly all of each row; what the others hold adds up
    from probabilities of 2^-25.  Those are off by their own rounding, or by
    2^-32 of the largest where fp16 has no more; p and o are rounded once
    each, and 32-bit scores of 17 are off by less than 2^-14 of p."""
    D = 8
    q, k, v = (torch.zeros(T, 1, D, device="cuda", dtype=dtype)
               for _ in range(3))
    q[..., 0] = 1.0
    k[7, 0, 0] = 17.25
    v[:] = normal((T, 1, D), dtype, 1).abs() * 40
    v[7] = 0
    o = flash_attention_packed(q, k, v, cu_of(0, T), scale=1.0)
    p = (q[:, 0].double() @ k[:, 0].double().T).softmax(-1)
    w = (p @ v[:, 0].double())[:, None]
    mass = (p @ v[:, 0].double().abs())[:, None]
    u = torch.finfo(dtype).eps / 2
    many = v[:, 0].double().abs().sum(0)
    tiny = 2.0 ** -25 if dtype == FH else 0.0
    room = u * (mass + w) + 2.0 ** -14 * mass + tiny
    if dtype == FH:
        room = room + 2.0 ** -32 * many
    assert ((o.double() - w).abs() <= room).all()
    assert (w > 4 * room).all()        # a lost row would show


# ---- few keys in a row -----------------------------------------------------

@pytest.mark.parametrize("dtype", [FH, BF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [2, 4, 8, 16, 32, 64])
def test_attention_narrow_window(window, D, dtype):
    """Rows of few keys: D owes nothing to a rounded o.  The mean error is a
    bound by itself (a value's rounding is off by 0.7 of u / sqrt(3) on the
    average of its mantissas), 65 to 131 thousand values stray by 1%."""
    T = 1024
    q, k, v = (leaf(normal((T, 1, D), dtype, i)) for i in range(3))
    do = normal((T, 1, D), dtype, 3)
    o = flash_attention_packed(q, k, v, cu_of(0, T), causal=True,
                               window=window)
    got = (o,) + torch.autograd.grad(o, (q, k, v), do)
    for g, (w, off), name in zip(got, spread(q, k, v, do, True, D ** -0.5,
                                             window, True),
                                 ("o", "dq", "dk", "dv")):
        err = (g.double() - w).norm()
        assert err <= off, f"{name}: {err / off:.3g} of the mean error"


# ---- a sequence by itself and among others ---------------------------------

@pytest.mark.parametrize("dtype", [FH, BF])
@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_does_not_depend_on_the_batch(causal, D, dtype):
    """A sequence has the same bits alone and behind others (of gradients of
    k and v where both calls sum without splits, as over short sequences)."""
    for spans, whole in (([40] * 25, True), ([300, 40, 700, 256, 5], False),
                         ([3000, 17, 100], False)):
        T = sum(spans)
        q, k, v, do = (normal((T, n, D), dtype, i)
                       for i, n in enumerate((4, 2, 2, 4)))
        q, k, v = leaf(q), leaf(k), leaf(v)
        cu = [sum(spans[:i]) for i in range(len(spans) + 1)]
        o = flash_attention_packed(q, k, v, cu_of(*cu), causal=causal)
        got = (o,) + torch.autograd.grad(o, (q, k, v), do)
        for b, e in zip(cu[:-1], cu[1:]):
            if e - b > 256:
                continue
            part = [leaf(t[b:e]) for t in (q, k, v)]
            o = flash_attention_packed(*part, cu_of(0, e - b), causal=causal)
            alone = (o,) + torch.autograd.grad(o, part, do[b:e])
            for x, y, name in zip(got, alone, ("o", "dq", "dk", "dv")):
                if whole or name in ("o", "dq"):
                    assert torch.equal(x[b:e], y), (name, e - b)


# ---- rows of no sequence ---------------------------------------------------

@pytest.mark.parametrize("T,cu", [(300, (5, 105, 300)), (700, (300, 301)),
                                  (520, (128, 128, 390, 400)), (64, (64, 64)),
                                  (200, (130, 200))])
@pytest.mark.parametrize("padded", [False, True])
def test_attention_rows_in_front(padded, T, cu):
    """cu_seqlens may begin behind the first row: rows in front of it get
    zeros, the others what they get without those rows."""
    q, k, v, do = (normal((T, n, 64), BF, i)
                   for i, n in enumerate((4, 2, 2, 4)))
    lengths = torch.tensor([max(b - a - 3, 0) for a, b in zip(cu, cu[1:])],
                           dtype=torch.int32, device="cuda") \
        if padded else None
    for t in (q, k, v, do):
        t[:cu[0]] = math.nan
    q, k, v = leaf(q), leaf(k), leaf(v)
    # memory that is handed out next holds no zeros
    junk = torch.full((T * 64 * 4 * 8,), math.nan, device="cuda", dtype=BF)
    del junk
    o = flash_attention_packed(q, k, v, cu_of(*cu), lengths, causal=True)
    got = (o,) + torch.autograd.grad(o, (q, k, v), do)
    part = [leaf(t[cu[0]:]) for t in (q, k, v)]
    o = flash_attention_packed(*part, cu_of(*(n - cu[0] for n in cu)),
                               lengths, causal=True)
    rest = (o,) + torch.autograd.grad(o, part, do[cu[0]:])
    for x, y in zip(got, rest):
        assert (x[:cu[0]] == 0).all() and torch.equal(x[cu[0]:], y)


# ---- together --------------------------------------------------------------

class Rounded(torch.autograd.Function):
    """To bf16 and back, and its gradient too, as between two operators."""

    @staticmethod
    def forward(ctx, x):
        return x.to(BF).to(x.dtype)

    @staticmethod
    def backward(ctx, g):
        return g.to(BF).to(g.dtype)


def plain_block(x, params, cu, angle, r):
    """One block of packed tokens in 64 bits, `r` behind every operator."""
    wqkv, wo, w1, w2, g = params
    T, D = x.shape[0], 64
    q, k, v = r(x @ wqkv).split([256, 128, 128], -1)
    q, k, v = (t.unflatten(-1, (-1, D)).transpose(0, 1) for t in (q, k, v))
    q, k = (r(torch.cat([t[..., :32] * angle.cos() - t[..., 32:] * angle.sin(),
                         t[..., 32:] * angle.cos() + t[..., :32] * angle.sin()],
                        -1)) for t in (q, k))
    k, v = (t.repeat_interleave(2, 0) for t in (k, v))
    row = torch.arange(T, device=x.device)
    seq = torch.searchsorted(cu.long(), row, right=True)
    seen = (seq[:, None] == seq) & (seq <= len(cu) - 1) & (row <= row[:, None])
    s = (q @ k.mT / 8).masked_fill(~seen, -1e300)
    o = r((s.softmax(-1) * seen) @ v).transpose(0, 1).reshape(T, 256)
    h = r(o @ wo)
    S = 0.9 * x + g * h * (h.square().mean(-1, keepdim=True)
                           + 1e-6).rsqrt() * w1
    return S * (S.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w2, S


def test_together_each_gradient_by_itself():
    """rope, attention, block norm and clipping in one step: every
    parameter's gradient, and the q, k and v columns by themselves, against
    64 bits.  What they may be off is what bf16 between the operators costs,
    taken from the same 64-bit step with that rounding; its errors are other
    ones of the same size, and twice their norm is allowed."""
    T = 300
    x = normal((T, 256), BF, 0)
    params = [normal((256, 512), BF, 1, 0.06), normal((256, 256), BF, 2, 0.06)]
    params += [(1 + normal((256,), FP, 3 + i, 0.2)).to(BF) for i in range(3)]
    params = [torch.nn.Parameter(p) for p in params]
    cu, pos = cu_of(0, 120, 120, 270), torch.randint(
        0, 400, (3, T), generator=torch.Generator().manual_seed(5)).cuda()
    inv = 1e4 ** (-torch.arange(32, dtype=torch.float64) / 32)
    table = torch.outer(torch.arange(400, dtype=torch.float64), inv).cuda()
    out_grads = normal((T, 256), BF, 7), normal((T, 256), BF, 8)

    wqkv, wo, w1, w2, g = params
    q, k, v = (x @ wqkv).split([256, 128, 128], -1)
    q, k, v = (t.unflatten(-1, (-1, 64)) for t in (q, k, v))
    q, k = fused_rope_axes(q, k, pos, table.cos().float(),
                           table.sin().float(), [8, 12, 12])
    o = flash_attention_packed(q, k, v, cu, causal=True)
    out = fused_block_norm(o.reshape(T, 256) @ wo, x, w1, w2, g, 0.9)
    for p, grad in zip(params, torch.autograd.grad(out, params, out_grads)):
        p.grad = grad
    total = clip_grad_norm_(params, 1.0)

    axis = torch.tensor([0] * 8 + [1] * 12 + [2] * 12, device="cuda")
    angle = table[pos[axis].t(), torch.arange(32, device="cuda")]
    grads = []
    for r in (lambda t: t, Rounded.apply):
        p64 = [p.detach().double().requires_grad_() for p in params]
        res = plain_block(x.double(), p64, cu, angle, r)
        grads.append(torch.autograd.grad(
            res, p64, [t.double() for t in out_grads]))
    want = sum(t.square().sum() for t in grads[0]) ** 0.5
    assert (total.double() - want).abs() <= 2 ** -6 * want
    names = ["q", "k", "v", "wo", "post", "pre", "gate"]

    def parts(ts):
        return [*ts[0].split([256, 128, 128], -1), *ts[1:]]

    for name, got, exact, rounded in zip(names, parts(
            [p.grad.double() for p in params]), *map(parts, grads)):
        off = (Rounded.apply(rounded) - exact).norm()
        assert 0 < off <= 0.05 * exact.norm(), name   # it says something
        err = (got * total.double() - exact).norm()
        assert err <= 2 * off, f"{name}: {err / off:.3g} of bf16's error"


def test_attention_too_many_blocks_are_refused():
    """More threads than a launch may have, before anything is allocated."""
    q = torch.zeros(1, 32, 8, device="cuda", dtype=BF).expand(1 << 27, 32, 8)
    before = torch.cuda.memory_allocated()
    with pytest.raises(RuntimeError, match="too many rows"):
        flash_attention_packed(q, q, q, cu_of(0, 1 << 27))
    many = torch.zeros(1 << 23, device="cuda", dtype=torch.int32)
    with pytest.raises(RuntimeError, match="too many rows"):
        flash_attention_packed(q[:1], q[:1], q[:1], many)
    del many
    assert torch.cuda.memory_allocated() <= before + 4096
