"""Cases and plain forms of the packed-sequence training operators.

Four operators of one training step over packed token sequences:

* ``attention``: attention over packed (or padded) sequences, with gradients
* ``rope``: rotary positions on one or several axes, with gradients
* ``block_norm``: norm after a block, gate, residual scale and sum, and the
  norm before the next block, with gradients
* ``clip``: the global norm of many gradients, and clipping by it

``run`` computes each in plain torch operations in 32 bits, or, where ``own``
is true, through this framework's entry points.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16,
          "fp32": torch.float32}


# ---- cases ---------------------------------------------------------------

def listed():
    return [
        # an encoder's batch of short padded rows, as one job's step has it:
        # every row in a span of 128, some nearly empty, one empty
        {"name": "attention padded encoder", "op": "attention",
         "spans": ",".join(["128"] * 32),
         "lengths": "128,97,128,64,31,128,5,110,128,128,77,1,128,90,128,16,"
                    "128,128,50,0,128,101,127,33,128,128,60,128,8,119,128,128",
         "rows": 4096, "heads": 12, "kv_heads": 12, "dim": 64,
         "causal": False, "window": 0, "dtype": "bf16", "train": True},
        # the smallest call: a handful of short pieces, nothing but latency
        {"name": "attention few tokens", "op": "attention",
         "spans": "1,7,24,0,33", "lengths": "", "rows": 72, "heads": 8,
         "kv_heads": 4, "dim": 64, "causal": True, "window": 0,
         "dtype": "bf16", "train": False},
        # documents of ragged lengths packed into one row of 8k tokens
        {"name": "attention packed documents", "op": "attention",
         "spans": "2900,511,64,1733,9,1200,640,130,1005", "lengths": "",
         "rows": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "causal": True, "window": 0, "dtype": "bf16", "train": True},
        # one long document: nothing but matrix work
        {"name": "attention long document", "op": "attention",
         "spans": "8192", "lengths": "", "rows": 8192, "heads": 16,
         "kv_heads": 4, "dim": 128, "causal": True, "window": 0,
         "dtype": "bf16", "train": True},
        # odd lengths, heads of an odd size and a sliding window
        {"name": "attention window odd", "op": "attention",
         "spans": "1999,1,745,254", "lengths": "", "rows": 3001, "heads": 6,
         "kv_heads": 2, "dim": 80, "causal": True, "window": 257,
         "dtype": "fp16", "train": True},
        # one short prompt, forward only
        {"name": "rope one prompt", "op": "rope", "tokens": 37, "heads": 8,
         "kv_heads": 4, "dim": 64, "rotary": 64, "sections": "32",
         "dtype": "fp16", "train": False},
        # packed text and image tokens on three axes, a training step
        {"name": "rope packed three axes", "op": "rope", "tokens": 16384,
         "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "sections": "16,24,24", "dtype": "bf16", "train": True},
        # few rows of a narrow model, forward only
        {"name": "block norm few rows", "op": "block_norm", "batch": 2,
         "seq": 29, "dim": 512, "gate": "channel", "alpha": 1.0,
         "dtype": "bf16", "train": False},
        # an odd width in 32 bits, gates by sequence
        {"name": "block norm odd fp32", "op": "block_norm", "batch": 5,
         "seq": 333, "dim": 1001, "gate": "sequence", "alpha": 0.81,
         "dtype": "fp32", "train": True},
        # a wide model's step, gates by sequence
        {"name": "block norm wide", "op": "block_norm", "batch": 4,
         "seq": 4096, "dim": 4096, "gate": "sequence", "alpha": 1.0,
         "dtype": "bf16", "train": True},
        # the gradients of a small decoder with an odd vocabulary: some
        # dozens of tensors, some of a few hundred values, 32-bit norms
        {"name": "clip small decoder", "op": "clip", "hidden": 512,
         "ffn": 1408, "layers": 4, "vocab": 1021, "dtype": "bf16",
         "norm_dtype": "fp32", "max_norm": 1.0},
        # the gradients of a decoder of about 0.9 billion weights
        {"name": "clip large decoder", "op": "clip", "hidden": 2048,
         "ffn": 5632, "layers": 16, "vocab": 32000, "dtype": "bf16",
         "norm_dtype": "bf16", "max_norm": 1.0},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_attention(rng):
    dim = rng.choice([64, 128, 64, 128, 32, 72, 80, 96, 120])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4])
    rows = _log_int(rng, 16, 8192)
    # the plain form holds rows x rows scores of every head
    heads = kv_heads if heads * rows * rows > 16 * 8192 * 8192 else heads
    spans, left = [], rows - rng.choice([0, 0, 0, rng.randint(0, rows // 8)])
    while left and len(spans) < 40:
        n = min(left, _log_int(rng, 1, rows))
        spans.append(n)
        left -= n
    lengths = ""
    if rng.random() < 0.3:
        lengths = ",".join(str(rng.choice([n, rng.randint(0, n)]))
                           for n in spans)
    causal = rng.random() < 0.7
    return {"op": "attention", "spans": ",".join(map(str, spans)),
            "lengths": lengths, "rows": rows, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "causal": causal,
            "window": _log_int(rng, 1, rows)
            if causal and rng.random() < 0.3 else 0,
            "dtype": rng.choice(["bf16", "bf16", "fp16"]),
            "train": rng.random() < 0.7}


def _draw_rope(rng):
    dim = rng.choice([64, 128, 128, 80, 96, 72, 256])
    rotary = rng.choice([dim, dim, dim // 4 * 2])
    half = rotary // 2
    axes = rng.choice([1, 2, 3, 3])
    cuts = sorted(rng.sample(range(1, half), axes - 1))
    sections = [b - a for a, b in zip([0] + cuts, cuts + [half])]
    kv_heads = rng.choice([1, 2, 4, 8] if dim < 256 else [1, 2, 4])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    return {"op": "rope",
            "tokens": _log_int(rng, 1, 8192 if dtype == "fp32" else 16384),
            "heads": kv_heads * rng.choice([1, 2, 4]), "kv_heads": kv_heads,
            "dim": dim, "rotary": rotary,
            "sections": ",".join(map(str, sections)), "dtype": dtype,
            "train": rng.random() < 0.7}


def _draw_block_norm(rng):
    dim = rng.choice([_log_int(rng, 64, 8192),
                      _log_int(rng, 8, 1024) * 8])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    most = 4 * 4096 * 4096 // dim // (2 if dtype == "fp32" else 1)
    rows = _log_int(rng, 1, min(16384, most))
    batch = rng.randint(1, min(rows, 8))
    return {"op": "block_norm", "batch": batch, "seq": rows // batch,
            "dim": dim, "gate": rng.choice(["none", "channel", "sequence",
                                            "token"]),
            "alpha": rng.choice([1.0, 0.5, 1.25]), "dtype": dtype,
            "train": rng.random() < 0.7}


def _draw_clip(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    wide = dtype != "fp32"
    return {"op": "clip", "hidden": _log_int(rng, 16, 2048 if wide else 1024),
            "ffn": _log_int(rng, 32, 5632 if wide else 4096),
            "layers": rng.randint(1, 16), "vocab": _log_int(rng, 100, 32000),
            "dtype": dtype, "norm_dtype": rng.choice([dtype, "fp32"]),
            "max_norm": rng.choice([0.5, 1.0, 5.0, 1e6])}


def draw(rng):
    return rng.choice([_draw_attention, _draw_rope, _draw_block_norm,
                       _draw_clip])(rng)


# ---- inputs --------------------------------------------------------------

def _ints(text):
    return [int(n) for n in text.split(",")] if text else []


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype, scale=1.0, shift=0.0):
    x = torch.randn(shape, device="cuda", generator=g)
    return x.mul_(scale).add_(shift).to(dtype)


def _heads_of(g, tokens, heads, kv_heads, dim, dtype):
    """q, k and v as slices of one fused projection, as models have them."""
    qkv = _normal(g, (tokens, (heads + 2 * kv_heads) * dim), dtype)
    q, k, v = qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], -1)
    return (q.unflatten(-1, (heads, dim)), k.unflatten(-1, (kv_heads, dim)),
            v.unflatten(-1, (kv_heads, dim)))


def _positions(axes, tokens, seed):
    """Positions of text pieces (all axes count on) between images (first
    axis held, the others walk a grid), as int64 [axes, tokens]."""
    r = torch.Generator()
    r.manual_seed(seed)
    out, at, made = [], 0, 0
    while made < tokens:
        text = int(torch.randint(1, 400, (), generator=r))
        n = torch.arange(text) + at
        out.append(torch.stack([n] * axes))
        at, made = at + text, made + text
        if axes > 1:
            h, w = (int(torch.randint(2, 33, (), generator=r))
                    for _ in range(2))
            p = torch.arange(h * w)
            grid = [torch.zeros_like(p), p // w, p % w]
            out.append(torch.stack(grid[:axes] if axes == 3
                                   else grid[1:]) + at)
            at, made = at + max(h, w), made + h * w
        if int(torch.randint(0, 8, (), generator=r)) == 0:
            at = 0  # the next packed sequence
    return torch.cat(out, -1)[:, :tokens].contiguous()


def _prepare_attention(case, seed):
    dtype, g = DTYPES[case["dtype"]], _generator(seed)
    H, HK, D, T = case["heads"], case["kv_heads"], case["dim"], case["rows"]
    spans, lengths = _ints(case["spans"]), _ints(case["lengths"])
    q, k, v = _heads_of(g, T, H, HK, D, dtype)
    cu = torch.tensor([0] + spans).cumsum(0).to("cuda", torch.int32)
    return {"q": q, "k": k, "v": v, "cu_seqlens": cu,
            "lengths": torch.tensor(lengths, device="cuda",
                                    dtype=torch.int32) if lengths else None,
            "do": _normal(g, (T, H, D), dtype) if case["train"] else None}


def _prepare_rope(case, seed):
    dtype, g = DTYPES[case["dtype"]], _generator(seed)
    T, H, HK, D = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    sections, R = _ints(case["sections"]), case["rotary"]
    q, k, _ = _heads_of(g, T, H, HK, D, dtype)
    pos = _positions(len(sections), T, seed)
    inv = 1e4 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    angle = torch.outer(torch.arange(int(pos.max()) + 1,
                                     dtype=torch.float64), inv)
    state = {"q": q, "k": k, "positions": pos.cuda(),
             "cos": angle.cos().float().cuda(),
             "sin": angle.sin().float().cuda(), "sections": sections}
    if case["train"]:
        state["dq"] = _normal(g, (T, H, D), dtype)
        state["dk"] = _normal(g, (T, HK, D), dtype)
    return state


def _prepare_block_norm(case, seed):
    dtype, g = DTYPES[case["dtype"]], _generator(seed)
    B, S, D = case["batch"], case["seq"], case["dim"]
    gate = {"none": None, "channel": (D,), "sequence": (B, D),
            "token": (B, S, D)}[case["gate"]]
    state = {"h": _normal(g, (B, S, D), dtype, 0.7),
             "x": _normal(g, (B, S, D), dtype, 2.0),
             "post_weight": _normal(g, (D,), dtype, 0.1, 1.0),
             "pre_weight": _normal(g, (D,), dtype, 0.1, 1.0),
             "gate": None if gate is None else
             _normal(g, gate, dtype, 0.3, 0.5)}
    if case["train"]:
        state["dn"] = _normal(g, (B, S, D), dtype)
        state["ds"] = _normal(g, (B, S, D), dtype)
    return state


def _shapes(case):
    """(shape, whether it is a norm's weight) of a decoder's parameters."""
    h, f, v = case["hidden"], case["ffn"], case["vocab"]
    layer = [((3 * h, h), False), ((h, h), False), ((h,), True),
             ((2 * f, h), False), ((h, f), False), ((h,), True)]
    return ([((v, h), False)] + layer * case["layers"]
            + [((h,), True), ((v, h), False)])


def _prepare_clip(case, seed):
    g = _generator(seed)
    shapes = _shapes(case)
    dtypes = [DTYPES[case["norm_dtype" if norm else "dtype"]]
              for _, norm in shapes]
    state = {"params": [], "reduced": [], "grads": []}
    for dtype in dict.fromkeys(dtypes):
        mine = [s for (s, _), d in zip(shapes, dtypes) if d == dtype]
        sizes = [math.prod(s) for s in mine]
        # reduced gradients arrive in one flat bucket of each type
        state["reduced"].append(_normal(g, (sum(sizes),), dtype, 0.02))
        flat = torch.zeros_like(state["reduced"][-1])
        state["grads"].append(flat)
        for s, piece in zip(mine, flat.split(sizes)):
            p = torch.nn.Parameter(torch.empty(s, device="cuda", dtype=dtype))
            p.grad = piece.view(s)
            state["params"].append(p)
    return state


def prepare(case, seed):
    state = {"attention": _prepare_attention, "rope": _prepare_rope,
             "block_norm": _prepare_block_norm,
             "clip": _prepare_clip}[case["op"]](case, seed)
    state["case"] = case
    for n in ("q", "k", "v", "h", "x", "post_weight", "pre_weight", "gate"):
        if case.get("train") and state.get(n) is not None:
            # a leaf of its own that keeps a slice's strides
            state[n] = state[n].detach().requires_grad_()
    return state


# ---- plain forms ---------------------------------------------------------

def _seen(s, c):
    """[rows, rows]: whether row i's query sees row j's key."""
    cu, T = s["cu_seqlens"].long(), c["rows"]
    row = torch.arange(T, device=cu.device)
    seq = torch.searchsorted(cu, row, right=True) - 1
    inside = row < cu[-1]
    seq = seq.clamp(max=cu.numel() - 2)
    if s["lengths"] is not None:
        inside = inside & (row - cu[seq] < s["lengths"].long()[seq])
    seen = (seq[:, None] == seq) & inside[:, None] & inside
    if c["causal"]:
        seen &= row <= row[:, None]
    if c["window"]:
        seen &= row > row[:, None] - c["window"]
    return seen


def _plain_attention(s, c):
    H, HK, D = c["heads"], c["kv_heads"], c["dim"]
    T, rep, dtype = c["rows"], H // HK, s["q"].dtype

    def split(x, n):  # [T, n, D] -> [HK, n / HK, T, D]
        return x.detach().float().transpose(0, 1).reshape(HK, n // HK, T, D)

    def merge(x):
        return x.reshape(-1, T, D).transpose(0, 1).to(dtype).contiguous()

    q, k, v = split(s["q"], H), split(s["k"], HK), split(s["v"], HK)
    scale, seen = 1.0 / math.sqrt(D), _seen(s, c)
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)
    p.masked_fill_(~seen, float("-inf"))
    p.sub_(p.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(total + (total == 0))
    o = torch.matmul(p, v)
    if not c["train"]:
        return merge(o)
    do = split(s["do"], H)
    dv = torch.matmul(p.transpose(-1, -2), do).sum(1, keepdim=True)
    ds = torch.matmul(do, v.transpose(-1, -2))
    ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2), q).sum(1, keepdim=True)
    return merge(o), merge(dq), merge(dk), merge(dv)


def _plain_rope(s, c):
    R = c["rotary"]
    half = R // 2
    at = torch.cat([p.expand(n, -1) for p, n in
                    zip(s["positions"], s["sections"])])   # [R/2, T]
    place = torch.arange(half, device=at.device)[:, None]
    cos = s["cos"][at, place].t()[:, None]                 # [T, 1, R/2]
    sin = s["sin"][at, place].t()[:, None]

    def turn(x, sin):
        x = x.detach()
        a, b = x[..., :half].float(), x[..., half:R].float()
        return torch.cat([(a * cos - b * sin).to(x.dtype),
                          (b * cos + a * sin).to(x.dtype), x[..., R:]], -1)

    out = turn(s["q"], sin), turn(s["k"], sin)
    if c["train"]:
        out += turn(s["dq"], -sin), turn(s["dk"], -sin)
    return out


def _plain_block_norm(s, c):
    dtype, D, alpha = s["h"].dtype, c["dim"], c["alpha"]
    gated = s["gate"] is not None
    h, x, w1, w2 = (s[n].detach().float()
                    for n in ("h", "x", "post_weight", "pre_weight"))
    g = s["gate"].detach().float() if gated else 1.0
    g = g[:, None] if c["gate"] == "sequence" else g
    r1 = torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6)
    h = h * r1
    y = alpha * x + g * (h * w1)
    r2 = torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)
    n = y * r2
    out = (n * w2).to(dtype), y.to(dtype)
    if not c["train"]:
        return out
    dn, ds = s["dn"].float(), s["ds"].float()
    dw2 = (dn * n).sum((0, 1))
    dn = dn * w2
    ds = ds + r2 * (dn - n * (dn * n).mean(-1, keepdim=True))
    t = ds * h
    dw1 = (g * t).sum((0, 1))
    u = g * ds * w1
    dh = r1 * (u - h * (u * h).mean(-1, keepdim=True))
    out += dh.to(dtype), (alpha * ds).to(dtype), dw1.to(dtype), dw2.to(dtype)
    if gated:
        dg = t * w1
        dg = (dg.sum((0, 1)) if c["gate"] == "channel" else
              dg.sum(1) if c["gate"] == "sequence" else dg)
        out += (dg.to(dtype),)
    return out


def _plain_clip(s, c):
    # one flat buffer of each type holds all its gradients
    total = sum(f.float().square().sum() for f in s["grads"]).sqrt()
    factor = (c["max_norm"] / (total + 1e-6)).clamp(max=1.0)
    for f in s["grads"]:
        f.copy_(f.float() * factor)
    return [total] + s["grads"]


# ---- the framework's calls -----------------------------------------------

def _own_attention(s, c):
    from gpuschedule_amd.ops import flash_attention_packed
    o = flash_attention_packed(s["q"], s["k"], s["v"], s["cu_seqlens"],
                               lengths=s["lengths"], causal=c["causal"],
                               window=c["window"] or None)
    if not c["train"]:
        return o
    return (o.detach(),) + torch.autograd.grad(
        o, (s["q"], s["k"], s["v"]), s["do"])


def _own_rope(s, c):
    from gpuschedule_amd.ops import fused_rope_axes
    q, k = fused_rope_axes(s["q"], s["k"], s["positions"], s["cos"],
                           s["sin"], s["sections"])
    if not c["train"]:
        return q, k
    return (q.detach(), k.detach()) + torch.autograd.grad(
        (q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))


def _own_block_norm(s, c):
    from gpuschedule_amd.ops import fused_block_norm
    n, y = fused_block_norm(s["h"], s["x"], s["post_weight"],
                            s["pre_weight"], gate=s["gate"],
                            residual_scale=c["alpha"], eps=1e-6)
    if not c["train"]:
        return n, y
    leaves = [s[m] for m in ("h", "x", "post_weight", "pre_weight")]
    leaves += [s["gate"]] if s["gate"] is not None else []
    return (n.detach(), y.detach()) + torch.autograd.grad(
        (n, y), leaves, (s["dn"], s["ds"]))


def _own_clip(s, c):
    from gpuschedule_amd.ops import clip_grad_norm_
    return [clip_grad_norm_(s["params"], c["max_norm"])] + s["grads"]


_PLAIN = {"attention": _plain_attention, "rope": _plain_rope,
          "block_norm": _plain_block_norm, "clip": _plain_clip}
_OWN = {"attention": _own_attention, "rope": _own_rope,
        "block_norm": _own_block_norm, "clip": _own_clip}


def run(state):
    case = state["case"]
    if case["op"] == "clip":
        # the reduced buckets go back into the gradients first, as a
        # data-parallel step does it: clipping changes them in place
        torch._foreach_copy_(state["grads"], state["reduced"])
    return (_OWN if own else _PLAIN)[case["op"]](state, case)


# ---- what a pass cannot do without ---------------------------------------

def _pairs(case):
    """Pairs of a query and a key that it sees."""
    spans = _ints(case["spans"])
    total = 0
    for n in _ints(case["lengths"]) or spans:
        w = min(case["window"] or n, n)
        total += (w * (w + 1) // 2 + (n - w) * w if case["causal"]
                  else n * n)
    return total


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "attention":
        row = case["rows"] * case["dim"] * size
        q, kv = row * case["heads"], row * case["kv_heads"]
        flops = 4 * case["dim"] * case["heads"] * _pairs(case)
        if not case["train"]:
            return {"bytes": 2 * q + 2 * kv, "flops": flops}
        # in: q, k, v, do; out: o and three gradients
        return {"bytes": 4 * q + 4 * kv, "flops": 3.5 * flops}
    if case["op"] == "rope":
        x = case["tokens"] * (case["heads"] + case["kv_heads"])
        passes = 2 if case["train"] else 1
        axes = len(_ints(case["sections"]))
        return {"bytes": passes * 2 * x * case["dim"] * size
                + 8 * axes * case["tokens"],
                "flops": passes * 3 * x * case["rotary"]}
    if case["op"] == "block_norm":
        n = case["batch"] * case["seq"] * case["dim"]
        gate = {"none": 0, "channel": case["dim"],
                "sequence": case["batch"] * case["dim"],
                "token": n}[case["gate"]]
        train = case["train"]
        # in: h, x (dn, ds); out: n, the sum (dh, dx)
        return {"bytes": size * ((8 if train else 4) * n
                                 + (2 if train else 1)
                                 * (gate + 2 * case["dim"])),
                "flops": (36 if train else 11) * n}
    total = flops = 0
    for shape, norm in _shapes(case):
        n = math.prod(shape)
        total += 2 * n * (4 if case["norm_dtype" if norm else "dtype"]
                          == "fp32" else 2)
        flops += 3 * n
    return {"bytes": total, "flops": flops}


# ---- the definitions in 64 bits ------------------------------------------

def _exact_attention(s, c):
    H, HK, D = c["heads"], c["kv_heads"], c["dim"]
    names = ("q", "k", "v") + (("do",) if c["train"] else ())
    q, k, v, *do = (s[n].detach().double() for n in names)
    o = torch.zeros_like(q)
    grads = [torch.zeros_like(x) for x in (q, k, v)] if do else []
    start = 0
    spans = _ints(c["spans"])
    for span, n in zip(spans, _ints(c["lengths"]) or spans):
        at = slice(start, start + n)
        start += span
        if n == 0:
            continue
        i = torch.arange(n, device=q.device)
        far = i[:, None] - i[None, :]
        bias = torch.zeros(n, n, device=q.device, dtype=torch.float64)
        if c["causal"]:
            bias[far < 0] = -math.inf
        if c["window"]:
            bias[far >= c["window"]] = -math.inf
        for h in range(H):
            kv = h * HK // H
            qh, kh, vh = q[at, h], k[at, kv], v[at, kv]
            prob = torch.softmax(qh @ kh.T / D ** 0.5 + bias, -1)
            o[at, h] = prob @ vh
            if do:
                doh = do[0][at, h]
                grads[2][at, kv] += prob.T @ doh
                dp = doh @ vh.T
                dz = prob * (dp - (prob * dp).sum(-1, keepdim=True))
                dz = dz / D ** 0.5
                grads[0][at, h] = dz @ kh
                grads[1][at, kv] += dz.T @ qh
    return (o, *grads) if do else o


def _exact_rope(s, c):
    half = c["rotary"] // 2
    T = c["tokens"]
    turn = torch.empty(T, 1, half, device="cuda", dtype=torch.complex128)
    j = 0
    for axis, n in enumerate(s["sections"]):
        rows = s["positions"][axis]
        turn[:, 0, j:j + n] = torch.complex(
            s["cos"][rows, j:j + n].double(), s["sin"][rows, j:j + n].double())
        j += n

    def rotate(x, by):
        x = x.detach().double().clone()
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * by
        x[..., :half], x[..., half:2 * half] = z.real, z.imag
        return x

    out = [rotate(s["q"], turn), rotate(s["k"], turn)]
    if c["train"]:
        out += [rotate(s["dq"], turn.conj()), rotate(s["dk"], turn.conj())]
    return tuple(out)


def _exact_block_norm(s, c):
    names = ["h", "x", "post_weight", "pre_weight"]
    names += ["gate"] if s["gate"] is not None else []
    with torch.enable_grad():
        leaf = {n: s[n].detach().double().requires_grad_() for n in names}
        g = leaf.get("gate", torch.ones((), device="cuda"))
        if c["gate"] == "sequence":
            g = g.unsqueeze(1)

        def norm(a, w):
            return w * a / torch.sqrt((a * a).mean(-1, keepdim=True) + 1e-6)

        y = c["alpha"] * leaf["x"] + g * norm(leaf["h"], leaf["post_weight"])
        n = norm(y, leaf["pre_weight"])
        out = (n.detach(), y.detach())
        if c["train"]:
            out += torch.autograd.grad(
                (n, y), [leaf[m] for m in names],
                (s["dn"].double(), s["ds"].double()))
    return out


def _exact_clip(s, c):
    squares = [torch.linalg.vector_norm(f, dtype=torch.float64) ** 2
               for f in s["reduced"]]
    total = torch.stack(squares).sum() ** 0.5
    factor = min(1.0, c["max_norm"] / (float(total) + 1e-6))
    return [total] + [f.double() * factor for f in s["reduced"]]


def exact(case, seed):
    return {"attention": _exact_attention, "rope": _exact_rope,
            "block_norm": _exact_block_norm,
            "clip": _exact_clip}[case["op"]](prepare(case, seed), case)
