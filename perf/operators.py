"""The token operators and the optimiser step, in their plain form and through the library.

Each case is one pass as a program makes it: a layer norm's forward (and backward) pass over the tokens of feature
maps, the rotation of queries and keys by the tokens' (frame, row, column), attention over image tokens or over a
clip with its backward pass, one frame's queries against a cached clip, and an AdamW step over a model's tensors.
`own` selects the library's calls; otherwise the same formulas run as elementary torch operations in 32 bits.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6          # layer norm
BASE = 10000.0      # rotary
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.05
BLOCK = 256         # elements of a tensor that share the scales of 8-bit moments
START_STEP = 100    # steps taken before the measured one

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}

# The depth network's weight tensors, by op: (kind, input channels, output channels, kernel size).
DEPTH_OPS = (
    ("conv", 4, 16, 3), ("dwpw", 16, 24, 3), ("dwpw", 24, 96, 3), ("pw", 96, 32, 1), ("pw", 32, 128, 1),
    ("dwpw", 128, 32, 3), ("dwpw", 32, 128, 5), ("pw", 128, 56, 1), ("pw", 56, 224, 1), ("dwpw", 224, 56, 5),
    ("pw", 56, 224, 1), ("dwpw", 224, 56, 5), ("dwpw", 56, 224, 5), ("pw", 224, 104, 1), ("pw", 104, 416, 1),
    ("dwpw", 416, 104, 5), ("pw", 104, 416, 1), ("dwpw", 416, 104, 5), ("pw", 104, 416, 1), ("dwpw", 416, 104, 5),
    ("dwpw", 104, 416, 5), ("pw", 416, 176, 1), ("pw", 176, 704, 1), ("dwpw", 704, 176, 5), ("pw", 176, 704, 1),
    ("dwpw", 704, 176, 5), ("pw", 176, 704, 1), ("dwpw", 704, 176, 5), ("pw", 176, 96, 1), ("pw", 104, 96, 1),
    ("dwpw", 96, 64, 3), ("pw", 56, 64, 1), ("dwpw", 64, 48, 3), ("pw", 32, 48, 1), ("dwpw", 48, 32, 3),
    ("pw", 24, 32, 1), ("dwpw", 32, 32, 3), ("pw", 32, 1, 1))


def _library():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                           "ai-illumination-depth-model_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import illumina
    import illumina.ops
    return illumina


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _norm(name, dtype, rows, c, step):
    return {"name": name, "op": "norm", "dtype": dtype, "rows": rows, "c": c, "step": step}


def _rotary(name, dtype, b, t, h, hk, d, axes, interleaved, inverse):
    return {"name": name, "op": "rotary", "dtype": dtype, "b": b, "t": t, "h": h, "hk": hk, "d": d, "axes": axes,
            "interleaved": interleaved, "inverse": inverse}


def _attention(name, dtype, b, tq, tk, h, hk, d, causal, ragged, step):
    return {"name": name, "op": "attention", "dtype": dtype, "b": b, "tq": tq, "tk": tk, "h": h, "hk": hk, "d": d,
            "causal": causal, "ragged": ragged, "step": step}


def _adamw(name, model, width, layers, bits, grad):
    return {"name": name, "op": "adamw", "model": model, "width": width, "layers": layers, "bits": bits, "grad": grad}


def listed():
    return [
        # one frame's 14 x 14 bottleneck tokens at inference: a call that is all latency
        _norm("norm forward, one frame", "f32", 196, 176, False),
        # training over a ragged set of tokens, an odd width: no vector loads
        _norm("norm step, odd width", "f32", 10007, 417, True),
        # training, 64 frames of 28 x 28 tokens
        _norm("norm step, 64 frames", "bf16", 64 * 784, 704, True),
        # one frame's queries and keys, rows and columns, neighbouring pairs
        _rotary("rotary, one frame", "f32", 1, 196, 6, 6, 48, 2, True, False),
        # two clips of 32 frames: time, rows and columns, four queries to a key head; the gradient's direction
        _rotary("rotary, clips, inverse", "bf16", 2, 32 * 196, 12, 4, 64, 3, False, True),
        # streaming: one frame's queries against a cache of 64 frames
        _attention("attention, frame over a clip", "bf16", 1, 196, 64 * 196, 12, 4, 64, 0, False, False),
        # training in 32 bits, a small batch of single frames of odd length with a class token
        _attention("attention step, f32 frames", "f32", 2, 197, 197, 4, 4, 32, 0, False, True),
        # training, a batch of 28 x 28 frames
        _attention("attention step, image batch", "bf16", 8, 784, 784, 6, 6, 64, 0, False, True),
        # training, a clip of 32 frames in which a frame sees itself and those before it
        _attention("attention step, causal clip", "bf16", 1, 32 * 196, 32 * 196, 12, 12, 64, 196, False, True),
        # training, a padded batch of token sequences with shared key heads
        _attention("attention step, padded batch", "bf16", 4, 2500, 2500, 16, 4, 128, 1, True, True),
        # the depth network's own 112 weight tensors
        _adamw("adamw, depth network", "depth", 0, 0, 32, "f32"),
        # a transformer's tensors, moments in 8 bits, gradients in bf16
        _adamw("adamw, 8-bit moments", "blocks", 1024, 12, 8, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "stream", "train", "adamw"])
    if op == "norm":
        c = _log_int(rng, 8, 2048)
        rows = _log_int(rng, 1, min(64 * 784, 30_000_000 // c))
        return _drawn(_norm("", rng.choice(["f32", "bf16"]), rows, c, rows >= 16 and rng.random() < 0.6))
    if op == "rotary":
        axes = rng.choice([1, 2, 3])
        h = rng.choice([1, 3, 4, 6, 8, 12, 16])
        return _drawn(_rotary("", rng.choice(["f32", "bf16"]), rng.choice([1, 2, 3]), _log_int(rng, 1, 6272), h,
                              rng.choice([k for k in range(1, h + 1) if h % k == 0]), 2 * rng.randint(8, 64), axes,
                              rng.random() < 0.5, rng.random() < 0.5))
    if op == "stream":
        hk = rng.choice([1, 2, 3, 4, 8])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        tk, h, b = _log_int(rng, 1, 25000 if dtype == "bf16" else 4000), hk * rng.choice([1, 2, 4]), rng.choice([1, 1, 2, 4])
        return _drawn(_attention("", dtype, b, _log_int(rng, 1, min(800, 200_000_000 // (b * h * tk))), tk, h, hk,
                                 8 * rng.randint(2, 16), rng.choice([0, 0, 1, 49, 196]), rng.random() < 0.3, False))
    if op == "train":
        hk = rng.choice([1, 2, 3, 4, 6])
        h = hk * rng.choice([1, 1, 2, 4])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        b, d = rng.choice([1, 2, 3, 5]), 8 * rng.randint(2, 16)
        most = math.isqrt((15_000_000_000 // d if dtype == "bf16" else 8_000_000) // (b * h))
        t = _log_int(rng, 48, min(6272, most))
        return _drawn(_attention("", dtype, b, t, t, h, hk, d, rng.choice([0, 0, 1, 49, 196]), rng.random() < 0.4, True))
    return _drawn(_adamw("", "blocks", 8 * rng.randint(8, 120) + rng.choice([0, 0, 1, 3]), rng.randint(1, 10),
                         rng.choice([8, 32]), rng.choice(["f32", "bf16"])))


def _drawn(case):
    del case["name"]
    return case


def _shapes(case):
    """The tensors of an AdamW case: a list of shapes."""
    shapes = []
    if case["model"] == "depth":
        for kind, cin, cout, k in DEPTH_OPS:
            if kind == "conv":
                shapes += [(cout, cin, k, k), (cout,)]
            elif kind == "dwpw":
                shapes += [(cin, k, k), (cin,), (cout, cin), (cout,)]
            else:
                shapes += [(cout, cin), (cout,)]
        return shapes
    w = case["width"]
    for _ in range(case["layers"]):
        shapes += [(w,), (w,), (w + 2 * (w // 4), w), (w, w), (w,), (w,), (2 * w, w), (2 * w,), (w, 2 * w), (w,)]
    return shapes


def _dims(case):
    return case["b"], case["tq"], case["tk"], case["h"], case["hk"], case["d"]


def _lengths(case, g):
    """(query lengths, key lengths) of a padded batch, on the host; the first sequence is full."""
    b, tq, tk = case["b"], case["tq"], case["tk"]
    part = torch.rand(b, generator=g) * 0.8 + 0.2
    part[0] = 1.0
    return (part * tq).ceil().to(torch.int32), (part * tk).ceil().to(torch.int32)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device=DEVICE) * std).to(dtype)

    s = {"case": case}
    if case["op"] == "norm":
        dtype, rows, c = TYPES[case["dtype"]], case["rows"], case["c"]
        # activations: every channel has its own offset and spread
        s["x"] = (normal(rows, c) * (0.5 + normal(c).abs()) + normal(c)).to(dtype)
        s["weight"], s["bias"] = 1 + normal(c, std=0.2), normal(c, std=0.2)
        s["dy"] = normal(rows, c, dtype=dtype) if case["step"] else None
    elif case["op"] == "rotary":
        dtype, b, t = TYPES[case["dtype"]], case["b"], case["t"]
        packed = normal(b, t, case["h"] + 2 * case["hk"], case["d"], dtype=dtype)  # a fused projection's output
        s["q"], s["k"] = packed[:, :, :case["h"]], packed[:, :, case["h"]:case["h"] + case["hk"]]
        # frames of 14 x 14 tokens from a time of the seed's own on
        i = torch.arange(t, device=DEVICE)
        first = torch.randint(0, 5000, (b, 1), generator=g, device=DEVICE)
        grid = [first + i // 196, (i // 14 % 14).expand(b, t), (i % 14).expand(b, t)]
        s["positions"] = torch.stack(grid[3 - case["axes"]:] if case["axes"] > 1 else grid[:1]).to(torch.int32)
        pairs = case["d"] // 2
        s["sections"] = n = [pairs // case["axes"] + (a < pairs % case["axes"]) for a in range(case["axes"])]
        s["axis"] = torch.tensor([a for a in range(len(n)) for _ in range(n[a])], device=DEVICE)
        s["freq"] = torch.tensor([BASE ** (-j / n[a]) for a in range(len(n)) for j in range(n[a])],
                                 dtype=torch.float64, device=DEVICE)
        if own:
            s["plan"] = _library().createRotary(case["d"], s["sections"], base=BASE, interleaved=case["interleaved"],
                                                device=DEVICE)
    elif case["op"] == "attention":
        dtype = TYPES[case["dtype"]]
        b, tq, tk, h, hk, d = _dims(case)
        if case["step"]:
            packed = normal(b, tq, h + 2 * hk, d, dtype=dtype)  # a fused projection's output
            s["q"], s["k"], s["v"] = packed[:, :, :h], packed[:, :, h:h + hk], packed[:, :, h + hk:]
            s["dout"] = normal(b, tq, h, d, dtype=dtype)
        else:
            s["q"], s["k"], s["v"] = (normal(b, n, m, d, dtype=dtype) for n, m in ((tq, h), (tk, hk), (tk, hk)))
        s["qlens"] = s["klens"] = None
        if case["ragged"]:
            host = torch.Generator().manual_seed(seed)
            s["qlens"], s["klens"] = (x.to(DEVICE) for x in _lengths(case, host))
    else:
        shapes = _shapes(case)
        counts = [math.prod(x) for x in shapes]
        blocks = [-(-n // BLOCK) for n in counts]
        total, nb = sum(counts), sum(blocks)
        spread = torch.repeat_interleave(torch.exp(normal(len(counts))), torch.tensor(counts, device=DEVICE))
        s["flat"] = normal(total, std=0.05)
        s["grad"] = (normal(total, std=1e-3) * spread).to(TYPES[case["grad"]])
        # every tensor's moments begin at a block of their own: element -> place in the moments
        first = torch.tensor([0] + blocks[:-1], device=DEVICE).cumsum(0) * BLOCK
        start = torch.tensor([0] + counts[:-1], device=DEVICE).cumsum(0)
        s["slot"] = torch.arange(total, device=DEVICE) + torch.repeat_interleave(
            first - start, torch.tensor(counts, device=DEVICE))
        decays = torch.tensor([len(x) > 1 for x in shapes], device=DEVICE)
        s["decays"] = torch.repeat_interleave(decays, torch.tensor(counts, device=DEVICE))
        held = torch.zeros(nb * BLOCK, dtype=torch.bool, device=DEVICE)
        held[s["slot"]] = True
        if case["bits"] == 8:
            s["m"] = (torch.randint(-127, 128, (nb * BLOCK,), generator=g, device=DEVICE) * held).to(torch.int8)
            s["v"] = (torch.randint(1, 256, (nb * BLOCK,), generator=g, device=DEVICE) * held).to(torch.uint8)
            s["m_scale"] = torch.rand(nb, generator=g, device=DEVICE) * 1e-5 + 1e-6
            s["v_scale"] = torch.rand(nb, generator=g, device=DEVICE) * 1e-5 + 1e-6
        else:
            s["m"] = normal(nb * BLOCK, std=3e-4) * held
            s["v"] = normal(nb * BLOCK, std=1e-3).square() * held
            s["m_scale"] = s["v_scale"] = None
        s["step"] = START_STEP
        if own:
            ends = start.tolist() + [total]
            s["grads"] = [s["grad"][a:b].view(x) for a, b, x in zip(ends, ends[1:], shapes)]
            s["optimizer"] = _library().createOptimizer(
                [s["flat"][a:b].view(x) for a, b, x in zip(ends, ends[1:], shapes)], lr=LR, betas=(BETA1, BETA2),
                eps=ADAM_EPS, weightDecay=DECAY, decay=[len(x) > 1 for x in shapes], momentBits=case["bits"],
                gradDtype=s["grad"].dtype)
            s["optimizer"].loadState({"step": START_STEP, "m": s["m"], "v": s["v"], "mScale": s["m_scale"],
                                      "vScale": s["v_scale"]})
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(s):
    case = s["case"]
    form = {"norm": (_plain_norm, _own_norm), "rotary": (_plain_rotary, _own_rotary),
            "attention": (_plain_attention, _own_attention), "adamw": (_plain_adamw, _own_adamw)}[case["op"]]
    return form[1 if own else 0](s, case)


def _own_norm(s, case):
    ops = _library().ops
    y, mean, rstd = ops.layerNorm(s["x"], s["weight"], s["bias"], eps=EPS)
    if not case["step"]:
        return {"y": y}
    dx, dw, db = ops.layerNormBackward(s["dy"], s["x"], mean, rstd, s["weight"])
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def _own_rotary(s, case):
    q, k = _library().ops.rotary(s["q"], s["positions"], s["plan"], k=s["k"], inverse=case["inverse"])
    return {"q": q, "k": k}


def _own_attention(s, case):
    ops = _library().ops
    masks = {"causalBlock": case["causal"], "qLens": s["qlens"], "kLens": s["klens"]}
    out, lse = ops.attention(s["q"], s["k"], s["v"], **masks)
    if not case["step"]:
        return {"out": out, "lse": lse}
    dq, dk, dv = ops.attentionBackward(s["dout"], s["q"], s["k"], s["v"], out, lse, **masks)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _own_adamw(s, case):
    s["optimizer"].step(s["grads"])
    m, v = s["optimizer"].moments()
    return {"p": s["flat"], "m": m, "v": v}


def _plain_norm(s, case):
    x = s["x"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = (centred.square().mean(1, keepdim=True) + EPS).rsqrt()
    xhat = centred * rstd
    y = (xhat * s["weight"] + s["bias"]).to(s["x"].dtype)
    if not case["step"]:
        return {"y": y}
    dy = s["dy"].float()
    wg = dy * s["weight"]
    dx = rstd * (wg - wg.mean(1, keepdim=True) - xhat * (wg * xhat).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dw": (dy * xhat).sum(0), "db": dy.sum(0)}


def _plain_rotary(s, case):
    # angles in 64 bits: 32 lose the phase of far positions
    angle = s["positions"].permute(1, 2, 0)[:, :, s["axis"]].double() * s["freq"]
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    if case["inverse"]:
        sin = -sin

    def turn(x):
        f = x.float()
        a, b = (f[..., 0::2], f[..., 1::2]) if case["interleaved"] else f.chunk(2, -1)
        ra, rb = a * cos - b * sin, a * sin + b * cos
        return (torch.stack((ra, rb), -1).flatten(-2) if case["interleaved"] else torch.cat((ra, rb), -1)).to(x.dtype)

    return {"q": turn(s["q"]), "k": turn(s["k"])}


def _plain_attention(s, case):
    b, tq, tk, h, hk, d = _dims(case)
    scale, group = d ** -0.5, h // hk
    qlen = s["qlens"] if s["qlens"] is not None else torch.full((b,), tq, device=DEVICE)
    klen = s["klens"] if s["klens"] is not None else torch.full((b,), tk, device=DEVICE)
    i, j = torch.arange(tq, device=DEVICE), torch.arange(tk, device=DEVICE)
    inq, ink = i < qlen[:, None], j < klen[:, None]
    seen = inq[:, :, None] & ink[:, None, :]
    if case["causal"]:
        # the last query stands at the last key; a query sees its own block of keys and those before it
        at = i + (klen - qlen)[:, None]
        end = (torch.div(at, case["causal"], rounding_mode="floor") + 1) * case["causal"]
        seen = seen & (j < end[:, :, None])
    seen = seen[:, None]

    def heads(x, valid, repeat):  # [b, h, t, d] in 32 bits, padded rows as zeros
        x = torch.where(valid[:, :, None, None], x.float(), 0.0).permute(0, 2, 1, 3)
        return x.repeat_interleave(repeat, 1)

    q, k, v = heads(s["q"], inq, 1), heads(s["k"], ink, group), heads(s["v"], ink, group)
    logits = (q @ k.transpose(2, 3)) * scale
    logits = torch.where(seen, logits, -math.inf)
    top = logits.amax(3, keepdim=True)
    p = torch.exp(logits - torch.where(top == -math.inf, 0.0, top))
    del logits
    total = p.sum(3, keepdim=True)
    lse = (torch.log(total) + top).squeeze(3)
    p = p / torch.where(total == 0, 1.0, total)
    out = p @ v
    result = {"out": out.permute(0, 2, 1, 3).to(s["q"].dtype), "lse": lse}
    if not case["step"]:
        return result
    dout = heads(s["dout"], inq, 1)
    dv = p.transpose(2, 3) @ dout
    dp = dout @ v.transpose(2, 3)
    ds = p * (dp - (dout * out).sum(3, keepdim=True)) * scale
    del dp, p
    dq, dk = ds @ k, ds.transpose(2, 3) @ q

    def shared(x):  # the sum over the query heads of a key head
        return x.view(b, hk, group, tk, d).sum(2).permute(0, 2, 1, 3).to(s["q"].dtype)

    result.update(dq=dq.permute(0, 2, 1, 3).to(s["q"].dtype), dk=shared(dk), dv=shared(dv))
    return result


def _plain_adamw(s, case):
    s["step"] += 1
    t, slot = s["step"], s["slot"]
    p, g = s["flat"], torch.zeros_like(s["m"], dtype=torch.float32)
    g[slot] = s["grad"].float()
    if case["bits"] == 8:
        m = (s["m"].view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        v = (s["v"].view(-1, BLOCK) * s["v_scale"][:, None]).view(-1)
        v = v * v
    else:
        m, v = s["m"], s["v"]
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    step = (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + ADAM_EPS)
    p.copy_(torch.where(s["decays"], p * (1 - LR * DECAY), p) - LR * step[slot])
    if case["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return {"p": p, "m": m, "v": v}
    # 8 bits: the moment and the second moment's root as multiples of their block's largest, rounded up where the
    # fraction passes a threshold that steps through [0, 1) with the place and the step
    place = torch.arange(m.numel(), device=DEVICE)
    u = (((place * 0x85EBCA6B + t * 0x9E3779B9) & 0xFFFFFFFF) >> 8).float() * 2.0 ** -24

    def coded(x, levels, low):
        top = x.abs().view(-1, BLOCK).amax(1)
        scale = torch.where(top < 2.0 ** -100, 0.0, top * (1 / levels))
        inv = torch.where(scale == 0, 0.0, scale.reciprocal())
        code = torch.floor((x.view(-1, BLOCK) * inv[:, None]) + u.view(-1, BLOCK))
        return code.clamp(low, levels), scale

    mc, s["m_scale"] = coded(m, 127, -127)
    r = v.sqrt()
    rc, s["v_scale"] = coded(r, 255, 0)
    # a second moment that is not zero does not become zero
    rc = torch.where((r.view(-1, BLOCK) > 0) & (s["v_scale"][:, None] > 0), rc.clamp_min(1), rc)
    s["m"].copy_(mc.view(-1))
    s["v"].copy_(rc.view(-1))
    root = rc * s["v_scale"][:, None]
    return {"p": p, "m": (mc * s["m_scale"][:, None]).view(-1), "v": (root * root).view(-1)}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def _pairs(case):
    """Expected (query, key) pairs of an attention case."""
    b, tq, tk, h, hk, d = _dims(case)
    if case["ragged"]:
        # lengths are full for the first sequence, else uniform in [0.2, 1] of the batch's
        mean = (1 + (b - 1) * (1 - 0.2 ** 3) / (3 * 0.8)) / b
    else:
        mean = 1.0
    full = b * h * tq * tk * mean
    if not case["causal"]:
        return full
    block = min(case["causal"], tk)
    unseen = max(0, min(tq, tk) - block) / 2 * min(tq, tk)
    return full * (1 - unseen / (tq * tk))


def work(case):
    size = 2 if case.get("dtype") == "bf16" else 4
    if case["op"] == "norm":
        n = case["rows"] * case["c"]
        if case["step"]:
            return {"bytes": 5 * n * size + 16 * case["c"], "flops": 20 * n}  # x, dy; y, dx, and x's second reading
        return {"bytes": 2 * n * size + 8 * case["c"], "flops": 8 * n}
    if case["op"] == "rotary":
        n = case["b"] * case["t"] * (case["h"] + case["hk"]) * case["d"]
        return {"bytes": 2 * n * size + 4 * case["axes"] * case["b"] * case["t"], "flops": 3 * n}
    if case["op"] == "attention":
        b, tq, tk, h, hk, d = _dims(case)
        rows, keys = b * tq * h * d * size, b * tk * hk * d * size
        if case["step"]:  # q, k, v, dout; out, lse, dq, dk, dv
            return {"bytes": 4 * rows + 4 * keys + 4 * b * h * tq, "flops": 14 * _pairs(case) * d}
        return {"bytes": 2 * rows + 2 * keys + 4 * b * h * tq, "flops": 4 * _pairs(case) * d}
    n = sum(math.prod(x) for x in _shapes(case))
    grad = 2 if case["grad"] == "bf16" else 4
    # parameters in and out, gradients, the moments in and out, and in 8 bits the values they stand for
    moments = 16 * n if case["bits"] == 32 else 4 * n + 8 * n
    return {"bytes": (8 + grad) * n + moments, "flops": 15 * n}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    global own
    was, own = own, False  # the inputs alone
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"norm": _exact_norm, "rotary": _exact_rotary, "attention": _exact_attention,
            "adamw": _exact_adamw}[case["op"]](s, case)


def _exact_norm(s, case):
    x, w = s["x"].double(), s["weight"].double()
    var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
    sigma = (var + EPS).sqrt()
    xhat = (x - mean) / sigma
    y = xhat * w + s["bias"].double()
    if not case["step"]:
        return {"y": y}
    dy = s["dy"].double()
    # dx = (I - 1 1'/c - xhat xhat'/c) (w dy) / sigma
    g, c = dy * w, case["c"]
    along = torch.einsum("rc,rc->r", g, xhat)[:, None] / c
    dx = (g - g.sum(1, keepdim=True) / c - along * xhat) / sigma
    return {"y": y, "dx": dx, "dw": torch.einsum("rc,rc->c", dy, xhat), "db": dy.sum(0)}


def _exact_rotary(s, case):
    angles = []
    for a, n in enumerate(s["sections"]):
        for p in range(n):
            angles.append(s["positions"][a].double() * BASE ** (-p / n))
    phase = torch.polar(torch.ones_like(angles[0])[..., None].expand(-1, -1, len(angles)).contiguous(),
                        torch.stack(angles, -1))
    if case["inverse"]:
        phase = phase.conj()

    def turn(x):
        x = x.double()
        half = x.shape[-1] // 2
        pairs = x.unflatten(-1, (half, 2)) if case["interleaved"] else x.unflatten(-1, (2, half)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * phase[:, :, None])
        return (z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2)

    return {"q": turn(s["q"]), "k": turn(s["k"])}


def _exact_attention(s, case):
    b, tq, tk, h, hk, d = _dims(case)
    group, block = h // hk, case["causal"]
    like = {"dtype": torch.float64, "device": DEVICE}
    out, lse = torch.zeros(b, tq, h, d, **like), torch.full((b, h, tq), -math.inf, **like)
    dq, dk, dv = torch.zeros(b, tq, h, d, **like), torch.zeros(b, tk, hk, d, **like), torch.zeros(b, tk, hk, d, **like)
    for n in range(b):
        nq = tq if s["qlens"] is None else int(s["qlens"][n])
        nk = tk if s["klens"] is None else int(s["klens"][n])
        ends = torch.full((nq,), nk, device=DEVICE)
        if block:
            place = torch.arange(nk - nq, nk, device=DEVICE)
            ends = ((place - place % block) + block).clamp(0, nk)
        hidden = torch.arange(nk, device=DEVICE)[None] >= ends[:, None]
        empty = (ends == 0)[:, None]
        for m in range(h):
            q, k, v = s["q"][n, :nq, m].double(), s["k"][n, :nk, m // group].double(), s["v"][n, :nk, m // group].double()
            logits = torch.einsum("id,jd->ij", q, k) / math.sqrt(d)
            logits.masked_fill_(hidden, -math.inf)
            z = torch.logsumexp(logits, 1, keepdim=True)
            lse[n, m, :nq] = z[:, 0]
            p = torch.exp(logits - z.masked_fill(empty, 0.0))
            out[n, :nq, m] = p @ v
            if case["step"]:
                do = s["dout"][n, :nq, m].double()
                dp = torch.einsum("id,jd->ij", do, v)
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(d)
                dq[n, :nq, m] = ds @ k
                dk[n, :nk, m // group] += ds.t() @ q
                dv[n, :nk, m // group] += p.t() @ do
    if not case["step"]:
        return {"out": out, "lse": lse}
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _exact_adamw(s, case):
    t, slot = START_STEP + 1, s["slot"]
    m, v, g = s["m"].double(), s["v"].double(), s["grad"].double()
    if case["bits"] == 8:
        block = torch.arange(m.numel(), device=DEVICE) // BLOCK
        m, v = m * s["m_scale"].double()[block], (v * s["v_scale"].double()[block]) ** 2
    m1 = BETA1 * m
    v1 = BETA2 * v
    m1[slot] += (1 - BETA1) * g
    v1[slot] += (1 - BETA2) * g ** 2
    p = s["flat"].double()
    p = p - LR * DECAY * p * s["decays"] - LR * (m1[slot] / (1 - BETA1 ** t)) / (torch.sqrt(v1[slot] / (1 - BETA2 ** t)) + ADAM_EPS)
    if case["bits"] == 8:
        # a value next to a threshold goes to either code by its last bit: the codes have no value of their own in 64 bits
        return {"p": p, "m": None, "v": None}
    return {"p": p, "m": m1, "v": v1}
