"""Plain 64-bit implementations of the token operators and of the AdamW step, with bounds on what rounding can do.

u: half a step of the storage type, relative (bf16 2^-8, float32 2^-24); e = 2^-24: half a step of the 32-bit
arithmetic. A sum of n products in 32 bits, in any order, is off by at most about n e times the sum of their absolute
values; a few more e cover the operations around it.
"""
import math

import torch

E32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def norm(x, w, b, eps):
    """(y, mean, rstd, tolerance of y)."""
    u, c = half_step(x.dtype), x.shape[-1]
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    rstd = (d.square().mean(-1, keepdim=True) + eps).rsqrt()
    h = d * rstd
    wd = torch.ones(c, dtype=torch.float64, device=x.device) if w is None else w.double()
    y = h * wd + (0 if b is None else b.double())
    # the mean is off by n e of the mean of |x|, the distances by that and e of themselves, the deviation by n e
    n = c + 8
    off = n * E32 * x.abs().mean(-1, keepdim=True) * rstd
    ty = u * y.abs() + wd.abs() * (off * (1 + h.abs()) + (n + 8) * E32 * h.abs()) + 2 * E32 * y.abs()
    return y, mean.squeeze(-1), rstd.squeeze(-1), ty


def norm_backward(dy, x, w, eps):
    """((dx, dw, db), (their tolerances))."""
    u, c = half_step(x.dtype), x.shape[-1]
    _, mean, rstd, _ = norm(x, None, None, eps)
    dy, x = dy.double(), x.double()
    r = rstd[..., None]
    h = (x - mean[..., None]) * r
    g = dy if w is None else dy * w.double()
    gm, hm = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    dx = r * (g - gm - h * hm)
    n = c + 16
    # error of xhat: relative 2n e and an offset from the mean's error
    eh = 2 * n * E32 * h.abs() + n * E32 * x.abs().mean(-1, keepdim=True) * r
    ehm = (g.abs() * eh).mean(-1, keepdim=True) + n * E32 * (g * h).abs().mean(-1, keepdim=True)
    tx = u * dx.abs() + r * (n * E32 * g.abs().mean(-1, keepdim=True) + eh * hm.abs() + h.abs() * ehm) + \
        2 * n * E32 * r * (g.abs() + gm.abs() + (h * hm).abs())
    rows = dy.numel() // c
    flat = lambda t: t.reshape(rows, c)  # noqa: E731
    dw, db = flat(dy * h).sum(0), flat(dy).sum(0)
    tw = flat(dy.abs() * eh).sum(0) + (rows + 4) * E32 * flat((dy * h).abs()).sum(0)
    tb = (rows + 4) * E32 * flat(dy.abs()).sum(0)
    return (dx, dw, db), (tx, tw, tb)


def rotate(x, positions, turns, axis, interleaved, inverse):
    """(y, tolerance): x [b, t, h, d], positions [axes, b, t]."""
    u, xd, pairs = half_step(x.dtype), x.double(), turns.numel()
    angle = positions.double()[axis.long()].permute(1, 2, 0) * turns.double() * (2 * math.pi)
    c, s = angle.cos()[:, :, None], angle.sin()[:, :, None]
    if inverse:
        s = -s
    y = xd.clone()
    first, second = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    a, b = xd[..., first], xd[..., second]
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    tol = u * y.abs()
    # the turn is rounded to 32 bits (half of 2^-25 of a turn), sine and cosine to 2 steps, two products and a sum
    reach = (a.abs() + b.abs()) * (2 * math.pi * 2.0 ** -25 + 8 * E32)
    tol[..., first] += reach
    tol[..., second] += reach
    return y, tol


def seen(b, tq, tk, block, qlens, klens, device):
    """[b, tq, tk]: which keys a query sees."""
    i, j = torch.arange(tq, device=device), torch.arange(tk, device=device)
    out = torch.zeros(b, tq, tk, dtype=torch.bool, device=device)
    for n in range(b):
        nq = tq if qlens is None else min(max(int(qlens[n]), 0), tq)
        nk = tk if klens is None else min(max(int(klens[n]), 0), tk)
        m = (i < nq)[:, None] & (j < nk)[None]
        if block:
            m &= (j // block)[None] <= torch.div(i + nk - nq, block, rounding_mode="floor")[:, None]
        out[n] = m
    return out


def attention(q, k, v, scale, block, qlens, klens, dout=None, out=None, coarse=None):
    """Results and tolerances as dicts. `coarse`: half a step of the type the probabilities are rounded to before
    their products (default: the storage type's), `out`: the stored output the backward pass reads."""
    (b, tq, h, d), (tk, hk) = q.shape, k.shape[1:3]
    u = half_step(q.dtype)
    up = u if coarse is None else coarse
    mask = seen(b, tq, tk, block, qlens, klens, q.device)
    rows, cols = mask.any(2), mask.any(1)
    rep = lambda t: t.repeat_interleave(h // hk, 2)  # noqa: E731
    clean = lambda t, m: torch.where(m[:, :, None, None], t.double(), 0.0)  # noqa: E731
    # keys inside the length that nothing sees stay in; padding goes out
    q64, k64, v64 = clean(q, rows), clean(k, cols), clean(v, cols)
    Q, K, V = (t.permute(0, 2, 1, 3) for t in (q64, rep(k64), rep(v64)))
    s = (Q @ K.transpose(2, 3)) * scale
    ds = (d + 6) * E32 * abs(scale) * (Q.abs() @ K.abs().transpose(2, 3)) + 4 * E32 * s.abs()
    m4 = mask[:, None]
    s = torch.where(m4, s, -math.inf)
    lse = torch.logsumexp(s, 3, keepdim=True)
    p = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse))
    worst = torch.where(m4, ds, 0.0).amax(3, keepdim=True)
    g = 2 * worst + (tk + 16) * E32  # relative error of a probability, the normaliser's included
    O = p @ V
    back = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731
    res = {"out": back(O), "lse": lse.squeeze(3)}
    tol = {"out": back(u * O.abs() + (g + up + tk * E32) * (p @ V.abs())),
           "lse": (g + 4 * E32 + E32 * torch.where(lse == -math.inf, 0.0, lse).abs()).squeeze(3)}
    if dout is None:
        return res, tol
    G = clean(dout, rows).permute(0, 2, 1, 3)
    dp = G @ V.transpose(2, 3)
    delta = (G * O).sum(3, keepdim=True)
    dS = p * (dp - delta)
    # delta is read from the stored output: off by that output's tolerance
    edelta = (G.abs() * tol["out"].permute(0, 2, 1, 3)).sum(3, keepdim=True) + (d + 4) * E32 * (G * O).abs().sum(3, keepdim=True)
    e = (2 * g + up + 8 * E32) * dS.abs() + p * (d + 4) * E32 * (G.abs() @ V.abs().transpose(2, 3)) + p * (edelta + 2 * E32 * (dp.abs() + delta.abs()))
    fold = lambda t: back(t).reshape(b, tk, hk, h // hk, d).sum(3)  # noqa: E731
    T = lambda t: t.transpose(2, 3)  # noqa: E731
    res.update(dq=back(dS @ K) * scale, dk=fold(T(dS) @ Q) * scale, dv=fold(T(p) @ G))
    n = (tk + 8) * E32
    tol["dq"] = u * res["dq"].abs() + abs(scale) * back((e + n * dS.abs()) @ K.abs())
    n = (tq * (h // hk) + 8) * E32
    tol["dk"] = u * res["dk"].abs() + abs(scale) * fold(T(e + n * dS.abs()) @ Q.abs())
    tol["dv"] = u * res["dv"].abs() + fold(T((2 * g + up + n) * p) @ G.abs())
    return res, tol


def adamw(p, g, m, v, step, lr, b1, b2, eps, wd):
    """64-bit (p, m, v) after the step that makes the count `step`."""
    p, g, m, v = (t.double() for t in (p, g, m, v))
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p * (1 - lr * wd) - lr * (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)).sqrt() + eps), m, v


def close(got, want, tol, what=""):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    assert torch.isfinite(got[~inf]).all(), f"{what}: not finite"
    over = torch.where(inf, -1.0, (got - want).abs() - tol)
    bad = over > 0
    if bad.any():
        at = int(over.argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} beyond tolerance; worst at {at}: got "
                             f"{got.flatten()[at]:.9g}, want {want.flatten()[at]:.9g}, tolerance {tol.expand_as(want).flatten()[at]:.3g}")
