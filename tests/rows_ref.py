"""The row operators' definitions in plain torch: the parts that are fixed to the bit (the fold, the
checkpoint) in 32 bits, the rest in 64, and how far a 32-bit computation may be from that.

U is half a step of a 32-bit float at 1. The bounds count roundings on the longest path of the
computation: a row's sum adds 8 elements of a vector, at most 16 vectors of a lane and 64 partial sums
across lanes, so its error is under 96 U times the sum of magnitudes; 128 U covers the few operations
around it."""
import math

import torch

U = 2.0 ** -24
BLOCK = 128
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SMALLEST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def half_step(t, v):
    """How far rounding v (64 bits) to type t moves it at most."""
    return v.abs() * (torch.finfo(t).eps / 2) + SMALLEST[t] / 2


def fold(ts, residual=None):
    s = ts[0].float()
    for t in ts[1:]:
        s = s + t.float()
    if residual is not None:
        s = s + residual.float()
    return s.to(ts[0].dtype)


def save8(x):
    """(q, scale) of a matrix, bit for bit."""
    rows, cols = x.shape
    nb = -(-cols // BLOCK)
    t = torch.zeros(rows, nb * BLOCK, device=x.device)
    t[:, :cols] = x.float()
    t = t.view(rows, nb, BLOCK)
    a = t.abs().amax(2, keepdim=True)
    finite = torch.isfinite(a)
    a = a.clamp_min(2.0 ** -100)
    q = torch.where(finite, torch.round(t * (torch.full_like(a, 127.0) / a)), torch.zeros_like(t)).to(torch.int8)
    scale = torch.where(finite, a * torch.tensor(1.0 / 127.0, dtype=torch.float32, device=x.device), torch.full_like(a, math.nan))
    return q.view(rows, nb * BLOCK)[:, :cols].contiguous(), scale[:, :, 0].contiguous()


def restore8(q, scale):
    cols = q.shape[1]
    return q.float() * scale.repeat_interleave(BLOCK, 1)[:, :cols]


def layernorm(x, w, b, eps):
    """x: the rounded rows. (mean, rstd, y, bound of y before its rounding) in 64 bits."""
    x = x.double()
    n = x.shape[1]
    mean = x.mean(1, keepdim=True)
    rstd = (((x - mean) ** 2).sum(1, keepdim=True) / n + eps).rsqrt()
    xh = (x - mean) * rstd
    w = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(n, dtype=torch.float64, device=x.device) if b is None else b.double()
    y = xh * w + b
    big = x.abs().amax(1, keepdim=True)
    return mean[:, 0], rstd[:, 0], y, 128 * U * (w.abs() * (xh.abs() + rstd * big) + b.abs() + y.abs())


def stats_bounds(x, rstd):
    """How far mean and rstd (as a share) may be off."""
    big = x.double().abs().amax(1)
    return 128 * U * big, 128 * U * (1 + rstd * big)


def layernorm_grad(g, x, mean, rstd, w, dsum, exh=None):
    """In 64 bits, from 32-bit statistics: dx, dw, db and their bounds before they are rounded."""
    g, x, mean, rstd = g.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    n, rows = x.shape[1], x.shape[0]
    w = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w.double()
    xh = (x - mean) * rstd
    if exh is None:  # of xh itself; or `exh` times its size
        exh = 3 * U * (xh.abs() + rstd * (x.abs() + mean.abs()))
    else:
        exh = exh * xh.abs()
    gw = g * w
    c1, c2 = gw.mean(1, keepdim=True), (gw * xh).mean(1, keepdim=True)
    dx = rstd * (gw - c1 - xh * c2)
    e1 = 128 * U * gw.abs().mean(1, keepdim=True)
    e2 = 128 * U * (gw * xh).abs().mean(1, keepdim=True) + (gw.abs() * exh).mean(1, keepdim=True)
    ex = rstd * (8 * U * (gw.abs() + c1.abs() + (xh * c2).abs()) + e1 + xh.abs() * e2 + exh * c2.abs())
    if dsum is not None:
        dx = dx + dsum.double()
        ex = ex + 2 * U * (dx.abs() + dsum.double().abs())
    # a column's sum: rows / 16 terms in a lane at the most (16 rows side by side in one workgroup), then
    # 15 of those, then a 32nd of up to 1280 partial rows and 32 of their sums: 87, and 155 are counted
    depth = (-(-rows // 16) + 15 + 128 + 8 + 4) * U
    return dx, ex, (g * xh).sum(0), depth * (g * xh).abs().sum(0) + (g.abs() * exh).sum(0), g.sum(0), depth * g.abs().sum(0)


K = math.sqrt(2 / math.pi)


def act(kind, a):
    """value, slope and their bounds as 32-bit results, in 64 bits. The exponential's argument is off by
    2 U of itself, which the exponential turns into that many times its argument; the other operations
    are counted with 40 U. An exponential under 2^-126, the smallest normal 32-bit number, is zero in the
    hardware, and one over 2^128 infinite, so that its reciprocal is: either moves a probability by less
    than 2^-126, the value by |a| times that and the slope by 1 + |a| times."""
    a = a.double()
    flush = 2.0 ** -126 * (1 + a.abs())
    if kind == "silu":
        s = torch.sigmoid(a)
        value, slope, bv, bs = a * s, s + a * s * torch.sigmoid(-a), (a * s).abs(), s * (1 + a.abs())
        m = U * (40 + 4 * a.abs())
    elif kind == "gelu":
        p, e = torch.erfc(-a * math.sqrt(0.5)) / 2, torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)  # no cancellation in the tail
        value, slope, bv, bs = a * p, p + a * e, (a * p).abs(), p + a.abs() * e
        m = U * (40 + 4 * a * a)
    else:
        u = 2 * K * (a + 0.044715 * a ** 3)
        d = 2 * K * (1 + 3 * 0.044715 * a * a)
        s = torch.sigmoid(u)
        value, slope, bv, bs = a * s, s + a * s * torch.sigmoid(-u) * d, (a * s).abs(), s * (1 + a.abs() * d * (torch.sigmoid(-u) + U))
        m = U * (40 + 8 * u.abs())
        flush = flush * (1 + d)
    return value, slope, m * bv + flush, m * bs + flush


def close(got, want, bound, t=None):
    """got within `bound` of want, and half a step of got's type where it was rounded to it."""
    w = want.double()
    lim = bound + (half_step(got.dtype, w.abs() + bound) if t is None else 0)
    off = (got.double() - w).abs()
    bad = ~(off <= lim)
    if bool(bad.any()):
        k = int(torch.argmax((off / lim).nan_to_num(posinf=1e300, nan=1e300)))
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} outside: at {k} got {float(got.reshape(-1)[k])}, "
                             f"want {float(w.reshape(-1)[k])} +- {float(lim.reshape(-1)[k])}")
