"""The training operators' definitions in 64 bits, for the tests (torch float64 on the inputs' device)."""
import math

import torch

CODE_MAX = {False: 480.0, True: 496.0}


def attention(q, k, v, tq, tr, tz, mask, bq, br, bz, scale=None):
    """(out, p) of the definition, differentiable in float64; masked tokens are cleared first."""
    nq, d = q.shape[1], q.shape[3]
    live = mask.bool()
    rows = live[:, :nq]

    def clear(t, keep):
        return torch.where(keep[:, :, None, None], t, torch.zeros((), dtype=t.dtype, device=t.device))

    q, k, v = clear(q, rows), clear(k, live), clear(v, live)
    s = torch.einsum("bihd,bjhd->bhij", q, k) * (d ** -0.5 if scale is None else scale)
    for t, table in ((tq, bq), (tr, br), (tz, bz)):
        c = table.shape[0] // 2
        t = t.long().clamp(-(1 << 19), 1 << 19)
        index = (t[:, None, :] - t[:, :nq, None]).clamp(-c, c) + c
        s = s + table[index].permute(0, 3, 1, 2)
    keep = rows[:, None, :, None] & live[:, None, None, :]
    s = torch.where(keep, s, torch.full((), -math.inf, dtype=s.dtype, device=s.device))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top.isfinite(), top, torch.zeros_like(top)))
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
    return torch.einsum("bhij,bjhd->bihd", p, v), p


def attention_grads(dout, q, k, v, tq, tr, tz, mask, bq, br, bz, scale=None):
    """out and the gradients by the formulas, all float64."""
    q, k, v, dout, bq, br, bz = (t.double() for t in (q, k, v, dout, bq, br, bz))
    nq, d = q.shape[1], q.shape[3]
    scale = d ** -0.5 if scale is None else scale
    live = mask.bool()
    out, p = attention(q, k, v, tq, tr, tz, mask, bq, br, bz, scale)
    zero = torch.zeros((), dtype=torch.float64, device=q.device)
    q = torch.where(live[:, :nq, None, None], q, zero)
    k, v = (torch.where(live[:, :, None, None], t, zero) for t in (k, v))
    dout = torch.where(live[:, :nq, None, None], dout, zero)
    dp = torch.einsum("bihd,bjhd->bhij", dout, v)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq, dk = torch.einsum("bhij,bjhd->bihd", ds, k) * scale, torch.einsum("bhij,bihd->bjhd", ds, q) * scale
    dv = torch.einsum("bhij,bihd->bjhd", p, dout)
    tables = []
    for t, table in ((tq, bq), (tr, br), (tz, bz)):
        c = table.shape[0] // 2
        t = t.long().clamp(-(1 << 19), 1 << 19)
        index = (t[:, None, :] - t[:, :nq, None]).clamp(-c, c) + c
        tables.append(torch.stack([(ds * (index == x)[:, None]).sum((0, 2, 3)) for x in range(2 * c + 1)]))
    return [out, dq, dk, dv, *tables]


def norm(x, w, b, eps, dy, dsum=None):
    """y and (dx, dw, db) by the formulas, float64; x is what is normalised."""
    x, w, b, dy = x.double(), w.double(), b.double(), dy.double()
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    hat = (x - mean) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - hat * (g * hat).mean(-1, keepdim=True))
    lead = tuple(range(x.dim() - 1))
    if dsum is not None:
        dx = dx + dsum.double()
    return [hat * w + b, dx, (dy * hat).sum(lead), dy.sum(lead)]


def adamw(p, g, m, v, step, lr, betas, eps, wd):
    """(p, m, v) after a step, float64."""
    p, g, m, v = (t.double() for t in (p, g, m, v))
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    return (1 - lr * wd) * p - lr * (m / (1 - betas[0] ** step)) / ((v / (1 - betas[1] ** step)).sqrt() + eps), m, v


def code_values(second):
    """The 256 values (times scale) that 8-bit codes stand for: float64."""
    c = torch.arange(256)
    bits = 4 if second else 3
    mag = c if second else c & 127
    e, f = mag >> bits, (mag & ((1 << bits) - 1)).double() / (1 << bits)
    y = torch.where(e > 0, (1 + f) * torch.pow(2.0, (e - 7).double()), f * 2.0 ** -6)
    return y if second else torch.where(c > 127, -y, y)
