"""Plain float64 forms of the training operators (net_ops.py), with how far a correct f32 computation of
each output may be from them.  u is f32's half step; k counts the additions behind one sum; a result rounded
to its type is off by half a step of it more (and half the type's least value)."""
import math

import torch

U = 2.0 ** -24


def half_step(t, dtype):
    return t.abs() * (torch.finfo(dtype).eps / 2) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def off(got, want, tol):
    """The largest share of its tolerance that a value of `got` takes; inf where one is not finite that should
    be, or the other way round."""
    got = got.double()
    same = (got == want) | (got.isnan() & want.isnan())
    r = torch.where(same, 0.0, (got - want).abs() / tol)
    return float(torch.nan_to_num(r, nan=float("inf")).max()) if r.numel() else 0.0


def norm(x, w, b, eps, dh=None, dres=None, dtype=None):
    """x [rows, d] float64 (already the sum), w / b / dh / dres float64 or None -> {name: (value, tolerance)}."""
    dtype = dtype or torch.float32
    rows, d = x.shape
    k = d / 64 + 16
    mu = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps)
    n = (x - mu) * r
    big = x.abs().mean(-1, keepdim=True)
    # n: the mean is off by k u big, r by (k + 4) u relative (and by the mean's square, of second order)
    dn = U * ((k + 2) * (r * big) + (k + 8) * n.abs()) + (U * (k + 2) * r * big) ** 2 * n.abs()
    ww = w if w is not None else torch.ones(d, dtype=torch.float64, device=x.device)
    bb = b if b is not None else torch.zeros(d, dtype=torch.float64, device=x.device)
    y = n * ww + bb
    out = {"h": (y, half_step(y, dtype) + ww.abs() * dn + 2 * U * ((n * ww).abs() + bb.abs()))}
    if dh is None:
        return out
    g = dh * ww
    a, c = g.mean(-1, keepdim=True), (g * n).mean(-1, keepdim=True)
    ga, gn = g.abs().mean(-1, keepdim=True), (g * n).abs().mean(-1, keepdim=True)
    dx = r * (g - a - n * c)
    dc = U * (k + 4) * gn + (g.abs() * dn).mean(-1, keepdim=True)
    tol = r * (U * (k + 8) * (g.abs() + ga + n.abs() * gn) + dn * c.abs() + n.abs() * dc) + U * (k + 8) * r * (g - a - n * c).abs()
    if dres is not None:
        dx = dx + dres
        tol = tol + 2 * U * (dx.abs() + dres.abs())
    out["dx"] = (dx, half_step(dx, dtype) + tol)
    kr = rows / 16 + 64
    out["dw"] = ((dh * n).sum(0), U * kr * (dh * n).abs().sum(0) + (dh.abs() * dn).sum(0))
    out["db"] = (dh.sum(0), U * kr * dh.abs().sum(0))
    return out


def logp(logits, tokens, mask, temperature, dlogp=None, dent=None, dtype=torch.float32):
    """logits [rows, vocab] float64, tokens [rows, n] int64, mask bool or None -> ({name: (value, tolerance)},
    every entry's log probability, the tolerance of log sum e^z)."""
    rows, vocab = logits.shape
    z = logits / temperature
    if mask is not None:
        z = torch.where(mask, z, -torch.inf)
    m = z.amax(-1, keepdim=True)
    empty = m == -torch.inf
    m0 = torch.where(empty, 0.0, m)
    e = torch.exp(z - m0)
    s = e.sum(-1, keepdim=True)
    lse = m + torch.log(s)
    lp = torch.where(empty, -torch.inf, z - lse)
    p = torch.where(empty, 0.0, e / s)
    fin = torch.where(z == -torch.inf, 0.0, lp)
    ent = -(p * fin).sum(-1, keepdim=True)
    lv = math.log(vocab) + 1
    # S: k additions; every exponential's argument is off by 4 u of |z| (1 / T, the product, the difference, the base)
    zz = torch.where(torch.isfinite(z), z.abs(), 0.0)
    k = vocab / 64 + 32
    spread = (p * torch.where(z == -torch.inf, 0.0, m0 - z)).sum(-1, keepdim=True)
    tl = U * (k + 8 * (m0.abs() + lse.abs().nan_to_num(posinf=0.0) + spread + lv))
    pad, over = tokens < 0, tokens >= vocab
    t = tokens.clamp(0, vocab - 1)
    given = lp.gather(1, t)
    given = torch.where(over, torch.nan, torch.where(pad, 0.0, given))
    out = {"logprobs": (given, tl + 8 * U * (zz.gather(1, t) + given.abs().nan_to_num(posinf=0.0) + 1)),
           "entropy": (ent[:, 0], (tl * (ent + lv) + U * (k + 8) * (ent + spread + lv) + 8 * U * (m0.abs() + 1))[:, 0])}
    if dlogp is None and dent is None:
        return out, lp, tl
    g = torch.zeros_like(given) if dlogp is None else torch.where(pad | over | (z.gather(1, t) == -torch.inf), 0.0, dlogp)
    ge = torch.zeros_like(ent) if dent is None else dent[:, None]
    total = g.sum(-1, keepdim=True)
    d = -p * (total + ge * (fin + ent))
    spent = p * (g.abs().sum(-1, keepdim=True) + ge.abs() * (fin.abs() + ent))
    for i in range(tokens.shape[1]):
        d.scatter_add_(1, t[:, i:i + 1], g[:, i:i + 1])
        spent.scatter_add_(1, t[:, i:i + 1], g[:, i:i + 1].abs())
    rel = tl + U * (8 * zz + 80)
    tol = spent * rel + p * ge.abs() * (out["entropy"][1][:, None] + rel * (1 + fin.abs()))
    out["dlogits"] = (d / temperature, half_step(d / temperature, dtype) + (tol + 4 * U * d.abs()) / temperature)
    return out, lp, tl


def adamw(p, g, m, v, t, lr, betas, eps, wd):
    """One step in float64 -> (p, m, v) and the f32 tolerances of each."""
    b1, b2 = betas
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    size, root = lr / (1 - b1 ** t), (1 - b2 ** t) ** 0.5
    den = v1.sqrt() / root + eps
    upd = size * m1 / den
    tm = 6 * U * (b1 * m.abs() + (1 - b1) * g.abs()) + 2.0 ** -149
    tv = 6 * U * v1 + 2.0 ** -148
    # sqrt(v) inherits half of v's relative error; below f32's least normal its absolute one
    p1 = p * (1 - lr * wd) - upd
    tp = 4 * U * p.abs() + size * tm / den + 24 * U * upd.abs()
    return (p1, m1, v1), (tp, tm, tv)
