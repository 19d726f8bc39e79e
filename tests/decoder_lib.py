"""Layer norm, 8-bit dense layers and drawn labels in float64, with bounds on how far a
float32-accumulating kernel may be from them (heads_lib has the dense layers' own).

Bounds, elementwise, from the arithmetic (u = 2^-24, half a float32 step; n = additions in the longest chain
that a kernel makes of a row's sum, at most K / 16 + 40):

* the mean as rounded is off by e0 <= n u mean|x|, and is corrected by the mean of what is left, so d = x - mean
  is off by 3 u |d| + (n + 4) u (sd + e0), sd the row's spread; the sum of d^2 by (2 n + 8) u relative, so
  1 / sqrt(var + eps) by (n + 8) u, and h = d / sqrt(var + eps) by
  bh = (n + 12) u (|h| + (sd + e0) r) ;
* y = h w + b: |w| bh + 2 u (|h w| + |b|), and the last rounding;
* dx = r (g - mean g - h mean(g h)): the means are off by (n + 4) u of the mean magnitudes, and the last also by
  mean(|g| bh); r by (n + 8) u; h by bh;
* dw = sum dy h and db = sum dy: a chain of at most M / 148 + 1300 additions (rows over blocks, then blocks).

8-bit rows: scale and q are the definition's own, bit for bit; the sum is exact, made a float (u) and
scaled by a rounded product of scales (2 u); then as the dense layer's epilogue.
"""
import math

import torch

import heads_lib as hl

U = 2.0 ** -24


def last(dt, v):
    """The final rounding of a result of magnitude v."""
    return (torch.finfo(dt).eps / 2) * v + (2.0 ** -25 if dt == torch.float16 else 0.0)


def layer_norm(x, w, b, eps, dy=None):
    """[(value, bound)]: y, then dx, dweight, dbias when dy is given."""
    dt = x.dtype
    x = x.double()
    M, K = x.shape
    one = torch.ones(K, dtype=torch.float64, device=x.device)
    wd = one if w is None else w.double()
    bd = 0 * one if b is None else b.double()
    n = K / 16 + 40
    mean = x.mean(1, keepdim=True)
    d = x - mean
    var = (d * d).mean(1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    h = d * r
    e0 = n * U * x.abs().mean(1, keepdim=True)
    bh = (n + 12) * U * (h.abs() + (var.sqrt() + e0) * r)
    y = h * wd + bd
    by = wd.abs() * bh + 2 * U * ((h * wd).abs() + bd.abs())
    out = [(y, by + last(dt, y.abs() + by))]
    if dy is None:
        return out
    dy = dy.double()
    g = dy * wd
    mg, mgh = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx = r * (g - mg - h * mgh)
    bm = (n + 4) * U * g.abs().mean(1, keepdim=True)
    bmh = (g.abs() * bh).mean(1, keepdim=True) + (n + 4) * U * (g * h).abs().mean(1, keepdim=True)
    size = g.abs() + mg.abs() + (h * mgh).abs()
    bx = r * (3 * U * size + bm + h.abs() * bmh + bh * (mgh.abs() + bmh)) + (n + 8) * U * r * size
    out.append((dx, bx + last(dt, dx.abs() + bx)))
    m = M / 148 + 1300
    for v, e, mag in (((dy * h).sum(0), (dy.abs() * bh).sum(0), (dy * h).abs().sum(0)),
                      (dy.sum(0), 0, dy.abs().sum(0))):
        bv = e + min(m, M + 40) * U * mag
        out.append((v, bv + last(dt, v.abs() + bv)))
    return out


def quantize(x):
    """(q, scale): the definition."""
    x = x.double()
    top = x.abs().amax(1)
    bad = ~torch.isfinite(top)
    scale = torch.where(bad, torch.full_like(top, math.nan), (top / 127)).float()
    s = scale.double()
    ok = (s > 0) & ~bad
    q = torch.where(ok[:, None], torch.round(x / torch.where(ok, s, torch.ones_like(s))[:, None]), torch.zeros_like(x))
    return q.clamp(-127, 127).to(torch.int8), scale


def linear_act_int8(q, xs, p, ws, b, r, act, dt):
    """(value, bound) of act(xs ws sum q p + b) + r."""
    z = (q.double() @ p.double().t()) * xs.double()[:, None] * ws.double()[None, :]
    dz = 4 * U * z.abs()
    if b is not None:
        z = z + b.double()
        dz = dz + U * z.abs()
    y, _ = hl.act64(act, z)
    by = 1.13 * dz + (32 if dt == torch.float32 else 64) * hl.E * y.abs() + 1e-7
    if r is not None:
        y = y + r.double()
        by = by + U * (y.abs() + r.double().abs())
    return y, by + last(dt, y.abs() + by)


def sample(z, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The labels, row by row, by the definition."""
    z = z.double().cpu()
    M, V = z.shape
    get = [v.tolist() if torch.is_tensor(v) else [v] * M for v in (temperature, top_k, top_p, min_p, u)]
    out = []
    for m, (t, k, p, q, uu) in enumerate(zip(*get)):
        row = z[m]
        best = float(row.max())
        if torch.isnan(row).any() or t != t or best == -math.inf:
            out.append(-1)
            continue
        if not t > 0:
            out.append(int(torch.nonzero(row == best)[0]))
            continue
        w = torch.where(row == best, torch.ones(()).double(), torch.exp((row - best) / t))
        w = torch.where(torch.isneginf(row), torch.zeros(()).double(), w)
        order = torch.sort(row, descending=True, stable=True).indices
        if k > 0:
            order = order[:k]
        ws = w[order]
        if p < 1:
            before = ws.cumsum(0) - ws
            n = max(1, int((before < p * ws.sum()).sum()))
            order, ws = order[:n], ws[:n]
        order = order[(ws >= q) | (row[order] == best)]
        order = torch.sort(order).values
        order = order[w[order] > 0]
        run = w[order].cumsum(0)
        at = int((run <= uu * run[-1]).sum())
        out.append(int(order[min(at, len(order) - 1)]))
    return torch.tensor(out)
