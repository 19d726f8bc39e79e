"""The per-pixel heads in float64, with bounds on how far a float32-accumulating
kernel may be from them.

Bounds, elementwise, from the arithmetic (u = half a step of the element type,
torch.finfo(t).eps / 2; e = 2^-23, a truncated float32 step):

* a product of K terms, |error| <= (K + 16) e (|x| |w|^T + |b|) =: dz.  Each of the K
  additions is off by at most one step of a running sum that never exceeds the
  sum of magnitudes; the 16 covers the split of a float32 operand into three
  16-bit parts (dropped products, 3 * 2^-24) and the bias;
* act has slope at most 1.13 and act' slope at most 1 (relu's act' jumps: there an
  error of 1 is allowed where |z| <= dz); act and act' are evaluated to 32 e
  relative plus 1e-7 absolute, beside 16-bit types to 64 e (7.6e-6: gelu's polynomial is
  6.1e-6 off in float32, and act' = Q + x phi cancels, so its error counts against Q <= 1/2);
* y is rounded once: u |y|; float16 adds half its smallest step, 2^-25;
* s = dy act': act' is kept in T and the product rounded to T: 2u + u^2 relative
  (float16: 2^-25 absolute each);
* a gradient sums s times x or w: s's error times their magnitudes, plus its own
  (terms + 16) e times the sum of magnitudes, plus the last rounding;
* lse: dz at its worst column plus (V + 16) e (the sum) plus 8 e |lse|; the loss
  adds the target logit's dz;
* G = coef (p - onehot), p off by p (dz + dlse + 16 e (1 + |z - lse|)), rounded to T.
"""
import math

import torch

E = 2.0 ** -23
ACTS = ("none", "relu", "silu", "gelu", "sigmoid")


def half_step(dt):
    return 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2


def tiny(dt):
    return 2.0 ** -25 if dt == torch.float16 else 0.0


def last(dt, v):
    """The final rounding of a result of magnitude v (float32: one step)."""
    u = half_step(dt) or E
    return u * v + tiny(dt)


def act64(act, z):
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * torch.sigmoid(-z))
    if act == "gelu":
        c = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "sigmoid":
        s = torch.sigmoid(z)
        return s, s * torch.sigmoid(-z)
    return z, torch.ones_like(z)


def product(x, w, b):
    """z and its bound."""
    x, w = x.double(), w.double()
    z, mag = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    return z, (x.shape[1] + 16) * E * mag


def weighted_sum(s, ds, o, dt):
    """(s @ o, bound) for s known to ds."""
    o = o.double()
    v, mag = s @ o, (s.abs() + ds) @ o.abs()
    return v, ds @ o.abs() + (s.shape[1] + 16) * E * mag


def linear_act(x, w, b, r, act, dy=None):
    """[(value, bound)]: y, then dx, dw, db when dy is given."""
    dt = x.dtype
    z, dz = product(x, w, b)
    y, d = act64(act, z)
    rel = (32 if dt in (torch.float32, torch.float64) else 64) * E
    by = 1.13 * dz + rel * y.abs() + 1e-7
    if r is not None:
        y = y + r.double()
        by = by + E * (y.abs() + r.double().abs())
    out = [(y, by + last(dt, y.abs() + by))]
    if dy is None:
        return out
    g = dy.double()
    s = g * d
    u = half_step(dt)
    bd = dz + rel * (d.abs() if rel == 32 * E else d.abs().clamp(min=0.5)) + 1e-7
    if act == "relu":
        bd = (z.abs() <= dz).double()
    if act == "none":
        bs = torch.zeros_like(s)
    else:
        bs = g.abs() * (bd + (2 * u + u * u + 2 * E) * (d.abs() + bd) + tiny(dt)) + tiny(dt)
    for v, bv in (weighted_sum(s, bs, w, dt), weighted_sum(s.t(), bs.t(), x, dt),
                  weighted_sum(s.t(), bs.t(), torch.ones(x.shape[0], 1, device=x.device), dt)):
        out.append((v, bv + last(dt, v.abs() + bv)))
    out[3] = (out[3][0].squeeze(1), out[3][1].squeeze(1))
    return out


def linear_ce(x, w, b, t, ignore, reduction, dl=None):
    """[(value, bound)]: loss, then dx, dw, db when dl is given."""
    dt = x.dtype
    live = t != ignore
    n = int(live.sum())
    xx = torch.where(live[:, None], x.double(), torch.zeros((), dtype=torch.float64, device=x.device))
    z, dz = product(xx, w, b)
    dz = torch.where(torch.isfinite(z), dz, torch.zeros_like(dz))
    idx = torch.where(live, t, 0)[:, None]
    lse = torch.logsumexp(z, 1, keepdim=True)
    zt = z.gather(1, idx)
    V = w.shape[0]
    blse = dz.max(1, keepdim=True).values + (V + 16) * E + 8 * E * lse.abs()
    rows = torch.where(live[:, None], lse - zt, torch.zeros_like(lse)).squeeze(1)
    brows = torch.where(live[:, None], blse + dz.gather(1, idx) + 2 * E * (lse.abs() + zt.abs()),
                        torch.zeros_like(lse)).squeeze(1)
    if reduction == "none":
        out = [(rows, brows)]
    else:
        k = 1.0 if reduction == "sum" else 1.0 / max(n, 1)
        out = [(rows.sum() * k, (brows.sum() + (512 + rows.numel() / 256) * E * rows.abs().sum()) * k)]
    if dl is None:
        return out
    g = dl.double()
    if reduction == "mean":
        g = g / max(n, 1)
    g = torch.where(live, g.expand(live.shape), torch.zeros((), dtype=torch.float64, device=x.device))[:, None]
    p = torch.exp(z - lse)
    fin = torch.where(torch.isfinite(z), (z - lse).abs(), torch.zeros_like(z))
    G = p.clone()
    G.scatter_add_(1, idx, -torch.ones_like(zt))
    bG = p * (dz + blse + 16 * E * (1 + fin)) + 4 * E * G.abs()
    # rounded to T; float16 keeps G lifted by 2^14, so its smallest step is 2^-25 / 2^14
    bG = bG + half_step(dt) * (G.abs() + bG) + tiny(dt) * 2.0 ** -14
    if reduction == "none":
        # rows are scaled by a power of two at or above the largest |g|, at most twice it
        bG = bG * g.abs() + tiny(dt) * 2.0 ** -14 * 2 * g.abs().max()
    else:
        bG = bG * g.abs()
    bG = bG + 1e-38
    G = G * g
    for v, bv in (weighted_sum(G, bG, w, dt), weighted_sum(G.t(), bG.t(), xx, dt),
                  weighted_sum(G.t(), bG.t(), torch.ones(x.shape[0], 1, device=x.device), dt)):
        bv = bv + 4 * E * v.abs()
        out.append((v, bv + last(dt, v.abs() + bv)))
    out[3] = (out[3][0].squeeze(1), out[3][1].squeeze(1))
    return out


def assert_within(name, got, want):
    value, bound = want
    assert tuple(got.shape) == tuple(value.shape), (name, got.shape, value.shape)
    err = (got.double() - value).abs()
    bad = ~(err <= bound)
    if bool(bad.any()):
        i = int(torch.argmax(torch.where(bad, err / bound.clamp(min=1e-300), torch.zeros_like(err))
                             .nan_to_num(nan=float("inf")).reshape(-1)))
        raise AssertionError("%s: %d of %d outside the bound; worst at %d: got %r, want %r, bound %r"
                             % (name, int(bad.sum()), bad.numel(), i, float(got.reshape(-1)[i]),
                                float(value.reshape(-1)[i]), float(bound.reshape(-1)[i])))


def matrix(rows, cols, dt, gen, order="rows", scale=1.0, device="cuda"):
    """[rows, cols] in an order: rows; image ([cols, rows] in memory); padded (row
    stride beyond the row); odd (rows at an odd offset and stride); steps (every
    second column); same (every row the same memory)."""
    def new(*shape):
        return (torch.randn(*shape, generator=gen, device=device) * scale).to(dt)
    if order == "image":
        return new(cols, rows).t()
    if order == "padded":
        return new(rows, (cols + 15) // 8 * 8)[:, :cols]
    if order == "odd":
        return new(rows, cols + 3)[:, 1:cols + 1]
    if order == "image-odd":
        return new(cols, rows + 3)[:, 1:rows + 1].t()
    if order == "steps":
        return new(rows, 2 * cols)[:, ::2]
    if order == "same":
        return new(1, cols).expand(rows, cols)
    return new(rows, cols)
