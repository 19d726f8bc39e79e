"""Measured cases of what surrounds the per-pixel heads' dense layers: the layer norm before
them (``layer_norm``), their display-time form in 8-bit integers (``linear_act_int8``),
and the label or codebook index drawn from their logits (``sample_labels``).

``run`` computes a case either with elementary torch operations (``own`` false) or through
``volume_integration.heads`` (``own`` true); ``exact`` computes it in float64 another way.
All of them return the same outputs: for a training case the result and the gradient of every
float input, else the result.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
ACTIVATIONS = ("none", "relu", "silu", "gelu", "sigmoid")
EPS = 1e-5


def _norm(name, M, K, dtype, train, image=False, affine=True):
    return dict(name=name, op="layer_norm", M=M, K=K, dtype=dtype, train=train, image=image, affine=affine)


def _int8(name, M, K, N, dtype, act, image=False, bias=True, residual=False):
    return dict(name=name, op="linear_act_int8", M=M, K=K, N=N, dtype=dtype, act=act, image=image, bias=bias,
                residual=residual)


def _draw_label(name, M, V, dtype, top_k=0, top_p=1.0, min_p=0.0, temperature=1.0, per_row=False, image=False,
                masked=0.0):
    return dict(name=name, op="sample_labels", M=M, V=V, dtype=dtype, top_k=top_k, top_p=top_p, min_p=min_p,
                temperature=temperature, per_row=per_row, image=image, masked=masked)


def listed():
    return [
        # the feature vector under the cursor: latency
        _norm("norm-pick", 1, 256, "bf16", train=False),
        # the hidden features of a whole 1920x1080 frame at display time, channel-first as the renderer's image
        _norm("norm-frame", 1920 * 1080, 64, "bf16", train=False, image=True),
        # a hidden block trained on a batch of rays
        _norm("norm-rays", 65536, 512, "bf16", train=True),
        # a float32 training step at ragged sizes
        _norm("norm-ragged", 5001, 515, "f32", train=True),
        # the wide block of a decoder, trained
        _norm("norm-wide", 32768, 4096, "f16", train=True),
        # the feature vector under the cursor through one hidden layer: latency
        _int8("int8-pick", 1, 256, 256, "bf16", "silu"),
        # a hidden block over a whole 1920x1080 frame at display time
        _int8("int8-frame", 1920 * 1080, 64, 64, "bf16", "gelu", image=True, residual=True),
        # the expanding layer of a wide decoder, at display time
        _int8("int8-wide", 32768, 1024, 4096, "f16", "relu"),
        # a label for one picked pixel: latency
        _draw_label("label-pick", 1, 1000, "f32", temperature=0.7),
        # one label for every pixel of an 800x800 view, a third of the classes ruled out
        _draw_label("label-view", 800 * 800, 150, "f16", min_p=0.02, image=True, masked=0.3),
        # a batch of rays against an odd-sized open vocabulary, each ray with its own settings
        _draw_label("vocab-rays", 1024, 30011, "f32", top_k=50, top_p=0.9, min_p=0.01, temperature=0.8, per_row=True),
        # codebook indices, 65536 codes
        _draw_label("codebook", 2048, 65536, "bf16", top_p=0.9, temperature=0.8),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(("f32", "f16", "bf16", "bf16"))
    image = rng.random() < 0.35
    op = rng.choice(("layer_norm", "linear_act_int8", "sample_labels"))
    if op == "layer_norm":
        while True:
            M, K = _log_int(rng, 1, 1920 * 1080), _log_int(rng, 4, 8192)
            if M * K <= 1 << 27:
                break
        return dict(op=op, M=M, K=K, dtype=dtype, train=rng.random() < 0.6, image=image, affine=rng.random() < 0.8)
    if op == "linear_act_int8":
        while True:
            M, K, N = _log_int(rng, 1, 1920 * 1080), _log_int(rng, 1, 1024), _log_int(rng, 1, 4096)
            if M * K * N <= 1 << 37 and M * (K + N) <= 1 << 28:
                break
        return dict(op=op, M=M, K=K, N=N, dtype=dtype, act=rng.choice(ACTIVATIONS), image=image,
                    bias=rng.random() < 0.75, residual=rng.random() < 0.5)
    while True:
        M, V = _log_int(rng, 1, 800 * 800), _log_int(rng, 2, 65536)
        if M * V <= 1 << 27:
            break
    return dict(op=op, M=M, V=V, dtype=dtype, top_k=rng.choice((0, _log_int(rng, 1, V))),
                top_p=rng.choice((1.0, rng.uniform(0.1, 0.99))), min_p=rng.choice((0.0, rng.uniform(0.001, 0.3))),
                temperature=rng.choice((0.0, 1.0, rng.uniform(0.2, 2.0))), per_row=rng.random() < 0.4, image=image,
                masked=rng.choice((0.0, 0.3, 0.95)))


def _quantised(w):
    """Rows of w as 8-bit integers and a float32 scale each; rows lie a multiple of 16 bytes apart."""
    rows, K = w.shape
    scale = _row_scale(w.double())
    q = torch.zeros(rows, (K + 15) // 16 * 16, dtype=torch.int8, device=w.device)[:, :K]
    q.copy_(torch.round(w.double() / scale.double().unsqueeze(1)))
    return q, scale


def _row_scale(x64):
    return (x64.abs().amax(1) / 127.0).float()


def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    M, image = case["M"], case["image"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device=dev)

    def pixels(cols, scale=1.0, shift=None):
        # the renderer's image is [channels, pixels] in memory: rows are the columns of it
        v = (randn(cols, M) if image else randn(M, cols)).mul_(scale)
        if shift is not None:
            v.add_(shift if image else shift.unsqueeze(1))
        v = v.to(dt)
        return v.t() if image else v

    if case["op"] == "layer_norm":
        K = case["K"]
        s = dict(x=pixels(K, 1.5, randn(M)), w=None, b=None, dy=None)
        if case["affine"]:
            s["w"], s["b"] = (1 + 0.2 * randn(K)).to(dt), (0.2 * randn(K)).to(dt)
        if case["train"]:
            s["dy"] = pixels(K)
        return s
    if case["op"] == "linear_act_int8":
        K, N = case["K"], case["N"]
        s = dict(x=pixels(K), b=None, r=None)
        s["w"] = _quantised((rand(N, K) * 2 - 1) * (1.7 / math.sqrt(K)))
        if case["bias"]:
            s["b"] = (0.3 * randn(N)).to(dt)
        if case["residual"]:
            s["r"] = pixels(N)
        return s
    # logits of a spread of about 3, as a trained head has
    V = case["V"]
    z = pixels(V, 3.0)
    if case["masked"]:
        z[:, rand(V) < case["masked"]] = -math.inf
    s = dict(z=z, u=rand(M))
    for name in ("temperature", "top_k", "top_p", "min_p"):
        s[name] = case[name]
    if case["per_row"]:
        s["temperature"] = case["temperature"] * (0.5 + rand(M))
        s["top_k"] = (case["top_k"] * (0.5 + rand(M))).long()
        s["top_p"] = (1 - (1 - case["top_p"]) * (0.5 + rand(M))).clamp(min=0.05)
        s["min_p"] = case["min_p"] * (0.5 + rand(M))
        if M > 3:
            z[M // 2] = -math.inf  # a ray whose mask leaves nothing
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        pkg = os.path.join(root, "volume-integration_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from volume_integration import heads
        s["heads"] = heads
        if case.get("train"):
            s["leaves"] = [s[k] for k in ("x", "w", "b") if s[k] is not None]
            for leaf in s["leaves"]:
                leaf.requires_grad_(True)
    return s


def run(state):
    op = state["case"]["op"]
    if op == "layer_norm":
        return _run_norm_own(state) if own else _run_norm_plain(state)
    if op == "linear_act_int8":
        return _run_int8_own(state) if own else _run_int8_plain(state)
    return _run_draw_own(state) if own else _run_draw_plain(state)


def _run_norm_own(s):
    y = s["heads"].layer_norm(s["x"], s["w"], s["b"], eps=EPS)
    if not s["case"]["train"]:
        return [y]
    return [y.detach()] + list(torch.autograd.grad(y, s["leaves"], s["dy"]))


def _run_int8_own(s):
    c = s["case"]
    return [s["heads"].linear_act_int8(s["x"], s["w"], s["b"], residual=s["r"], activation=c["act"])]


def _run_draw_own(s):
    return [s["heads"].sample_labels(s["z"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                     top_p=s["top_p"], min_p=s["min_p"])]


def _run_norm_plain(s):
    dt = s["x"].dtype
    x = s["x"].float()
    d = x - x.mean(1, keepdim=True)
    r = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    h = d * r
    w = s["w"].float() if s["w"] is not None else None
    y = h if w is None else h * w + s["b"].float()
    outs = [y.to(dt)]
    if not s["case"]["train"]:
        return outs
    dy = s["dy"].float()
    g = dy if w is None else dy * w
    dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    outs.append(dx.to(dt))
    if w is not None:
        outs += [(dy * h).sum(0).to(dt), dy.sum(0).to(dt)]
    return outs


def _run_int8_plain(s):
    dt, act = s["x"].dtype, s["case"]["act"]
    x = s["x"].float()
    p, t = s["w"]
    top = x.abs().amax(1, keepdim=True)
    scale = top / torch.full_like(top, 127.0)
    # the quotient in 64 bits: in 32 it may round to a half that it is not
    q = torch.round(x.double() / torch.where(scale > 0, scale, torch.ones_like(scale)).double()).float()
    # sums of at most 1024 products of at most 127^2 are whole numbers under 2^24
    z = (q @ p.float().t()) * (scale * t)
    if s["b"] is not None:
        z = z + s["b"].float()
    if act == "relu":
        z = torch.where(z > 0, z, torch.zeros_like(z))
    elif act == "silu":
        z = z / (1 + torch.exp(-z))
    elif act == "gelu":
        z = z * (0.5 * (1 + torch.erf(z * math.sqrt(0.5))))
    elif act == "sigmoid":
        z = 1 / (1 + torch.exp(-z))
    return [(z + s["r"].float() if s["r"] is not None else z).to(dt)]


def _column(v, z):
    """A setting of the call as a column: one value a row."""
    if not torch.is_tensor(v):
        v = torch.full((z.shape[0],), v, device=z.device, dtype=torch.float64 if isinstance(v, float) else torch.int64)
    return v.unsqueeze(1)


def _run_draw_plain(s):
    # weights and their sums in 64 bits: a draw may fall next to a border
    z = s["z"].float() + 0.0
    V = z.shape[1]
    T = _column(s["temperature"], z).double()
    top = z.amax(1, keepdim=True)
    first = (z == top).to(torch.uint8).argmax(1, keepdim=True)
    dead = top == -math.inf
    safe = torch.where(dead, torch.zeros_like(top), top).double()
    w = torch.exp((z.double() - safe) / torch.where(T > 0, T, torch.ones_like(T)))
    k, p, m = _column(s["top_k"], z), _column(s["top_p"], z).double(), _column(s["min_p"], z).double()
    keep = w >= m
    if not (isinstance(s["top_k"], int) and s["top_k"] == 0 and isinstance(s["top_p"], float) and s["top_p"] >= 1):
        order = torch.sort(z, dim=1, descending=True, stable=True).indices
        ws = w.gather(1, order)
        rank = torch.arange(V, device=z.device).unsqueeze(0)
        ws = torch.where((k <= 0) | (rank < k), ws, torch.zeros_like(ws))
        before = ws.cumsum(1)
        live = ((k <= 0) | (rank < k)) & ((p >= 1) | (before - ws < p * before[:, -1:]) | (rank == 0))
        keep = keep & torch.zeros_like(live).scatter_(1, order, live)
    total = torch.where(keep, w, torch.zeros_like(w)).cumsum(1)
    t = s["u"].double().unsqueeze(1) * total[:, -1:]
    label = (total <= t).sum(1, keepdim=True)
    label = torch.where(T > 0, label, first)
    return [torch.where(dead, torch.full_like(label, -1), label).squeeze(1)]


def work(case):
    M, e = case["M"], BYTES[case["dtype"]]
    if case["op"] == "layer_norm":
        K, n = case["K"], 2 * case["K"] if case["affine"] else 0
        if case["train"]:  # x, dy in; y, dx out; the weights in, their gradients out
            return {"bytes": e * (4 * M * K + 2 * n), "flops": 24 * M * K}
        return {"bytes": e * (2 * M * K + n), "flops": 8 * M * K}
    if case["op"] == "linear_act_int8":
        K, N = case["K"], case["N"]
        b = e * (M * K + M * N + (N if case["bias"] else 0) + (M * N if case["residual"] else 0)) + N * K + 4 * N
        return {"bytes": b, "flops": 2 * M * N * K}
    return {"bytes": M * (e * case["V"] + 4 + 8 + (20 if case["per_row"] else 0)), "flops": 4 * M * case["V"]}


def exact(case, seed):
    s = _inputs(case, seed)
    M = case["M"]
    cols = max(case.get("K", 0), case.get("N", 0), case.get("V", 0))
    step = max(1, min(M, (1 << 25) // cols))
    pieces = [slice(i, min(M, i + step)) for i in range(0, M, step)]
    if case["op"] == "layer_norm":
        return _exact_norm(case, s, pieces)
    if case["op"] == "linear_act_int8":
        return _exact_int8(case, s, pieces)
    return [torch.cat([_exact_draw(s, p) for p in pieces])]


def _exact_norm(case, s, pieces):
    K, dev = case["K"], s["x"].device
    w = s["w"].double() if s["w"] is not None else torch.ones(K, dtype=torch.float64, device=dev)
    b = s["b"].double() if s["b"] is not None else torch.zeros(K, dtype=torch.float64, device=dev)
    ys, dxs, dw, db = [], [], torch.zeros_like(w), torch.zeros_like(b)
    for p in pieces:
        x = s["x"][p].double()
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        r = torch.rsqrt(var + EPS)
        h = x.sub_(mean).mul_(r)
        ys.append(torch.addcmul(b, h, w))
        if case["train"]:
            dy = s["dy"][p].double()
            g = dy.mul(w)
            along = torch.linalg.vecdot(g, h).unsqueeze(1) / K
            dxs.append((g - g.sum(1, keepdim=True) / K).addcmul_(h, along, value=-1).mul_(r))
            dw += torch.einsum("mk,mk->k", dy, h)
            db += torch.einsum("mk->k", dy)
    outs = [torch.cat(ys)]
    if case["train"]:
        outs.append(torch.cat(dxs))
        if s["w"] is not None:
            outs += [dw, db]
    return outs


def _exact_int8(case, s, pieces):
    p8, t = s["w"]
    w = p8.double()
    ys = []
    for p in pieces:
        x = s["x"][p].double()
        scale = _row_scale(x).double().unsqueeze(1)
        q = (x / scale.clamp(min=1e-300)).round_()
        z = torch.matmul(q, w.transpose(0, 1)).mul_(scale).mul_(t.double())
        if s["b"] is not None:
            z += s["b"].double()
        act = case["act"]
        if act == "relu":
            z = z.clamp_(min=0)
        elif act == "silu":
            z = z * torch.sigmoid(z)
        elif act == "gelu":
            z = z * torch.erfc(z / -math.sqrt(2.0)) * 0.5
        elif act == "sigmoid":
            z = torch.sigmoid(z)
        ys.append(z if s["r"] is None else z + s["r"][p].double())
    return [torch.cat(ys)]


def _exact_draw(s, p):
    z = s["z"][p].double()
    n, V = z.shape

    def setting(name):
        v = s[name]
        return (v[p].double() if torch.is_tensor(v) else torch.full((n,), float(v), device=z.device,
                                                                    dtype=torch.float64)).unsqueeze(1)

    T, k, top_p, min_p = (setting(name) for name in ("temperature", "top_k", "top_p", "min_p"))
    best = z.amax(1, keepdim=True)
    dead = torch.isneginf(best)
    cold = T == 0
    prob = torch.softmax(torch.where(dead, torch.zeros_like(z), z) / torch.where(cold, torch.ones_like(T), T), dim=1)
    ranked, order = torch.sort(-z, dim=1, stable=True)
    prob = prob.gather(1, order)
    place = torch.arange(1, V + 1, device=z.device).expand(n, V)
    prob = prob * ((place <= k) | (k == 0))
    after = prob.flip(1).cumsum(1).flip(1)  # an entry's own mass and what comes behind it
    mass = after[:, :1]
    inside = (after > (1 - top_p) * mass) | (top_p >= 1)
    inside[:, 0] = True
    prob = prob * inside * (prob >= min_p * prob[:, :1])
    prob = torch.zeros_like(prob).scatter_(1, order, prob)
    run_sum = prob.cumsum(1)
    at = torch.searchsorted(run_sum, s["u"][p].double().unsqueeze(1) * run_sum[:, -1:], right=True)
    at = torch.where(cold, order[:, :1], at)
    return at.masked_fill(dead, -1).squeeze(1)
