"""Measured cases of the per-pixel heads: dense layers on rendered feature images
(``linear_act``) and the label loss over a vocabulary (``linear_cross_entropy``).

``run`` computes a case either with elementary torch operations in float32
(``own`` false) or through ``volume_integration.heads`` (``own`` true);
``exact`` computes it in float64.  All of them return the same outputs: for a
forward case the result, for a training case the result and the gradient of
every float input.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
ACTIVATIONS = ("none", "relu", "silu", "gelu", "sigmoid")
IGNORE = -100


def _act(name, M, K, N, dtype, act, train, image=False, bias=True, residual=False):
    return dict(name=name, op="linear_act", M=M, K=K, N=N, dtype=dtype, act=act, train=train, image=image,
                bias=bias, residual=residual)


def _ce(name, M, K, V, dtype, train, reduction, image=False, bias=True, ignored=0.0):
    return dict(name=name, op="linear_ce", M=M, K=K, V=V, dtype=dtype, train=train, reduction=reduction,
                image=image, bias=bias, ignored=ignored)


def listed():
    return [
        # the feature vector under the cursor through one hidden layer: latency
        _act("pick", 1, 256, 256, "bf16", "silu", train=False),
        # a few probe rays, odd sizes that no vector load or tile divides
        _act("probe", 37, 203, 131, "f16", "gelu", train=False, residual=True),
        # first decoder layer of a training step on the 800x800 views: the renderer's own float32 image of
        # four feature channels, channel-first
        _act("first-layer", 800 * 800, 4, 64, "f32", "relu", train=True, image=True),
        # a hidden block over a whole 1920x1080 frame at display time
        _act("frame", 1920 * 1080, 64, 64, "bf16", "gelu", train=False, image=True, residual=True),
        # a wide hidden block trained on a batch of rays
        _act("rays", 65536, 512, 512, "bf16", "silu", train=True, residual=True),
        # the expanding layer of a wide decoder
        _act("wide", 32768, 1024, 4096, "f16", "relu", train=True),
        # a float32 training step at ragged sizes
        _act("ragged", 5001, 515, 257, "f32", "sigmoid", train=True),
        # score of one picked pixel against a vocabulary of labels
        _ce("label-pick", 1, 256, 1000, "bf16", train=False, reduction="none"),
        # label loss of a 128x128 view, float32 channel-first features, unlabelled pixels ignored
        _ce("label-view", 128 * 128, 64, 21, "f32", train=True, reduction="mean", image=True, ignored=0.3),
        # validation loss of an 800x800 view, per pixel
        _ce("label-frame", 800 * 800, 64, 150, "f16", train=False, reduction="none", image=True, ignored=0.1),
        # a batch of rays against an odd-sized open vocabulary
        _ce("vocab-rays", 8192, 256, 30011, "bf16", train=True, reduction="mean", ignored=0.05),
        # the largest: codebook indices, 65536 codes
        _ce("codebook", 16384, 512, 65536, "bf16", train=True, reduction="sum", bias=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(("f32", "f16", "bf16", "bf16"))
    train, image, bias = rng.random() < 0.6, rng.random() < 0.4, rng.random() < 0.75
    if rng.random() < 0.5:
        while True:
            M, K, N = _log_int(rng, 1, 1920 * 1080), _log_int(rng, 1, 1024), _log_int(rng, 1, 4096)
            # float32 work is capped lower, so that no draw outweighs the largest listed case
            if M * K * N <= (1 << 37) // (8 if dtype == "f32" else 1) and M * (K + N) <= 1 << 28:
                break
        return dict(op="linear_act", M=M, K=K, N=N, dtype=dtype, act=rng.choice(ACTIVATIONS), train=train,
                    image=image, bias=bias, residual=rng.random() < 0.5)
    while True:
        M, K, V = _log_int(rng, 1, 800 * 800), _log_int(rng, 1, 512), _log_int(rng, 2, 65536)
        if M * K * V <= (1 << 38) // (8 if dtype == "f32" else 1) and M * V <= 1 << 29:
            break
    return dict(op="linear_ce", M=M, K=K, V=V, dtype=dtype, train=train,
                reduction=rng.choice(("mean", "sum", "none")), image=image, bias=bias,
                ignored=rng.choice((0.0, 0.05, 0.5)))


def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    M, K = case["M"], case["K"]
    n_out = case["N"] if case["op"] == "linear_act" else case["V"]

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(dt)

    # the renderer's image is [channels, pixels] in memory: rows are the columns of it
    x = randn(K, M).t() if case["image"] else randn(M, K)
    s = dict(x=x)
    if case["op"] == "linear_act":
        bound = 1.0 / math.sqrt(K)
        s["w"] = ((torch.rand(n_out, K, generator=gen, device=dev) * 2 - 1) * bound * 1.7).to(dt)
        s["b"] = randn(n_out, scale=0.3) if case["bias"] else None
        s["r"] = None
        if case["residual"]:
            s["r"] = randn(n_out, M).t() if case["image"] else randn(M, n_out)
        s["dy"] = None
        if case["train"]:
            s["dy"] = randn(n_out, M).t() if case["image"] else randn(M, n_out)
    else:
        # logits of a spread of about 3, as a trained head has
        s["w"] = randn(n_out, K, scale=3.0 / math.sqrt(K))
        s["b"] = randn(n_out, scale=0.5) if case["bias"] else None
        t = torch.randint(0, n_out, (M,), generator=gen, device=dev)
        drop = torch.rand(M, generator=gen, device=dev) < case["ignored"]
        if case["reduction"] == "mean":
            drop[0] = False  # a mean over no pixel at all is not a number
        s["t"] = torch.where(drop, torch.full_like(t, IGNORE), t)
        s["dl"] = None
        if case["train"]:
            shape = (M,) if case["reduction"] == "none" else ()
            s["dl"] = torch.rand(shape, generator=gen, device=dev) + 0.5
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
        if case["train"]:
            s["leaves"] = [s[k] for k in ("x", "w", "b", "r") if s.get(k) is not None]
            for leaf in s["leaves"]:
                leaf.requires_grad_(True)
    return s


def run(state):
    case = state["case"]
    if case["op"] == "linear_act":
        return _run_act_own(state) if own else _run_act_plain(state)
    return _run_ce_own(state) if own else _run_ce_plain(state)


def _run_act_own(s):
    c = s["case"]
    y = s["heads"].linear_act(s["x"], s["w"], s["b"], residual=s["r"], activation=c["act"])
    if not c["train"]:
        return [y]
    return [y.detach()] + list(torch.autograd.grad(y, s["leaves"], s["dy"]))


def _run_ce_own(s):
    c = s["case"]
    loss = s["heads"].linear_cross_entropy(s["x"], s["w"], s["t"], s["b"], ignore_index=IGNORE,
                                           reduction=c["reduction"])
    if not c["train"]:
        return [loss]
    return [loss.detach()] + list(torch.autograd.grad(loss, s["leaves"], s["dl"]))


def _run_act_plain(s):
    c = s["case"]
    dt = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    act = c["act"]
    if act == "none":
        y = z
    elif act == "relu":
        y = torch.where(z > 0, z, torch.zeros_like(z))
    elif act == "silu":
        y = z / (1 + torch.exp(-z))
    elif act == "gelu":
        y = z * (0.5 * (1 + torch.erf(z * math.sqrt(0.5))))
    else:
        y = 1 / (1 + torch.exp(-z))
    out = y + s["r"].float() if s["r"] is not None else y
    outs = [out.to(dt)]
    if not c["train"]:
        return outs
    g = s["dy"].float()
    if act == "relu":
        g = g * (z > 0)
    elif act == "silu":
        sig = 1 / (1 + torch.exp(-z))
        g = g * (sig * (1 + z * (1 - sig)))
    elif act == "gelu":
        g = g * (0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    elif act == "sigmoid":
        g = g * (y * (1 - y))
    outs += [(g @ w).to(dt), (g.t() @ x).to(dt)]
    if s["b"] is not None:
        outs.append(g.sum(0).to(dt))
    if s["r"] is not None:
        outs.append(s["dy"])
    return outs


def _run_ce_plain(s):
    c = s["case"]
    dt = s["x"].dtype
    x, w, t = s["x"].float(), s["w"].float(), s["t"]
    live = t != IGNORE
    idx = torch.where(live, t, torch.zeros_like(t)).unsqueeze(1)
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    top = z.max(1, keepdim=True).values
    lse = top + torch.log(torch.exp(z - top).sum(1, keepdim=True))
    rows = torch.where(live, (lse - z.gather(1, idx)).squeeze(1), torch.zeros_like(lse.squeeze(1)))
    n = live.sum()
    if c["reduction"] == "none":
        loss = rows
    else:
        loss = rows.sum() if c["reduction"] == "sum" else rows.sum() / n
    if not c["train"]:
        return [loss]
    scale = s["dl"] / n if c["reduction"] == "mean" else s["dl"]
    scale = torch.where(live, scale.expand(live.shape), torch.zeros_like(lse.squeeze(1))).unsqueeze(1)
    g = torch.exp(z - lse) * scale
    g.scatter_add_(1, idx, -scale)
    outs = [loss, (g @ w).to(dt), (g.t() @ x).to(dt)]
    if s["b"] is not None:
        outs.append(g.sum(0).to(dt))
    return outs


def work(case):
    M, K = case["M"], case["K"]
    e = BYTES[case["dtype"]]
    if case["op"] == "linear_act":
        N = case["N"]
        params = N * K + (N if case["bias"] else 0)
        b = e * (M * K + params + M * N + (M * N if case["residual"] else 0))
        if case["train"]:
            b += e * (M * N + M * K + params)
        return {"bytes": b, "flops": (6 if case["train"] else 2) * M * N * K}
    V = case["V"]
    params = V * K + (V if case["bias"] else 0)
    b = e * (M * K + params) + 8 * M + 4 * (M if case["reduction"] == "none" else 1)
    if case["train"]:
        b += e * (M * K + params) + 4 * (M if case["reduction"] == "none" else 1)
    return {"bytes": b, "flops": (6 if case["train"] else 2) * M * V * K}


def exact(case, seed):
    s = _inputs(case, seed)
    w = s["w"].double()
    b = s["b"].double() if s["b"] is not None else None
    M = case["M"]
    cols = w.shape[0]
    step = max(1, min(M, (1 << 26) // max(cols, case["K"])))
    pieces = [slice(i, min(M, i + step)) for i in range(0, M, step)]
    if case["op"] == "linear_act":
        return _exact_act(case, s, w, b, pieces)
    return _exact_ce(case, s, w, b, pieces)


def _affine64(x, w, b):
    z = torch.matmul(x.double(), w.transpose(0, 1))
    return z if b is None else z.add_(b)


def _exact_act(case, s, w, b, pieces):
    act, train = case["act"], case["train"]
    ys, dxs = [], []
    dw = torch.zeros_like(w)
    db = torch.zeros(w.shape[0], dtype=torch.float64, device=w.device)
    for p in pieces:
        xp = s["x"][p].double()
        z = _affine64(xp, w, b)
        if act == "none":
            a, d = z, torch.ones_like(z)
        elif act == "relu":
            a, d = z.clamp(min=0), z.gt(0).double()
        elif act == "sigmoid":
            a = torch.sigmoid(z)
            d = a * torch.sigmoid(-z)
        elif act == "silu":
            a = z * torch.sigmoid(z)
            d = torch.sigmoid(z) + a * torch.sigmoid(-z)
        else:
            cdf = 0.5 * torch.erfc(-z / math.sqrt(2.0))
            a = z * cdf
            d = cdf + z * torch.exp(z.square() * -0.5) * (1.0 / math.sqrt(2.0 * math.pi))
        ys.append(a if s["r"] is None else a + s["r"][p].double())
        if train:
            d = d * s["dy"][p].double()
            dxs.append(torch.matmul(d, w))
            dw += torch.matmul(d.transpose(0, 1), xp)
            db += d.sum(dim=0)
    outs = [torch.cat(ys)]
    if train:
        outs += [torch.cat(dxs), dw]
        if s["b"] is not None:
            outs.append(db)
        if s["r"] is not None:
            outs.append(s["dy"].double())
    return outs


def _exact_ce(case, s, w, b, pieces):
    t = s["t"]
    live = t.ne(IGNORE)
    count = int(live.sum())
    rows, dxs = [], []
    dw = torch.zeros_like(w)
    db = torch.zeros(w.shape[0], dtype=torch.float64, device=w.device)
    for p in pieces:
        xp = s["x"][p].double()
        logp = torch.log_softmax(_affine64(xp, w, b), dim=1)
        lp = live[p]
        tp = t[p].clamp(min=0)
        at = torch.arange(tp.numel(), device=tp.device)
        rows.append(-logp[at, tp] * lp)
        if case["train"]:
            g = logp.exp_()
            g[at, tp] -= 1.0
            k = s["dl"].double()
            k = k[p] if case["reduction"] == "none" else k.expand(tp.numel())
            if case["reduction"] == "mean":
                k = k / count
            g *= (k * lp).unsqueeze(1)
            dxs.append(torch.matmul(g, w))
            dw += torch.matmul(g.transpose(0, 1), xp)
            db += g.sum(dim=0)
    rows = torch.cat(rows)
    if case["reduction"] == "none":
        outs = [rows]
    else:
        outs = [rows.sum() if case["reduction"] == "sum" else rows.sum() / count]
    if case["train"]:
        outs += [torch.cat(dxs), dw]
        if s["b"] is not None:
            outs.append(db)
    return outs
