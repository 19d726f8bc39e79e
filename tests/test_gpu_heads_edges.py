"""GPU tests of the per-pixel heads at the ends of their ranges: values that are not finite or far out, long
sums, tiles made by pairs of blocks, tangents, and incoming gradients that are not finite.

Bounds are those of heads_lib unless a test derives its own: u is half a step of the element type, e = 2^-23."""
import ctypes
import math

import pytest
import torch

import heads_abi as ha
import heads_lib as hl

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = dict(argvalues=[F32, F16, BF16], ids=["f32", "f16", "bf16"])
NAN, INF = float("nan"), float("inf")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inputs(M, K, N, dt, order, bias, residual, seed):
    g = _gen(seed)
    x = hl.matrix(M, K, dt, g, order)
    w = hl.matrix(N, K, dt, g, scale=1.5 / K ** 0.5)
    b = hl.matrix(1, N, dt, g, scale=0.3)[0] if bias else None
    r = hl.matrix(M, N, dt, g, "image" if order.startswith("image") else "rows") if residual else None
    dy = hl.matrix(M, N, dt, g, "image" if order == "image" else "rows")
    return x, w, b, r, dy


def _step(x, w, b, r, act, dy):
    """y and the gradients of the float inputs that are there."""
    import volume_integration.heads as heads
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b, r)]
    y = heads.linear_act(*leaves, activation=act)
    return y.detach(), list(torch.autograd.grad(y, [t for t in leaves if t is not None], dy))


def _check(x, w, b, r, act, dy):
    y, grads = _step(x, w, b, r, act, dy)
    want = hl.linear_act(x, w, b, r, act, dy)
    hl.assert_within("y", y, want[0])
    hl.assert_within("dx", grads[0], want[1])
    hl.assert_within("dweight", grads[1], want[2])
    if b is not None:
        hl.assert_within("dbias", grads[2], want[3])


def _pairs():
    # launches so far with tiles of two blocks
    lib = ha.load()
    lib.vi_heads_pair_launches.restype = ctypes.c_uint64
    return lib.vi_heads_pair_launches()


# ---- values that are not finite ----
# M, K, N and order: the small products, the tensor cores, an image of few channels, an image
PATHS = [(90, 40, 70, "rows"), (900, 40, 70, "rows"), (900, 4, 70, "image"), (900, 40, 130, "image")]


@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("act", hl.ACTS)
@pytest.mark.parametrize("M,K,N,order", PATHS)
def test_a_nan_reaches_the_gradients(M, K, N, order, act, dt):
    # a row whose features hold a NaN: act' is NaN there, but relu's, which is 0 (z > 0 is false) and 1
    x, w, b, _, dy = _inputs(M, K, N, dt, order, True, False, 60)
    clean_y, clean = _step(x, w, b, None, act, dy)
    x2 = x.clone(memory_format=torch.preserve_format)
    x2[5, 3] = NAN
    y, (dx, dw, db) = _step(x2, w, b, None, act, dy)
    keep = torch.arange(M, device="cuda") != 5
    assert bool(torch.isnan(y[5]).all())
    assert torch.equal(y[keep], clean_y[keep]) and torch.equal(dx[keep], clean[0][keep])
    assert bool(torch.isnan(dw[:, 3]).all())  # 0 * NaN too
    if act in ("silu", "gelu", "sigmoid"):
        assert bool(torch.isnan(dx[5]).all()) and bool(torch.isnan(dw).all()) and bool(torch.isnan(db).all())
    else:
        s = dy[5] if act == "none" else torch.zeros_like(dy[5])
        want = hl.linear_act(x, w, b, None, act, dy)
        assert bool(torch.isfinite(dx[5]).all()) and bool(torch.isfinite(db).all())
        value, bound = hl.weighted_sum(s[None].double(), torch.zeros(1, N, device="cuda", dtype=torch.float64), w, dt)
        hl.assert_within("dx", dx[5:6], (value, bound + hl.last(dt, value.abs() + bound)))
        d5 = (dy[5].double() * hl.act64(act, hl.product(x[5:6], w, b)[0])[1][0]) - s.double()
        value, bound = want[3]
        hl.assert_within("dbias", db, (value - d5, bound + hl.last(dt, d5.abs())))


@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("M,K,N,order", PATHS)
def test_infinite_preactivations(M, K, N, order, dt):
    # through the bias, which float32's planes do not pass: sigmoid and relu have limits, silu's derivative is NaN
    x, w, b, _, dy = _inputs(M, K, N, dt, order, True, False, 61)
    b[1], b[2] = INF, -INF
    for act, high, low, dhigh, dlow in (("relu", INF, 0.0, 1.0, 0.0), ("sigmoid", 1.0, 0.0, 0.0, 0.0),
                                        ("silu", INF, NAN, NAN, NAN)):
        y, (_, _, db) = _step(x, w, b, None, act, dy)
        for j, v, d in ((1, high, dhigh), (2, low, dlow)):
            want = torch.full_like(y[:, j], v)
            assert torch.equal(y[:, j].nan_to_num(nan=7.0), want.nan_to_num(nan=7.0)), (act, j, y[:3, j])
            if math.isnan(d):
                assert bool(torch.isnan(db[j]))
            else:
                total = dy[:, j].double().sum() * d
                assert abs(float(db[j]) - float(total)) <= float((M + 16) * hl.E * dy[:, j].double().abs().sum() * d
                                                                 + hl.last(dt, total.abs()))


# ---- the far tails ----
def _tail_values(dt):
    v = [0.0, 2.0 ** -9, 0.5, 3.0, 5.0, 5.5, 6.0, 6.5, 7.0, 8.0, 9.0, 10.0, 11.0, 12.0, 12.5, 13.0, 13.5, 14.0, 15.0,
         16.0, 17.0, 18.0, 19.0, 20.0, 24.0, 30.0, 40.0, 43.0, 60.0, 80.0, 86.5, 87.5, 88.0, 89.0, 100.0, 127.0, 200.0,
         1000.0, 60000.0]
    if dt != F16:
        v += [1e6, 1e20, 1e30, 1e37, 2e38, torch.finfo(dt).max]
    t = torch.tensor(v, dtype=torch.float64).to(dt)
    return torch.cat([t, -t]).cuda()


@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("act", hl.ACTS)
@pytest.mark.parametrize("M,K,N,image", [(90, 16, 8, False), (700, 16, 64, False), (700, 4, 8, True), (700, 16, 130, True),
                                         (700, 136, 64, False)])
def test_activations_far_out(M, K, N, image, act, dt):
    # z is one element of x, so it is exact; y and act' at every magnitude the type holds, with and without gradients
    import volume_integration.heads as heads
    values = _tail_values(dt)
    z = values.repeat(M // values.numel() + 1)[:M]
    x = torch.zeros(K, M, device="cuda", dtype=dt).t() if image else torch.zeros(M, K, device="cuda", dtype=dt)
    w = torch.zeros(N, K, device="cuda", dtype=dt)
    x[:, 1], w[:, 1] = z, 1.0
    dy = torch.zeros(N, M, device="cuda", dtype=dt).t() if image else torch.zeros(M, N, device="cuda", dtype=dt)
    dy[:, 3] = 1.0
    y, (dx, _) = _step(x, w, None, None, act, dy)
    with torch.no_grad():
        assert torch.equal(heads.linear_act(x, w, None, None, act), y)
    y64, d64 = hl.act64(act, z.double())
    u = hl.half_step(dt)
    # silu and sigmoid to 64 e of the value; where 1 / (1 + exp(-z)) is below 2^-126 the 16-bit forms may take it for 0,
    # 87.4 * 2^-126 of a product with z there.
    # gelu's polynomial beside 16-bit types: 64 e of the value down to 1e-3, then 1e-7 absolute of it to -5,
    # and 2% of what is left (below 1e-6) beyond, where Phi < 3e-7.
    by = (u + 64 * hl.E) * y64.abs() + hl.tiny(dt) + 2.0 ** -119
    bd = (3 * u + 64 * hl.E) * d64.abs() + 2.0 ** -119
    if act == "gelu":
        zd = z.double()
        far = zd < -5
        floor = torch.full_like(zd, 1e-7)
        by = by + torch.where(far, 0.02 * y64.abs(), torch.where(zd < 0, floor, 0 * floor))
        # act' = Q + x phi: its terms are up to 1/2, and cancel near their zero
        bd = bd + torch.where(far, 0.02 * d64.abs(), 64 * hl.E * torch.full_like(zd, 0.5) + floor)
    if dt == BF16:
        bd = bd + 2.0 ** -40  # half the kept form's smallest step
    if dt == F16:
        bd = bd + 2.0 ** -26 + 2.0 ** -24  # the kept form's, and s's and dx's own
    hl.assert_within("y", y[:, 5], (y64, by))
    hl.assert_within("act'", dx[:, 1], (d64, bd))


@pytest.mark.parametrize("M,K,N,order", [(60, 25, 40, "rows"), (60, 24, 40, "rows"), (900, 24, 40, "rows"),
                                         (900, 4, 40, "image"), (900, 24, 130, "image")])
@pytest.mark.parametrize("residual", [False, True])
def test_relu_of_a_value_under_the_type(M, K, N, order, residual):
    # float16: z = 2^-26 rounds to a result of 0, but it is positive, and its gradient passes
    x, _, _, r, dy = _inputs(M, K, N, F16, order, False, residual, 62)
    x.zero_()
    w = torch.zeros(N, K, device="cuda", dtype=F16)
    x[:, 2] = 2.0 ** -13
    x[::3, 2] = -2.0 ** -13
    w[:, 2] = 2.0 ** -13
    y, grads = _step(x, w, None, r, "relu", dy)
    assert torch.equal(y, r if residual else torch.zeros_like(y))
    s = dy.double() * (x[:, 2:3] > 0)
    value, bound = hl.weighted_sum(s, torch.zeros_like(s), w, F16)
    hl.assert_within("dx", grads[0], (value, bound + hl.last(F16, value.abs() + bound)))
    value, bound = hl.weighted_sum(s.t(), torch.zeros_like(s.t()), x, F16)
    hl.assert_within("dweight", grads[1], (value, bound + hl.last(F16, value.abs() + bound)))


# ---- long sums ----
# The tensor core cuts what it adds towards zero, so a sum of positive terms drifts down: measured, 1.5e-3 over 262144
# terms, as if each of four additions per 16 terms lost half a step of a running sum that is on average half its end: a step e
# per 16 terms.  The chain without a rounded addition in between is 768 terms in float32 (48 e) and 16384 beside
# float16 (1024 e), whatever the length.
F32_CHAIN = 48 + 16


@pytest.mark.parametrize("K,act,order", [(32768, "none", "rows"), (20011, "silu", "image")])
def test_long_float32_products(K, act, order):
    # every term positive: the whole drift adds up
    import volume_integration.heads as heads
    g = _gen(63)
    x = torch.rand(K, 300, generator=g, device="cuda").t() if order == "image" else torch.rand(300, K, generator=g, device="cuda")
    w = torch.rand(140, K, generator=g, device="cuda") / K
    y = heads.linear_act(x, w, activation=act)
    z = x.double() @ w.double().t()
    y64, d = hl.act64(act, z)
    # rounded additions of the pieces: half a step each
    bound = (F32_CHAIN + K / 768 / 2) * hl.E * z * d.abs().clamp(min=1) + 32 * hl.E * y64.abs() + 1e-7
    hl.assert_within("y", y, (y64, bound))


@pytest.mark.parametrize("V", [2, 300])
def test_long_float32_logits(V):
    # class 0 has logit 0, the others about 20 from positive terms, so that a drift does not cancel
    K, M = 32768, 260
    g = _gen(64)
    x = torch.rand(M, K, generator=g, device="cuda")
    w = torch.rand(V, K, generator=g, device="cuda") * (80.0 / K)
    w[0] = 0.0
    t = torch.zeros(M, dtype=torch.int64, device="cuda")
    import volume_integration.heads as heads
    wl = w.clone().requires_grad_(True)
    loss = heads.linear_cross_entropy(x, wl, t, reduction="none")
    (dw,) = torch.autograd.grad(loss.sum(), (wl,))
    z = x.double() @ w.double().t()
    lse = torch.logsumexp(z, 1)
    dz = (F32_CHAIN + K / 768 / 2) * hl.E * z
    bound = dz.max(1).values + (V + 16) * hl.E + 8 * hl.E * lse
    hl.assert_within("loss", loss.detach(), (lse, bound))
    # G = p - onehot: p off by p (dz + dlse + 16 e (1 + |z - lse|))
    p = torch.exp(z - lse[:, None])
    G = p.clone()
    G[:, 0] -= 1
    bG = p * (dz + bound[:, None] + 16 * hl.E * (1 + (z - lse[:, None]).abs())) + 4 * hl.E * G.abs() + 1e-38
    value, vb = hl.weighted_sum(G.t(), bG.t(), x, F32)
    hl.assert_within("dweight", dw, (value, vb + 4 * hl.E * value.abs() + hl.last(F32, value.abs() + vb)))


@pytest.mark.parametrize("dt", [F16, BF16], ids=["f16", "bf16"])
def test_long_logits_of_16_bit_features(dt):
    # the loss is float32 whatever the features are: a chain of logits is 4096 terms (256 e)
    import volume_integration.heads as heads
    K, M, V = 32768, 260, 300
    g = _gen(78)
    x = torch.rand(M, K, generator=g, device="cuda").to(dt)
    w = (torch.rand(V, K, generator=g, device="cuda") * (80.0 / K)).to(dt)
    w[0] = 0.0
    t = torch.zeros(M, dtype=torch.int64, device="cuda")
    loss = heads.linear_cross_entropy(x, w, t, reduction="none")
    z = x.double() @ w.double().t()
    lse = torch.logsumexp(z, 1)
    bound = (256 + 16 + K / 4096 / 2) * hl.E * z.max(1).values + (V + 16) * hl.E + 8 * hl.E * lse
    hl.assert_within("loss", loss, (lse, bound))


def test_long_float16_weight_gradients():
    # 262144 rows into 2048 x 2048: as many tiles as run at a time, so each is one long sum.  The mean over many
    # elements leaves the drift: roundings of the result (u each, either way) average out.
    M, N = 262144, 2048
    g = _gen(65)
    x = torch.empty(M, N, device="cuda", dtype=F16).uniform_(0.5, 1.5, generator=g)
    dy = torch.empty(M, N, device="cuda", dtype=F16).uniform_(2.0 ** -12, 3 * 2.0 ** -12, generator=g)
    w = torch.zeros(N, N, device="cuda", dtype=F16).requires_grad_(True)
    import volume_integration.heads as heads
    (dw,) = torch.autograd.grad(heads.linear_act(x, w), (w,), dy)
    some = slice(0, N, 64)
    want = dy[:, some].double().t() @ x.double()
    drift = float(((dw[some].double() - want) / want).mean())
    # the chain's 1024 e; 2^18 / 2^14 rounded additions; 65536 roundings of at most u
    assert abs(drift) <= 1024 * hl.E + 16 * hl.E + 4 * 2.0 ** -11 / 256, drift


@pytest.mark.parametrize("M,K,N,act,order,dt", [
    (300, 20011, 140, "silu", "rows", F16), (300, 16448, 140, "gelu", "image", F16), (40, 20000, 1000, "relu", "rows", F16),
    (130, 140003, 70, "sigmoid", "rows", BF16), (130, 5000, 70, "gelu", "image", F32), (700, 1003, 300, "relu", "odd", F32),
])
def test_long_products_with_everything(M, K, N, act, order, dt):
    # more than a chain of k in the forward, with act', bias and residual; dx and dweight in their own tiles
    x, w, b, r, dy = _inputs(M, K, N, dt, order, True, True, 71)
    _check(x, w, b, r, act, dy)
    _check(x, w, b, None, act, dy)


@pytest.mark.parametrize("M,K,V,dt", [(260, 20000, 50, F16), (260, 16500, 300, F16), (130, 140000, 70, BF16),
                                      (700, 1000, 5003, F32), (20000, 24, 21, F32),
                                      (17000, 800, 1500, F32)])  # the last: several tiles a block, in runs
def test_long_logits_and_long_gradients(M, K, V, dt):
    import volume_integration.heads as heads
    g = _gen(72)
    x, w = hl.matrix(M, K, dt, g), hl.matrix(V, K, dt, g, scale=3.0 / K ** 0.5)
    b = hl.matrix(1, V, dt, g, scale=0.5)[0]
    t = torch.randint(0, V, (M,), generator=g, device="cuda")
    t[::7] = -100
    leaves = [v.detach().requires_grad_(True) for v in (x, w, b)]
    loss = heads.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
    grads = torch.autograd.grad(loss, leaves)
    want = hl.linear_ce(x, w, b, t, -100, "mean", torch.ones((), device="cuda"))
    for name, got, ref in zip(("loss", "dx", "dweight", "dbias"), (loss.detach(),) + grads, want):
        hl.assert_within(name, got, ref)


def test_long_sums_on_tiles_of_pairs():
    # dx over 16500 columns: 192 tiles for 74 pairs, each of two chains
    import volume_integration.heads as heads
    g = _gen(76)
    M, K, N = 12288, 1024, 16500
    w = hl.matrix(N, K, F16, g, scale=N ** -0.5)
    x = torch.zeros(M, K, device="cuda", dtype=F16, requires_grad=True)
    dy = hl.matrix(M, N, F16, g)
    before = _pairs()
    (dx,) = torch.autograd.grad(heads.linear_act(x, w), (x,), dy)
    assert _pairs() > before
    value, bound = hl.weighted_sum(dy.double(), torch.zeros(1, 1, device="cuda", dtype=torch.float64).expand(M, N), w, F16)
    hl.assert_within("dx", dx, (value, bound + hl.last(F16, value.abs() + bound)))


def test_long_float32_gradients():
    # positive terms again: dweight over 300000 rows, dx over 20000 columns
    import volume_integration.heads as heads
    g = _gen(73)
    for M, K, N in ((300000, 70, 130), (260, 140, 20000)):
        x = torch.rand(M, K, generator=g, device="cuda").requires_grad_(True)
        w = torch.rand(N, K, generator=g, device="cuda").requires_grad_(True)
        dy = torch.rand(M, N, generator=g, device="cuda") / max(M, N)
        dx, dw = torch.autograd.grad(heads.linear_act(x, w), (x, w), dy)
        for name, got, a, b, terms in (("dx", dx, dy, w, N), ("dweight", dw, dy.t(), x.t().contiguous().t(), M)):
            want = a.double() @ b.detach().double()
            hl.assert_within(name, got, (want, (F32_CHAIN + terms / 768 / 2) * hl.E * want))


# ---- tiles made by pairs of blocks ----
@pytest.mark.parametrize("dt", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("M,K,N,act,order,bias,residual,pairs", [
    # 64 tiles of 256 x 256 (one wave of 74 pairs, where narrower tiles take two and more): the forward's,
    # dx's where K is as wide, and dweight's in pieces
    (4096, 1024, 1024, "silu", "rows", True, True, 3),
    (4090, 1020, 1020, "gelu", "rows", True, True, 3),
    (4093, 1016, 1021, "gelu", "image", True, True, 3),
    (4090, 1020, 1020, "relu", "image", True, False, 3),
    (4088, 1024, 1016, "sigmoid", "image", True, True, 3),
    (4096, 520, 1024, "sigmoid", "padded", True, False, 1),
    (4090, 136, 1020, "none", "odd", False, True, 1),
])
def test_linear_act_on_tiles_of_pairs(M, K, N, act, order, bias, residual, pairs, dt):
    import volume_integration.heads as heads
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the sizes fill 148 SMs")
    x, w, b, r, dy = _inputs(M, K, N, dt, order, bias, residual, M + N)
    before = _pairs()
    with torch.no_grad():
        y = heads.linear_act(x, w, b, r, act)
    assert _pairs() == before + 1
    _check(x, w, b, r, act, dy)
    assert _pairs() >= before + 1 + pairs
    assert torch.equal(_step(x, w, b, r, act, dy)[0], y)


@pytest.mark.parametrize("dt", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("M,K,V,order", [(4096, 1024, 4096, "rows"), (4090, 1020, 4090, "image")])
def test_label_gradients_on_tiles_of_pairs(M, K, V, order, dt):
    import volume_integration.heads as heads
    g = _gen(M)
    x, w = hl.matrix(M, K, dt, g, order), hl.matrix(V, K, dt, g, scale=3.0 / K ** 0.5)
    t = torch.randint(0, V, (M,), generator=g, device="cuda")
    t[::9] = -100
    leaves = [v.detach().requires_grad_(True) for v in (x, w)]
    before = _pairs()
    loss = heads.linear_cross_entropy(leaves[0], leaves[1], t)
    grads = torch.autograd.grad(loss, leaves)
    assert torch.cuda.get_device_properties(0).multi_processor_count != 148 or _pairs() == before + 2
    want = hl.linear_ce(x, w, None, t, -100, "mean", torch.ones((), device="cuda"))
    for name, got, ref in zip(("loss", "dx", "dweight"), (loss.detach(),) + grads, want):
        hl.assert_within(name, got, ref)


def test_tiles_of_pairs_captured_and_on_two_streams():
    x, w, b, r, dy = _inputs(4090, 1020, 1020, BF16, "rows", True, True, 69)
    before = _pairs()
    want = _step(x, w, b, r, "silu", dy)
    assert _pairs() >= before + 3 or torch.cuda.get_device_properties(0).multi_processor_count != 148
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(x, w, b, r, "silu", dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(x, w, b, r, "silu", dy)
    torch.cuda.synchronize()
    results = []
    for _ in range(3):  # a replay beside two eager streams
        graph.replay()
        for s in (side, torch.cuda.Stream()):
            s.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(s):
                results.append(_step(x, w, b, r, "silu", dy))
    torch.cuda.synchronize()
    for y, grads in results + [out]:
        assert torch.equal(y, want[0])
        for a, c in zip(grads, want[1]):
            assert torch.equal(a, c)
    del graph


def test_a_wait_that_runs_out_in_a_long_sum_is_reported(monkeypatch):
    import volume_integration.heads as heads
    x, w, _, _, _ = _inputs(300, 3000, 200, F32, "rows", False, False, 77)
    want = heads.linear_act(x, w)
    assert heads.device_status(reset=True) == 0
    monkeypatch.setenv("VI_HEADS_TEST_TIMEOUT", "1")
    heads.linear_act(x, w)
    assert heads.device_status(reset=True) == 8
    monkeypatch.delenv("VI_HEADS_TEST_TIMEOUT")
    assert torch.equal(heads.linear_act(x, w), want)
    assert heads.device_status() == 0


@pytest.mark.parametrize("K", [200, 1000])  # fewer blocks of k than stages, and more
def test_a_wait_that_runs_out_in_a_pair_is_reported(K, monkeypatch):
    # the first load is withheld and the waits are short: both blocks of a pair give up and say so
    import volume_integration.heads as heads
    x, w, _, _, _ = _inputs(4090, K, 1020, BF16, "rows", False, False, 70)
    before = _pairs()
    want = heads.linear_act(x, w)
    assert _pairs() == before + 1 or torch.cuda.get_device_properties(0).multi_processor_count != 148
    assert heads.device_status(reset=True) == 0
    monkeypatch.setenv("VI_HEADS_TEST_TIMEOUT", "1")
    heads.linear_act(x, w)
    assert heads.device_status(reset=True) == 8
    monkeypatch.delenv("VI_HEADS_TEST_TIMEOUT")
    assert torch.equal(heads.linear_act(x, w), want)  # and nothing is left behind
    assert heads.device_status() == 0


# ---- incoming gradients ----
@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("M,V", [(60, 40), (900, 700)])
def test_ignored_rows_under_an_infinite_gradient(M, V, reduction, dt):
    # a scaled loss that overflows: ignored rows have no part in it
    import volume_integration.heads as heads
    g = _gen(66)
    x, w = hl.matrix(M, 24, dt, g), hl.matrix(V, 24, dt, g)
    t = torch.randint(0, V, (M,), generator=g, device="cuda")
    t[::4] = -100
    for v in (INF, NAN):
        xl = x.clone().requires_grad_(True)
        loss = heads.linear_cross_entropy(xl, w, t, reduction=reduction)
        (dx,) = torch.autograd.grad(loss, (xl,), torch.tensor(v, device="cuda"))
        assert float(dx[::4].abs().max()) == 0.0
        live = torch.arange(M, device="cuda") % 4 != 0
        assert not bool(torch.isfinite(dx[live]).any())


@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("M,K,N", [(40, 24, 30), (700, 72, 136)])
def test_c_callers_derivative_of_no_activation(M, K, N, dt):
    # dact is written for every activation, and a backward that is given it agrees with one that is not
    lib = ha.load()
    p = ctypes.c_void_p
    x, w, _, _, dy = _inputs(M, K, N, dt, "rows", False, False, 67)
    y, d = torch.empty_like(dy), torch.full_like(dy, NAN)
    stream = p(torch.cuda.current_stream().cuda_stream)
    args = (ha.DTYPE[dt], 0, ha.matrix(x), ha.matrix(w), None, None, ha.matrix(y), ha.matrix(d))
    n = lib.vi_linear_act_forward_scratch_bytes(*args)
    scratch = torch.empty(max(n, 1 << 22), device="cuda", dtype=torch.uint8)
    assert lib.vi_linear_act_forward(*args, p(scratch.data_ptr()), n, stream) == 0, lib.vi_last_error()
    hl.assert_within("y", y, hl.linear_act(x, w, None, None, "none")[0])
    grads = []
    for da in (None, ha.matrix(d)):
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        args = (ha.DTYPE[dt], 0, ha.matrix(dy), da, ha.matrix(x), ha.matrix(w), None, ha.matrix(dx), ha.matrix(dw), None)
        n = lib.vi_linear_act_backward_scratch_bytes(*args)
        scratch = torch.empty(n, device="cuda", dtype=torch.uint8)
        assert lib.vi_linear_act_backward(*args, p(scratch.data_ptr()), n, stream) == 0, lib.vi_last_error()
        grads.append((dx, dw))
    for a, b in zip(*grads):
        assert torch.equal(a, b)


# ---- tangents ----
def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwad
    import volume_integration.heads as heads
    x, w, b, r, _ = _inputs(20, 8, 9, F32, "rows", True, True, 68)
    t = torch.zeros(20, dtype=torch.int64, device="cuda")
    with fwad.dual_level():
        for i in range(4):
            v = [x, w, b, r]
            v[i] = fwad.make_dual(v[i], torch.ones_like(v[i]))
            for grad in (False, True):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    heads.linear_act(*v, activation="silu")
                if i < 3:
                    with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                        heads.linear_cross_entropy(v[0], v[1], t, v[2])
    heads.linear_act(x, w, b, r)  # and nothing is left behind
    # nor does a backward drop the tangent of what comes in
    y = heads.linear_act(x.requires_grad_(True), w, b, r)
    loss = heads.linear_cross_entropy(x, w, t, b)
    with fwad.dual_level():
        for out in (y, loss):
            dual = fwad.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, (x,), dual, retain_graph=True)
    torch.autograd.grad(y, (x,), torch.ones_like(y))


# ---- captures ----
def test_a_captured_backward_beside_a_living_eager_graph_is_refused():
    # autograd would make the default stream wait for the captured one, which ends the process
    import volume_integration.heads as heads
    x, w, b, r, dy = _inputs(200, 24, 40, F32, "rows", True, True, 74)
    t = torch.randint(0, 40, (200,), device="cuda")
    leaves = [v.detach().requires_grad_(True) for v in (x, w, b, r)]

    def act():
        y = heads.linear_act(*leaves, activation="silu")
        return torch.autograd.grad(y, leaves, dy)

    def loss():
        return torch.autograd.grad(heads.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2]), leaves[:3])
    for step, eager in ((act, lambda: heads.linear_act(*leaves, activation="silu")),
                        (loss, lambda: heads.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2]))):
        want = step()
        alive = eager()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="default stream"):
                step()
        for a, c in zip(step(), want):  # eagerly it may go on beside it
            assert torch.equal(a, c)
        del alive, graph
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, want):
            assert torch.equal(a, c)
        del graph, out


def test_a_captured_backward_beside_a_graph_of_another_stream():
    # as when the steps before the capture ran on a side stream and their result is kept
    import volume_integration.heads as heads
    x, w, b, _, dy = _inputs(200, 24, 40, F32, "rows", True, False, 75)
    leaves = [v.detach().requires_grad_(True) for v in (x, w, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = heads.linear_act(*leaves, activation="silu")
        want = torch.autograd.grad(alive, leaves, dy, retain_graph=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.autograd.grad(heads.linear_act(*leaves, activation="silu"), leaves, dy)
    graph.replay()
    torch.cuda.synchronize()
    for a, c in zip(out, want):
        assert torch.equal(a, c)
    del graph, alive


def test_a_captured_backward_to_other_leaves_than_the_living_ones():
    # the living graph is of x alone, and the capture asks for the other gradients
    import volume_integration.heads as heads
    x, w, b, r, dy = _inputs(200, 24, 40, F32, "rows", True, True, 79)
    leaves = [v.detach().requires_grad_(True) for v in (x, w, b, r)]
    want = torch.autograd.grad(heads.linear_act(*leaves, activation="silu"), leaves, dy)
    alive = heads.linear_act(leaves[0], w, b, activation="silu")
    for part in ((1, 2, 3), (3,), (2,)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = torch.autograd.grad(heads.linear_act(*leaves, activation="silu"), [leaves[i] for i in part], dy)
        graph.replay()
        torch.cuda.synchronize()
        for i, a in zip(part, out):
            assert torch.equal(a, want[i])
        del graph, out
    del alive
