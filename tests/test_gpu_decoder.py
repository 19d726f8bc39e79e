"""GPU tests of layer_norm, quantize_rows, linear_act_int8 and sample_labels against float64,
within bounds derived from the arithmetic (decoder_lib); labels have to be equal."""
import pytest
import torch

import decoder_lib as dl
import heads_lib as hl

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = dict(argvalues=[F32, F16, BF16], ids=["f32", "f16", "bf16"])
INF, NAN = float("inf"), float("nan")


def _heads():
    from volume_integration import heads
    return heads


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- layer_norm ----
def _norm_inputs(M, K, dt, order, dy_order, affine, seed, shift=1.0):
    g = _gen(seed)
    x = hl.matrix(M, K, dt, g, order)
    if shift and order != "same":
        x.add_((torch.randn(M, 1, generator=g, device="cuda") * shift).to(dt))
    dy = hl.matrix(M, K, dt, g, dy_order)
    w = (1 + 0.3 * torch.randn(K, generator=g, device="cuda")).to(dt) if affine != "none" else None
    b = (0.3 * torch.randn(K, generator=g, device="cuda")).to(dt) if affine == "both" else None
    return x, w, b, dy


def _norm_check(x, w, b, dy, eps=1e-5):
    heads = _heads()
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = heads.layer_norm(*leaves, eps=eps)
    live = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(y, live, dy)
    want = dl.layer_norm(x, w, b, eps, dy)
    assert y.dtype == x.dtype
    for name, got, ref in zip(("y", "dx", "dweight", "dbias"), (y,) + grads, want):
        hl.assert_within(name, got, ref)
    with torch.no_grad():
        assert torch.equal(heads.layer_norm(x, w, b, eps=eps), y)  # the form without gradients
    again = torch.autograd.grad(heads.layer_norm(*leaves, eps=eps), live, dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))  # the same bits
    return y, grads


NORM_CASES = [
    # M, K, order of x, order of dy, weight and bias
    (1, 1, "rows", "rows", "both"),
    (1, 256, "rows", "rows", "both"),
    (2, 3, "rows", "rows", "none"),
    (3, 8, "rows", "rows", "weight"),
    (5, 16, "padded", "rows", "both"),
    (7, 33, "odd", "rows", "both"),
    (17, 64, "rows", "steps", "both"),
    (33, 129, "rows", "image", "weight"),
    (65, 256, "rows", "rows", "none"),
    (100, 264, "rows", "same", "both"),
    (257, 512, "rows", "rows", "both"),
    (40, 515, "rows", "rows", "both"),
    (1000, 520, "padded", "rows", "both"),
    (31, 1024, "rows", "rows", "both"),
    (9, 1032, "rows", "odd", "both"),
    (300, 4096, "rows", "rows", "both"),
    (6, 4099, "rows", "rows", "both"),
    (13, 8192, "rows", "rows", "none"),
    (5, 8200, "rows", "rows", "both"),
    (3, 16384, "rows", "rows", "weight"),
    (4, 16392, "rows", "rows", "both"),
    (2, 40001, "rows", "rows", "both"),
    (20001, 24, "rows", "rows", "both"),
    (30, 70, "same", "rows", "both"),
    # images
    (1000, 1, "image", "image", "both"),
    (1024, 4, "image", "image", "both"),
    (1027, 4, "image", "image", "both"),
    (2048, 64, "image", "image", "both"),
    (2050, 64, "image", "rows", "none"),
    (513, 65, "image-odd", "image", "both"),
    (520, 100, "image", "image", "weight"),
    (514, 128, "image", "image-odd", "both"),
    (1000, 130, "image", "image", "both"),
    (256, 257, "image", "image", "both"),
    (131, 512, "image-odd", "image-odd", "both"),
    (264, 600, "image", "image", "both"),
    (77, 1100, "image", "same", "both"),
    (40000, 24, "image", "image", "both"),
    (36, 7216, "image", "image", "none"),       # few pixels of many channels
    (8194, 600, "image", "image", "both"),
    (9001, 300, "image", "image", "weight"),
    (4000, 256, "image", "image", "both"),
]


@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("M,K,order,dy_order,affine", NORM_CASES)
def test_layer_norm(M, K, order, dy_order, affine, dt):
    y, _ = _norm_check(*_norm_inputs(M, K, dt, order, dy_order, affine, M + K))
    if order == "image" and K > 1:
        assert y.t().is_contiguous()


@pytest.mark.parametrize("order", ["rows", "image"])
@pytest.mark.parametrize("K", [64, 300, 5000])
def test_layer_norm_of_rows_far_from_zero(K, order):
    # spread 1 at 10000: the mean's own rounding, 2^-24 of it and more, is taken out again
    x, w, b, dy = _norm_inputs(200, K, F32, order, "rows", "both", K, shift=10000.0)
    _norm_check(x, w, b, dy)


@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("M,K,order", [(40, 48, "rows"), (40, 2000, "rows"), (600, 40, "image"), (30, 20000, "rows"),
                                       (50, 33, "odd"), (300, 700, "image")])
def test_layer_norm_values_that_are_not_finite_stay_in_their_row(M, K, order, dt):
    heads = _heads()
    x, w, b, dy = _norm_inputs(M, K, dt, order, order if order == "image" else "rows", "both", 3)
    clean = x.clone()
    x[3, K // 2], x[7, 0], x[11, K - 1] = NAN, INF, -INF
    x.requires_grad_(True)
    y = heads.layer_norm(x, w, b)
    (dx,) = torch.autograd.grad(y, (x,), dy)
    bad = torch.zeros(M, dtype=torch.bool, device="cuda")
    bad[[3, 7, 11]] = True
    assert bool(torch.isnan(y[bad]).any(1).all()) and bool(torch.isnan(dx[bad]).any(1).all())
    want = dl.layer_norm(clean[~bad], w, b, 1e-5, dy[~bad])
    hl.assert_within("y", y[~bad], want[0])
    hl.assert_within("dx", dx[~bad], want[1])


@pytest.mark.parametrize("dt", **TYPES)
def test_layer_norm_of_constant_rows_and_eps(dt):
    heads = _heads()
    x = torch.full((70, 48), 3.0, device="cuda", dtype=dt)
    b = torch.arange(48, device="cuda").to(dt)
    assert torch.equal(heads.layer_norm(x, None, b), b.expand(70, 48))
    assert bool(torch.isnan(heads.layer_norm(x, eps=0.0)).all())  # 0 / 0, as the formula says
    for eps in (1e-12, 0.1, 100.0):
        _norm_check(*_norm_inputs(33, 56, dt, "rows", "rows", "both", 5), eps=eps)


def test_layer_norm_shapes_and_empty_batches():
    heads = _heads()
    x = torch.randn(2, 3, 5, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    y = heads.layer_norm(x, w)
    assert y.shape == x.shape
    hl.assert_within("y", y.reshape(-1, 8), dl.layer_norm(x.detach().reshape(-1, 8), w.detach(), None, 1e-5)[0])
    assert heads.layer_norm(x[0, 0, 0]).shape == (8,)
    e = torch.empty(0, 8, device="cuda", requires_grad=True)
    y = heads.layer_norm(e, w)
    de, dw = torch.autograd.grad(y, (e, w), torch.empty(0, 8, device="cuda"))
    assert y.shape == (0, 8) and de.shape == (0, 8) and torch.equal(dw, torch.zeros(8, device="cuda"))
    # a weight with strides of its own
    wide = torch.randn(16, device="cuda")
    assert torch.equal(heads.layer_norm(x.detach(), wide[::2]), heads.layer_norm(x.detach(), wide[::2].clone()))


@pytest.mark.parametrize("order,K", [("rows", 40), ("rows", 1000), ("image", 40), ("image", 600), ("rows", 20000)])
def test_layer_norm_single_gradients(order, K):
    heads = _heads()
    x, w, b, dy = _norm_inputs(50, K, F32, order, order, "both", 9)
    want = dl.layer_norm(x, w, b, 1e-5, dy)
    for which in range(3):
        leaves = [x.detach(), w.detach(), b.detach()]
        leaves[which] = leaves[which].requires_grad_(True)
        (got,) = torch.autograd.grad(heads.layer_norm(*leaves), (leaves[which],), dy)
        hl.assert_within(("dx", "dweight", "dbias")[which], got, want[1 + which])


@pytest.mark.parametrize("order,K", [("rows", 40), ("image", 40), ("rows", 1000)])
def test_layer_norm_with_a_bias_alone(order, K):
    heads = _heads()
    x, w, b, dy = _norm_inputs(50, K, F32, order, order, "both", 19)
    one = torch.ones_like(w)
    want = dl.layer_norm(x, one, b, 1e-5, dy)
    x.requires_grad_(True), b.requires_grad_(True)
    y = heads.layer_norm(x, None, b)
    dx, db = torch.autograd.grad(y, (x, b), dy)
    for name, got, ref in (("y", y, want[0]), ("dx", dx, want[1]), ("dbias", db, want[3])):
        hl.assert_within(name, got, ref)
    (db2,) = torch.autograd.grad(heads.layer_norm(x.detach(), None, b), (b,), dy)
    assert torch.equal(db, db2)


def test_layer_norm_gradients_against_differences():
    # the loss along a random direction, central differences of the kernel's own float32 results.  The step h makes
    # an error of h^2 / 6 times the third derivative along it (about 1 here: under 1e-3 of a slope of size sqrt(MK)), and the
    # values' rounding, 2^-24 of a sum of MK terms of size 1, 2 sqrt(MK) 2^-24 / h
    heads = _heads()
    x, w, b, dy = _norm_inputs(64, 96, F32, "rows", "rows", "both", 12, shift=0.0)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(heads.layer_norm(*leaves), leaves, dy)
    g, h = _gen(13), 1e-2
    for which in range(3):
        move = torch.randn(leaves[which].shape, generator=g, device="cuda")
        at = []
        for sign in (1, -1):
            args = [t.detach() for t in leaves]
            args[which] = args[which] + sign * h * move
            at.append((heads.layer_norm(*args).double() * dy.double()).sum())
        slope, want = (at[0] - at[1]) / (2 * h), (grads[which].double() * move.double()).sum()
        size = (64 * 96) ** 0.5
        assert abs(float(slope - want)) <= size * (h * h * 3 + 2 * 2 ** -24 / h) * 4, (which, float(slope), float(want))


def test_layer_norm_second_derivative_and_tangents_are_refused():
    import torch.autograd.forward_ad as fwAD
    heads = _heads()
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(heads.layer_norm(x).pow(2).sum(), (x,), create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    with fwAD.dual_level():
        d = fwAD.make_dual(torch.randn(4, 8, device="cuda"), torch.randn(4, 8, device="cuda"))
        q = heads.quantize_rows(torch.randn(5, 8, device="cuda"))
        for call in (lambda: heads.layer_norm(d), lambda: heads.quantize_rows(d), lambda: heads.linear_act_int8(d, q),
                     lambda: heads.sample_labels(d, torch.rand(4, device="cuda"))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


# ---- 8-bit integers ----
@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("M,K,order", [(1, 1, "rows"), (3, 7, "rows"), (5, 16, "rows"), (40, 256, "rows"), (33, 515, "odd"),
                                       (70, 96, "padded"), (300, 64, "image"), (257, 130, "image-odd"), (9, 5000, "rows"),
                                       (2, 70000, "rows"), (1030, 64, "image"), (600, 1000, "image"), (64, 48, "steps"),
                                       (2000, 4, "image"), (20, 33, "same")])
def test_quantize_rows(M, K, order, dt):
    x = hl.matrix(M, K, dt, _gen(M + K), order, scale=3.0)
    q, scale = _heads().quantize_rows(x)
    wq, ws = dl.quantize(x)
    assert q.dtype == torch.int8 and scale.dtype == F32
    assert torch.equal(scale, ws) and torch.equal(q, wq)
    assert q.stride(0) % 16 == 0 and q.stride(1) == 1


def test_quantize_rows_at_halves_and_ends():
    # quotients at and next to halves: 127 makes the scale 1, others make it any float
    base = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -126.5, 63.5], device="cuda")
    near = torch.nextafter(base, torch.zeros_like(base))
    rows = [base, torch.cat([base[:1], near[1:]]), base * 2.0 ** -100, base * 1e-40, base * 2.0 ** 100, base * 0.0,
            base * 3e-45, base * 2.0 ** 120]
    g = _gen(3)
    for s in (0.1, 1 / 3, 7.7, 1e-30):  # multiples of (scale / 2), as floats hold them
        top = torch.tensor(127.0 * s, device="cuda")
        scale = (top.double() / 127).float()
        k = torch.randint(-253, 254, (7,), generator=g, device="cuda")
        rows.append(torch.cat([top[None], (k.double() * scale.double() / 2).float()]))
    x = torch.stack(rows)
    q, scale = _heads().quantize_rows(x)
    wq, ws = dl.quantize(x)
    assert torch.equal(scale, ws) and torch.equal(q, wq)


@pytest.mark.parametrize("dt", **TYPES)
def test_quantize_rows_that_are_not_finite(dt):
    for order in ("rows", "image"):
        x = hl.matrix(300, 40, dt, _gen(1), order)
        x[2, 3], x[5, 0], x[9, 39], x[20] = NAN, INF, -INF, 0
        q, scale = _heads().quantize_rows(x)
        wq, ws = dl.quantize(x)
        assert torch.equal(q, wq) and torch.equal(torch.isnan(scale), torch.isnan(ws))
        fine = ~torch.isnan(ws)
        assert torch.equal(scale[fine], ws[fine]) and int(fine.sum()) == 297 and float(scale[20]) == 0


INT8_CASES = [
    # M, K, N, act, order, bias, residual
    (1, 1, 1, "none", "rows", False, False),
    (1, 256, 256, "silu", "rows", True, False),
    (2, 7, 3, "relu", "rows", True, True),
    (4, 1024, 130, "gelu", "rows", True, True),
    (7, 100, 1000, "sigmoid", "odd", True, False),
    (16, 300, 77, "silu", "rows", True, True),
    (31, 64, 64, "relu", "image", True, True),
    (127, 64, 64, "relu", "image", True, True),
    (130, 65, 9, "gelu", "image-odd", True, True),
    (129, 128, 200, "silu", "image", False, True),
    (257, 200, 257, "relu", "steps", True, False),
    (1000, 72, 136, "silu", "rows", True, True),
    (1025, 512, 320, "gelu", "padded", True, False),
    (2000, 1, 33, "sigmoid", "image", True, True),
    (4100, 130, 1, "none", "rows", True, False),
    (3000, 1000, 600, "relu", "rows", True, True),
    (2560, 384, 2560, "gelu", "image", True, True),
    (300, 5000, 70, "none", "rows", True, False),
    (40000, 64, 64, "gelu", "image", True, True),
]


@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("M,K,N,act,order,bias,residual", INT8_CASES)
def test_linear_act_int8(M, K, N, act, order, bias, residual, dt):
    heads, g = _heads(), _gen(M + K + N)
    x = hl.matrix(M, K, dt, g, order)
    w = heads.quantize_rows(hl.matrix(N, K, F32, g, scale=1.5 / K ** 0.5))
    b = hl.matrix(1, N, dt, g, scale=0.3)[0] if bias else None
    r = hl.matrix(M, N, dt, g, "image" if order.startswith("image") else "rows") if residual else None
    y = heads.linear_act_int8(x, w, b, residual=r, activation=act)
    assert y.dtype == dt and (order != "image" or N == 1 or y.t().is_contiguous())
    want = dl.linear_act_int8(*dl.quantize(x), *w, b, r, act, dt)
    hl.assert_within("y", y, want)
    # features quantised once for several layers give the same sums; another path may round differently
    y2 = heads.linear_act_int8(heads.quantize_rows(x), w, b, residual=r, activation=act, dtype=dt)
    hl.assert_within("y", y2, want)
    assert torch.equal(heads.linear_act_int8(x, w, b, residual=r, activation=act), y)
    # weights that lie otherwise
    odd = torch.zeros(N, K + 3, device="cuda", dtype=torch.int8)
    odd[:, 1:K + 1] = w[0]
    hl.assert_within("y", heads.linear_act_int8(x, (odd[:, 1:K + 1], w[1]), b, residual=r, activation=act), want)


def test_linear_act_int8_longest_sums():
    # all products of one sign: the sum of 2^17 - 1 is just within 32 bits, with a caller's -128 too
    heads, K = _heads(), (1 << 17) - 1
    for M in (1, 3, 140):
        x = torch.ones(M, K, device="cuda")
        x[1::2] = -1
        w = heads.quantize_rows(torch.ones(5, K, device="cuda"))
        y = heads.linear_act_int8(x, w)
        want = dl.linear_act_int8(*dl.quantize(x), *w, None, None, "none", F32)
        hl.assert_within("y", y, want)
    low, one = torch.full((150, K), -128, device="cuda", dtype=torch.int8), torch.ones(150, device="cuda")
    assert bool((heads.linear_act_int8((low, one), (low[:4], one[:4]), dtype=F32) == float(128 * 128 * K)).all())
    with pytest.raises(RuntimeError, match="2\\^17"):
        heads.linear_act_int8(torch.ones(2, K + 1, device="cuda"), heads.quantize_rows(torch.ones(2, K + 1, device="cuda")))


@pytest.mark.parametrize("M", [1, 6, 300])
def test_linear_act_int8_rows_that_are_not_finite(M):
    heads, g = _heads(), _gen(4)
    x = hl.matrix(M, 64, BF16, g)
    w = heads.quantize_rows(hl.matrix(48, 64, F32, g))
    clean = heads.linear_act_int8(x, w, activation="silu")
    x[M // 2, 5] = NAN
    y = heads.linear_act_int8(x, w, activation="silu")
    assert bool(torch.isnan(y[M // 2]).all())
    keep = torch.arange(M, device="cuda") != M // 2
    assert torch.equal(y[keep], clean[keep])


def test_linear_act_int8_shapes_gradients_and_empty_batches():
    heads = _heads()
    w = heads.quantize_rows(torch.randn(5, 8, device="cuda"))
    x = torch.randn(2, 3, 8, device="cuda")
    r = torch.randn(2, 3, 5, device="cuda")
    y = heads.linear_act_int8(x, w, residual=r)
    assert torch.equal(y.reshape(6, 5), heads.linear_act_int8(x.reshape(6, 8), w, residual=r.reshape(6, 5)))
    q, s = heads.quantize_rows(x)
    assert q.shape == (2, 3, 8) and s.shape == (2, 3)
    assert heads.linear_act_int8((q, s), w, dtype=BF16).shape == (2, 3, 5)
    q, s = heads.quantize_rows(x[0, 0])
    assert q.shape == (8,) and s.shape == ()
    assert heads.linear_act_int8(x[0, 0], w).shape == (5,)
    assert heads.linear_act_int8(torch.empty(0, 8, device="cuda"), w).shape == (0, 5)
    assert heads.quantize_rows(torch.empty(0, 8, device="cuda"))[0].shape == (0, 8)
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match="no backward"):
        heads.linear_act_int8(x, w)
    with torch.no_grad():
        assert heads.linear_act_int8(x, w).shape == (2, 3, 5)
    assert heads.quantize_rows(x)[1].requires_grad is False


def test_quantize_rows_into_a_part_of_a_matrix():
    # a C caller's q may be columns of a wider matrix: what lies beside them stays
    import ctypes
    import heads_abi as ha
    lib, p = ha.load(), ctypes.c_void_p
    lib.vi_quantize_rows.argtypes = [ctypes.c_int, ctypes.POINTER(ha.Matrix), ctypes.POINTER(ha.Matrix), p, p]
    for dt, order, K in ((BF16, "image", 5), (F32, "image", 130), (F16, "rows", 24), (BF16, "odd", 7), (F16, "image", 601)):
        x = hl.matrix(300, K, dt, _gen(K), order)
        wide = torch.full((300, (K + 31) // 16 * 16), 77, device="cuda", dtype=torch.int8)
        scale = torch.empty(300, device="cuda")
        q = wide[:, :K]
        assert lib.vi_quantize_rows(ha.DTYPE[dt], ha.matrix(x), ha.matrix(q), p(scale.data_ptr()),
                                    p(torch.cuda.current_stream().cuda_stream)) == 0, lib.vi_last_error()
        wq, ws = dl.quantize(x)
        assert torch.equal(q, wq) and torch.equal(scale, ws) and bool((wide[:, K:] == 77).all())


# ---- labels ----
def _labels(z, u, **settings):
    got = _heads().sample_labels(z, u, **settings)
    want = dl.sample(z, u, **settings)
    assert got.dtype == torch.int64
    assert torch.equal(got.cpu(), want), (got.cpu()[got.cpu() != want], want[got.cpu() != want])
    return got


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.3, top_k=1), dict(top_k=5), dict(top_p=0.5, temperature=1.7),
            dict(min_p=0.05), dict(top_k=40, top_p=0.9, min_p=0.01, temperature=0.8), dict(top_p=1e-6), dict(min_p=1.0),
            dict(top_k=10 ** 9, top_p=2.0)]


@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("M,V,order", [(1, 1, "rows"), (3, 2, "rows"), (5, 21, "rows"), (40, 64, "image"), (33, 150, "image-odd"),
                                       (64, 257, "odd"), (20, 1000, "rows"), (300, 33, "image"), (9, 1025, "image"),
                                       (7, 4099, "rows"), (6, 5000, "padded"), (2, 30011, "rows"), (1, 65536, "rows"),
                                       (4, 70001, "steps"), (1, 300000, "rows")])
def test_sample_labels(M, V, order, dt):
    g = _gen(M + V)
    z = hl.matrix(M, V, dt, g, order, scale=3.0)
    u = torch.rand(M, generator=g, device="cuda")
    for settings in SETTINGS:
        _labels(z, u, **settings)


@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("M,V,order", [(400, 21, "rows"), (300, 150, "image"), (50, 3000, "rows"), (12, 20000, "rows")])
def test_sample_labels_settings_by_row_and_masks(M, V, order, dt):
    g = _gen(V)
    z = hl.matrix(M, V, dt, g, order, scale=3.0)
    z[:, torch.rand(V, generator=g, device="cuda") < 0.4] = -INF
    z[1] = -INF                       # nothing left
    z[2] = torch.finfo(dt).min        # a mask of the lowest value: all equal
    z[3, V // 2] = NAN
    z[4, [1, V - 1]] = INF
    z[5] = 0.0
    z[5, ::2] = -0.0                  # equal to 0
    z[6, : V // 2] = -INF
    z[7] = -INF
    z[7, V - 1] = -1000.0             # one left
    u = torch.rand(M, generator=g, device="cuda")
    r = lambda: torch.rand(M, generator=g, device="cuda")  # noqa: E731
    t = (r() * 2 - 0.2)
    t[8] = NAN
    k = torch.randint(-2, V, (M,), generator=g, device="cuda")
    got = _labels(z, u, temperature=t, top_k=k, top_p=r() * 1.3, min_p=r() * 0.3)
    assert int(got[1]) == -1 and int(got[3]) == -1 and int(got[8]) == -1 and int(got[7]) in (-1, V - 1)
    _labels(z, u, temperature=t.clamp(min=0.1).nan_to_num(1.0))
    _labels(z, u, top_p=r())
    _labels(z, u, top_k=k)


@pytest.mark.parametrize("V", [3, 40, 700, 5000])
def test_sample_labels_ends_of_u_and_ties(V):
    g = _gen(V)
    z = (hl.matrix(64, V, F32, g, scale=1.0) * 2).round() / 2  # many equal logits
    u = torch.rand(64, generator=g, device="cuda")
    u[0], u[1], u[2], u[3] = 0.0, 1 - 2.0 ** -24, 1.0, 2.0 ** -24
    for settings in (dict(), dict(top_k=2), dict(top_k=V // 2 + 1), dict(top_p=0.6), dict(top_k=V // 2 + 1, top_p=0.55),
                     dict(min_p=0.3)):
        _labels(z, u, **settings)
    for V_u, u_same in ((-3.0, 0.0), (NAN, 0.0)):  # under 0, or no number: 0
        low = _heads().sample_labels(z, torch.full_like(u, V_u), top_k=2)
        assert torch.equal(low, _heads().sample_labels(z, torch.full_like(u, u_same), top_k=2))
        assert torch.equal(_heads().sample_labels(z, torch.full_like(u, V_u)), _heads().sample_labels(z, torch.full_like(u, u_same)))
    z[:] = 0.25  # all equal: the front of the order is the front of the row
    got = _labels(z, u, top_k=2)
    assert int(got.max()) <= 1


def test_sample_labels_rows_are_drawn_by_their_share():
    z = torch.tensor([0.3, 2.0, -1.0, 1.1, 0.0], device="cuda")
    u = (torch.arange(100000, device="cuda") + 0.5) / 100000
    got = _heads().sample_labels(z.expand(100000, 5), u)
    share = torch.bincount(got, minlength=5).double() / 100000
    assert float((share - torch.softmax(z.double(), 0)).abs().max()) <= 2e-5


def test_sample_labels_of_more_long_rows_than_are_drawn_at_a_time():
    g = _gen(8)
    z = hl.matrix(16390, 8200, BF16, g, scale=3.0)
    u = torch.rand(16390, generator=g, device="cuda")
    got = _heads().sample_labels(z, u, top_k=9)
    at = torch.tensor([0, 1, 16382, 16383, 16384, 16385, 16389], device="cuda")
    assert torch.equal(got[at].cpu(), dl.sample(z[at], u[at], top_k=9))


@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("M,V", [(3, 9000), (200, 20011), (2, 100003)])
def test_sample_labels_of_long_rows_of_every_kind(M, V, dt):
    # flat and peaked, sorted both ways, constant, with all mass in front or behind: guesses from a sample go wrong here
    g = _gen(V)
    kinds = [hl.matrix(M, V, dt, g, scale=0.01), hl.matrix(M, V, dt, g, scale=30.0),
             hl.matrix(M, V, dt, g, scale=3.0).sort(1).values, hl.matrix(M, V, dt, g, scale=3.0).sort(1, descending=True).values,
             torch.full((M, V), -2.5, device="cuda", dtype=dt)]
    spike = hl.matrix(M, V, dt, g, scale=1.0)
    spike[:, V - 1] = 40.0
    kinds.append(spike)
    rows = slice(0, 3)
    for z in kinds:
        u = torch.rand(M, generator=g, device="cuda")
        for settings in (dict(), dict(top_p=0.9), dict(top_p=0.999, temperature=1.9), dict(top_k=V // 2), dict(top_k=3, top_p=0.4),
                         dict(min_p=0.001), dict(min_p=0.9, temperature=0.4), dict(temperature=0.0)):
            got = _heads().sample_labels(z, u, **settings)
            assert torch.equal(got[rows].cpu(), dl.sample(z[rows], u[rows], **settings)), settings


def test_sample_labels_shapes():
    heads = _heads()
    z, u = torch.randn(2, 3, 9, device="cuda"), torch.rand(2, 3, device="cuda")
    t = torch.rand(2, 3, device="cuda")
    got = heads.sample_labels(z, u, temperature=t)
    assert got.shape == (2, 3)
    assert torch.equal(got.reshape(-1), heads.sample_labels(z.reshape(6, 9), u.reshape(6), temperature=t.reshape(6)))
    assert heads.sample_labels(z[0, 0], u[0, 0]).shape == ()
    assert heads.sample_labels(torch.empty(0, 4, device="cuda"), torch.empty(0, device="cuda")).shape == (0,)
    z.requires_grad_(True)
    assert torch.equal(heads.sample_labels(z, u, temperature=t), got)


# ---- together, and how calls are made ----
@pytest.mark.parametrize("dt", **TYPES)
def test_a_decoder_trained_and_served(dt):
    # features of an image through layer norm, a dense layer with its residual, the label loss; then the display form
    heads, g = _heads(), _gen(21)
    M, K, V = 2000, 48, 30
    x = hl.matrix(M, K, dt, g, "image")
    nw, nb = (1 + 0.1 * torch.randn(K, generator=g, device="cuda")).to(dt), (0.1 * torch.randn(K, generator=g, device="cuda")).to(dt)
    w = hl.matrix(K, K, dt, g, scale=K ** -0.5)
    wv = hl.matrix(V, K, dt, g, scale=2 * K ** -0.5)
    t = torch.randint(0, V, (M,), generator=g, device="cuda")
    leaves = [v.detach().requires_grad_(True) for v in (x, nw, nb, w, wv)]
    h = heads.layer_norm(*leaves[:3])
    loss = heads.linear_cross_entropy(heads.linear_act(h, leaves[3], residual=leaves[0], activation="gelu"), leaves[4], t)
    grads = torch.autograd.grad(loss, leaves)
    ref = [v.detach().double().requires_grad_(True) for v in (x, nw, nb, w, wv)]
    hr = torch.nn.functional.layer_norm(ref[0], (K,), ref[1], ref[2], 1e-5)
    lr = torch.nn.functional.cross_entropy((torch.nn.functional.gelu(hr @ ref[3].t()) + ref[0]) @ ref[4].t(), t)
    want = torch.autograd.grad(lr, ref)
    # roundings to the type on the way (h, the layer's result, their gradients, act', the sum): at most a dozen of a half
    # step each, relative to the sizes that are summed; compared by norms
    tol = 12 * torch.finfo(dt).eps / 2 + 1e-5
    assert abs(float(loss) - float(lr)) <= tol * max(1.0, float(lr))
    for got, ref_g in zip(grads, want):
        assert float((got.double() - ref_g).norm() / ref_g.norm()) <= tol
    with torch.no_grad():
        w8, wv8 = heads.quantize_rows(w), heads.quantize_rows(wv)
        h = heads.layer_norm(x, nw, nb)
        f = heads.linear_act_int8(h, w8, residual=x, activation="gelu")
        z = heads.linear_act_int8(f, wv8)
        u = torch.rand(M, generator=g, device="cuda")
        label = heads.sample_labels(z, u, temperature=0.7, top_p=0.9)
    hl.assert_within("f", f, dl.linear_act_int8(*dl.quantize(h), *w8, None, x, "gelu", dt))
    hl.assert_within("z", z, dl.linear_act_int8(*dl.quantize(f), *wv8, None, None, "none", dt))
    assert torch.equal(label.cpu(), dl.sample(z, u, temperature=0.7, top_p=0.9))


def _serve(heads, x, nw, w8, u):
    z = heads.linear_act_int8(heads.layer_norm(x, nw), w8, activation="silu")
    return z, heads.sample_labels(z, u, top_k=7, top_p=0.8)


@pytest.mark.parametrize("M", [1, 5, 700])
def test_captured_replayed_and_on_two_streams(M):
    heads, g = _heads(), _gen(31)
    K, V = 64, 40
    x, u = hl.matrix(M, K, BF16, g), torch.rand(M, generator=g, device="cuda")
    nw = hl.matrix(1, K, BF16, g)[0]
    w8 = heads.quantize_rows(hl.matrix(V, K, F32, g))
    want = _serve(heads, x, nw, w8, u)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        xs, us = torch.zeros_like(x), torch.zeros_like(u)
        with torch.cuda.graph(graph):
            out = _serve(heads, xs, nw, w8, us)
        graphs.append((graph, xs, us, out))
    for graph, xs, us, out in graphs:
        xs.copy_(x), us.copy_(u)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (graph, *_r) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for graph, xs, us, out in graphs:
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    # eager, two at once, again and again
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(_serve(heads, x, nw, w8, u))
    torch.cuda.synchronize()
    for out in outs:
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_a_training_step_captured_and_replayed():
    heads = _heads()
    x, w, b, dy = _norm_inputs(600, 96, BF16, "rows", "rows", "both", 33)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = torch.autograd.grad(heads.layer_norm(*leaves), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = torch.autograd.grad(heads.layer_norm(*leaves), leaves, dy)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_a_captured_backward_beside_a_living_eager_graph_is_refused():
    heads = _heads()
    x = torch.randn(300, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    alive = heads.layer_norm(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(heads.layer_norm(x, w).sum(), (x, w))
    del alive
    torch.cuda.synchronize()
    y = heads.layer_norm(x, w)
    torch.autograd.grad(y.sum(), (x, w))


def test_results_beyond_2_31_elements():
    heads = _heads()
    M, K = (1 << 21) + 3, 1032  # 2^31 elements and more
    x = torch.empty(M, K, device="cuda", dtype=BF16)
    x.normal_(generator=_gen(2))
    y = heads.layer_norm(x)
    at = slice(M - 5, M)
    hl.assert_within("y", y[at], dl.layer_norm(x[at], None, None, 1e-5)[0])
    del y
    q, scale = heads.quantize_rows(x)
    wq, ws = dl.quantize(x[at])
    assert torch.equal(q[at], wq) and torch.equal(scale[at], ws)
    del q
    u = torch.rand(M, generator=_gen(4), device="cuda")
    got = heads.sample_labels(x, u, top_p=0.9)
    assert torch.equal(got[at].cpu(), dl.sample(x[at], u[at], top_p=0.9))


def test_results_of_images_beyond_2_31_elements():
    heads = _heads()
    M, K = (1 << 25) + 8, 64
    x = torch.empty(K, M, device="cuda", dtype=BF16).normal_(generator=_gen(5)).t()
    at = slice(M - 5, M)
    y = heads.layer_norm(x)
    hl.assert_within("y", y[at], dl.layer_norm(x[at], None, None, 1e-5)[0])
    del y
    w8 = heads.quantize_rows(torch.randn(64, K, generator=_gen(6), device="cuda"))
    y = heads.linear_act_int8(x, w8)
    hl.assert_within("y", y[at], dl.linear_act_int8(*dl.quantize(x[at]), *w8, None, None, "none", BF16))
    del y
    u = torch.rand(M, generator=_gen(4), device="cuda")
    got = heads.sample_labels(x, u, min_p=0.02)
    assert torch.equal(got[at].cpu(), dl.sample(x[at], u[at], min_p=0.02))


def test_waits_that_run_out_are_reported(monkeypatch):
    # the first copy is never issued: a limit on every wait, then the status word; no fault
    heads, g = _heads(), _gen(41)
    w = heads.quantize_rows(hl.matrix(200, 64, F32, g))
    w64 = (w[0][:64], w[1][:64])
    x, z = hl.matrix(33000, 64, BF16, g, "image"), hl.matrix(1024, 20, F16, g, "image")
    u = torch.rand(1024, generator=g, device="cuda")
    calls = (lambda: heads.linear_act_int8(x, w), lambda: heads.linear_act_int8(x, w64, activation="gelu"),
             lambda: heads.linear_act_int8(x.contiguous(), w64), lambda: heads.sample_labels(z, u))
    before = [call() for call in calls]
    assert heads.device_status() == 0
    monkeypatch.setenv("VI_HEADS_TEST_TIMEOUT", "1")
    for call in calls:
        call()
        assert heads.device_status(reset=True) == 8
    monkeypatch.delenv("VI_HEADS_TEST_TIMEOUT")
    for call, want in zip(calls, before):
        assert torch.equal(call(), want)
    assert heads.device_status() == 0


def test_heads_status_stays_clear():
    assert _heads().device_status() == 0


@pytest.mark.parametrize("dt", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("M,K,N,act,order,bias,residual", [
    (32768, 64, 64, "none", "rows", True, False),
    (32769, 64, 33, "relu", "rows", False, True),
    (40001, 8, 64, "silu", "rows", True, True),
    (33000, 40, 5, "gelu", "padded", True, False),
    (32768, 64, 64, "gelu", "image", True, True),
    (32770, 33, 64, "sigmoid", "image", True, True),
    (100002, 5, 40, "silu", "image", False, False),
    (38001, 64, 64, "none", "image-odd", True, True),  # not in whole pairs
])
def test_linear_act_int8_of_few_features(M, K, N, act, order, bias, residual, dt):
    heads, g = _heads(), _gen(M + K + N)
    x = hl.matrix(M, K, dt, g, order)
    if K > 1:
        x[M - 1, 1], x[7, 0], x[M // 2] = NAN, INF, 0
    w = heads.quantize_rows(hl.matrix(N, K, F32, g, scale=1.5 / K ** 0.5))
    b = hl.matrix(1, N, dt, g, scale=0.3)[0] if bias else None
    r = hl.matrix(M, N, dt, g, "image" if order.startswith("image") else "rows") if residual else None
    y = heads.linear_act_int8(x, w, b, residual=r, activation=act)
    fine = torch.ones(M, dtype=torch.bool, device="cuda")
    fine[[7, M - 1]] = False
    assert bool(torch.isnan(y[~fine]).all())
    q, s = dl.quantize(x)
    value, bound = dl.linear_act_int8(q, s, *w, b, r, act, dt)
    hl.assert_within("y", y[fine], (value[fine], bound[fine]))
