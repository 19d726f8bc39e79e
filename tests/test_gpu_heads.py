"""GPU tests of the per-pixel heads (linear_act, linear_cross_entropy) against
float64, within bounds derived from the arithmetic (heads_lib)."""
import pytest
import torch

import heads_lib as hl

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _act_inputs(M, K, N, dt, order, bias, residual, seed):
    g = _gen(seed)
    x = hl.matrix(M, K, dt, g, order)
    w = hl.matrix(N, K, dt, g, scale=1.5 / K ** 0.5)
    b = hl.matrix(1, N, dt, g, scale=0.3)[0] if bias else None
    r = hl.matrix(M, N, dt, g, "image" if order.startswith("image") else "rows") if residual else None
    dy = hl.matrix(M, N, dt, g, "image" if order == "image" else "rows")
    return x, w, b, r, dy


def _act_check(x, w, b, r, dy, act):
    import volume_integration.heads as heads
    leaves = [t.detach().requires_grad_(True) for t in (x, w)]
    bl = b.detach().requires_grad_(True) if b is not None else None
    rl = r.detach().requires_grad_(True) if r is not None else None
    y = heads.linear_act(leaves[0], leaves[1], bl, rl, act)
    live = leaves + [t for t in (bl, rl) if t is not None]
    grads = list(torch.autograd.grad(y, live, dy))
    want = hl.linear_act(x, w, b, r, act, dy)
    hl.assert_within("y", y, want[0])
    hl.assert_within("dx", grads[0], want[1])
    hl.assert_within("dweight", grads[1], want[2])
    if b is not None:
        hl.assert_within("dbias", grads[2], want[3])
    if r is not None:
        torch.testing.assert_close(grads[-1], dy, rtol=0, atol=0)
    with torch.no_grad():
        z = heads.linear_act(x, w, b, r, act)
    assert z.dtype == x.dtype and torch.equal(z, y)  # the form without gradients
    return y


ACT_CASES = [
    # M, K, N, act, order, bias, residual
    (1, 1, 1, "none", "rows", False, False),
    (1, 256, 256, "silu", "rows", True, False),
    (2, 7, 3, "relu", "rows", True, True),
    (3, 64, 130, "gelu", "rows", False, True),
    (5, 129, 64, "sigmoid", "odd", True, False),
    (16, 300, 77, "silu", "rows", True, True),
    (17, 33, 1000, "gelu", "padded", True, False),
    (127, 64, 64, "relu", "image", True, True),
    (128, 4, 64, "sigmoid", "image", True, False),
    (129, 8, 65, "silu", "image", False, True),
    (130, 65, 9, "gelu", "image-odd", True, True),
    (257, 200, 257, "relu", "steps", True, False),
    (300, 96, 40, "none", "same", True, True),
    (1000, 72, 136, "silu", "rows", True, True),
    (1025, 512, 320, "gelu", "rows", True, False),
    (2000, 1, 33, "sigmoid", "image", True, True),
    (4100, 130, 1, "none", "rows", True, False),
    (40000, 24, 16, "relu", "image", True, False),
]


@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,K,N,act,order,bias,residual", ACT_CASES)
def test_linear_act(M, K, N, act, order, bias, residual, dt):
    _act_check(*_act_inputs(M, K, N, dt, order, bias, residual, M + K + N), act)


@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", hl.ACTS)
def test_linear_act_every_activation(act, dt):
    _act_check(*_act_inputs(200, 48, 72, dt, "rows", True, True, 3), act)


@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,K,N,act,order,residual,dy_order", [
    (1031, 3, 300, "gelu", "image", True, "image"),      # more channels than one backward pass keeps
    (2052, 7, 256, "silu", "image", False, "image"),
    (517, 5, 20, "sigmoid", "image-odd", True, "image-odd"),
    (4096, 4, 64, "relu", "image", False, "rows"),       # the gradient comes in the other order
    (3, 2, 9, "gelu", "image", True, "image"),
    (700, 8, 130, "none", "image", True, "image"),
    (900, 9, 40, "silu", "image", False, "image"),       # one channel too many for the narrow path
    (20001, 4, 16, "gelu", "image", False, "image"),
])
def test_linear_act_images_of_few_channels(M, K, N, act, order, residual, dy_order, dt):
    x, w, b, r, _ = _act_inputs(M, K, N, dt, order, True, residual, M + N)
    dy = hl.matrix(M, N, dt, _gen(M), dy_order)
    y = _act_check(x, w, b, r, dy, act)
    assert y.t().is_contiguous() or order != "image"


@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_relu_keeps_its_result_and_nothing_else(dt):
    # the backward reads relu's derivative off the result, which an in-place change would spoil: torch says so
    import volume_integration.heads as heads
    x, w, b, _, dy = _act_inputs(1200, 40, 200, dt, "rows", True, False, 42)
    x.requires_grad_(True)
    y = heads.linear_act(x, w, b, activation="relu")
    used = torch.cuda.memory_allocated()
    z = heads.linear_act(x, w, b, activation="relu")
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - used <= z.numel() * z.element_size() + 4096
    (dx,) = torch.autograd.grad(y, (x,), dy)
    hl.assert_within("dx", dx, hl.linear_act(x.detach(), w, b, None, "relu", dy)[1])
    z.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(z, (x,), dy)


def test_backward_without_the_kept_derivative():
    # a C ABI caller that kept no act': it is computed again from x, weight and bias
    import ctypes
    import heads_abi as ha
    lib = ha.load()
    p = ctypes.c_void_p
    for dt, order in ((BF16, "rows"), (F32, "odd"), (F16, "image")):
        x, w, b, _, dy = _act_inputs(300, 40, 70, dt, order, True, False, 41)
        dx, dw, db = torch.empty(300, 40, device="cuda", dtype=dt), torch.empty_like(w), torch.empty_like(b)
        args = (ha.DTYPE[dt], 2, ha.matrix(dy), None, ha.matrix(x), ha.matrix(w), p(b.data_ptr()), ha.matrix(dx),
                ha.matrix(dw), p(db.data_ptr()))
        n = lib.vi_linear_act_backward_scratch_bytes(*args)
        assert n > 0, lib.vi_last_error()
        scratch = torch.empty(n, device="cuda", dtype=torch.uint8)
        rc = lib.vi_linear_act_backward(*args, p(scratch.data_ptr()), n, p(torch.cuda.current_stream().cuda_stream))
        assert rc == 0, lib.vi_last_error()
        want = hl.linear_act(x, w, b, None, "silu", dy)
        for name, got, ref in (("dx", dx, want[1]), ("dweight", dw, want[2]), ("dbias", db, want[3])):
            hl.assert_within(name, got, ref)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
def test_linear_act_memory_order_of_the_result(dt):
    import volume_integration.heads as heads
    g = _gen(1)
    image = hl.matrix(8, 6 * 50, dt, g).view(8, 6, 50)
    w = hl.matrix(24, 8, dt, g)
    y = heads.linear_act(image.permute(1, 2, 0), w)  # [H, W, K] view of a [K, H, W] image
    assert y.shape == (6, 50, 24) and y.permute(2, 0, 1).is_contiguous()
    hl.assert_within("y", y.reshape(300, 24), hl.linear_act(image.flatten(1).t(), w, None, None, "none")[0])
    assert heads.linear_act(image.flatten(1).t().contiguous(), w).is_contiguous()
    v = heads.linear_act(image[:, 0, 0], w)
    assert v.shape == (24,)


@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_linear_act_strided_weight_and_shared_inputs(dt):
    # a transposed weight, a bias shared by expansion, the same tensor as input and residual
    import volume_integration.heads as heads
    g = _gen(5)
    x = hl.matrix(70, 40, dt, g).requires_grad_(True)
    wt = hl.matrix(40, 40, dt, g, scale=0.2).t().requires_grad_(True)
    one = hl.matrix(1, 1, dt, g)[0].requires_grad_(True)
    dy = hl.matrix(70, 40, dt, g)
    y = heads.linear_act(x, wt, one.expand(40), x, "silu")
    gx, gw, g1 = torch.autograd.grad(y, (x, wt, one), dy)
    want = hl.linear_act(x.detach(), wt.detach(), one.detach().expand(40), x.detach(), "silu", dy)
    hl.assert_within("y", y, want[0])
    v, bound = want[1]
    v = v + dy.double()  # both paths into x
    hl.assert_within("dx", gx, (v, bound + hl.last(dt, v.abs() + bound)))
    hl.assert_within("dweight", gw, want[2])
    v, bound = want[3][0].sum(), want[3][1].sum()
    # torch adds the 40 gradients in float32 and rounds once
    hl.assert_within("shared bias", g1[0], (v, bound + hl.last(dt, v.abs() + bound) + 64 * hl.E * want[3][0].abs().sum()))


@pytest.mark.parametrize("dt", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("M,K,N,act,order,bias,residual", [
    (4100, 72, 1100, "silu", "rows", True, True),
    (4099, 136, 1030, "gelu", "image", True, True),   # few more rows than tiles, an odd image
    (9000, 1100, 700, "relu", "padded", True, False),
    (5000, 2100, 1000, "none", "rows", False, False),
])
def test_linear_act_tiles_of_two_blocks(M, K, N, act, order, bias, residual, dt):
    # enough tiles that every product takes 256 x 256 ones, made by pairs of blocks
    _act_check(*_act_inputs(M, K, N, dt, order, bias, residual, M + K + N), act)


def test_linear_act_gradient_against_differences():
    # float32: (f(p + h) - f(p - h)) / 2h of the kernel's own output, h = 2^-6, with a
    # smooth activation.  Truncation: h^2/6 times the third derivative along the direction;
    # |gelu'''| <= 2 and |direction's dz| <= |v|_1-like sizes, computed below.
    import volume_integration.heads as heads
    g = _gen(6)
    x, w = hl.matrix(33, 12, F32, g), hl.matrix(20, 12, F32, g, scale=0.3)
    b = hl.matrix(1, 20, F32, g)[0]
    dy = hl.matrix(33, 20, F32, g)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(heads.linear_act(*leaves, activation="gelu"), leaves, dy)
    h = 2.0 ** -6
    for i, base in enumerate((x, w, b)):
        d = torch.randn(base.shape, generator=g, device="cuda")
        d = d / d.abs().max()
        p = [x, w, b]

        def f(sign):
            q = list(p)
            q[i] = base + sign * h * d
            return (heads.linear_act(*q, activation="gelu").double() * dy.double()).sum()
        got = (f(1) - f(-1)) / (2 * h)
        want = (grads[i].double() * d.double()).sum()
        dz = (lambda: d.double() @ w.double().t(), lambda: x.double() @ d.double().t(),
              lambda: d.double().expand(33, 20))[i]()
        y, by = hl.linear_act(x, w, b, None, "gelu")[0]
        slack = h * h / 6 * 2.0 * (dy.double().abs() * dz.abs() ** 3).sum() + \
            (dy.double().abs() * (by * 1.5 + hl.E)).sum() / h
        assert abs(float(got - want)) <= float(slack), (i, float(got), float(want), float(slack))


@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_linear_act_no_rows(dt):
    import volume_integration.heads as heads
    x = torch.empty(0, 5, device="cuda", dtype=dt, requires_grad=True)
    w = torch.ones(7, 5, device="cuda", dtype=dt, requires_grad=True)
    b = torch.ones(7, device="cuda", dtype=dt, requires_grad=True)
    y = heads.linear_act(x, w, b, activation="relu")
    assert y.shape == (0, 7)
    gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
    assert gx.shape == (0, 5) and float(gw.abs().sum()) == 0 and float(gb.abs().sum()) == 0


@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_linear_act_not_finite_stays_in_its_rows_and_columns(dt):
    import volume_integration.heads as heads
    g = _gen(8)
    x, w, b, r, dy = _act_inputs(150, 40, 70, dt, "rows", True, True, 8)
    want = heads.linear_act(x, w, b, r, "gelu")
    x2, b2, r2 = x.clone(), b.clone(), r.clone()
    x2[3, 5], x2[140, 0] = float("nan"), float("inf")
    b2[69] = float("inf")
    r2[10, 0] = float("-inf")
    y = heads.linear_act(x2, w, b2, r2, "gelu")
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[3], bad[140], bad[:, 69], bad[10, 0] = True, True, True, True
    assert torch.equal(y[~bad], want[~bad])
    assert bool(torch.isnan(y[3]).all()) and not bool(torch.isfinite(y[:, 69]).any())
    assert float(y[10, 0]) == float("-inf")


def test_linear_act_writes_nothing_beside_its_result():
    # the result of one call lies between guards: torch's allocator packs these views
    from volume_integration import _C  # noqa: F401
    import ctypes
    import heads_abi as ha
    lib = ha.load()
    for dt, M, K, N, image in ((BF16, 129, 40, 67, False), (F32, 65, 5, 33, True), (F16, 200, 64, 72, True)):
        g = _gen(M)
        x, w = hl.matrix(M, K, dt, g, "image" if image else "rows"), hl.matrix(N, K, dt, g)
        pad = 7
        if image:
            guard = torch.full((N + 2, M + pad), 7.0, device="cuda", dtype=dt)
            y = guard[1:N + 1, :M].t()
        else:
            guard = torch.full((M + 2, N + pad), 7.0, device="cuda", dtype=dt)
            y = guard[1:M + 1, :N]
        mx, mw, my = ha.matrix(x), ha.matrix(w), ha.matrix(y)
        n = lib.vi_linear_act_forward_scratch_bytes(ha.DTYPE[dt], 0, mx, mw, None, None, my, None)
        assert n > 0, lib.vi_last_error()
        scratch = torch.empty(n, device="cuda", dtype=torch.uint8)
        rc = lib.vi_linear_act_forward(ha.DTYPE[dt], 0, mx, mw, None, None, my, None, ctypes.c_void_p(scratch.data_ptr()),
                                       n, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == 0, lib.vi_last_error()
        hl.assert_within("y", y, hl.linear_act(x, w, None, None, "none")[0])
        y.fill_(7.0)
        assert bool((guard == 7.0).all())


# ---------------------------------------------------------------------------
def _ce_inputs(M, K, V, dt, order, bias, ignored, seed, spread=3.0):
    g = _gen(seed)
    x = hl.matrix(M, K, dt, g, order)
    w = hl.matrix(V, K, dt, g, scale=spread / K ** 0.5)
    b = hl.matrix(1, V, dt, g, scale=0.5)[0] if bias else None
    t = torch.randint(0, V, (M,), generator=g, device="cuda")
    t[torch.rand(M, generator=g, device="cuda") < ignored] = -100
    return x, w, b, t


def _ce_check(x, w, b, t, reduction, seed=0, ignore=-100):
    import volume_integration.heads as heads
    g = _gen(seed)
    leaves = [v.detach().requires_grad_(True) for v in (x, w) + ((b,) if b is not None else ())]
    loss = heads.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2] if b is not None else None, ignore, reduction)
    dl = torch.randn(loss.shape, generator=g, device="cuda")
    grads = torch.autograd.grad(loss, leaves, dl)
    want = hl.linear_ce(x, w, b, t, ignore, reduction, dl)
    assert loss.dtype == torch.float32
    hl.assert_within("loss", loss, want[0])
    for name, got, ref in zip(("dx", "dweight", "dbias"), grads, want[1:]):
        hl.assert_within(name, got, ref)
    with torch.no_grad():
        again = heads.linear_cross_entropy(x, w, t, b, ignore, reduction)
    assert torch.equal(again, loss)


CE_CASES = [
    # M, K, V, order, bias, ignored, reduction
    (1, 1, 1, "rows", False, 0.0, "sum"),
    (1, 256, 1000, "rows", True, 0.0, "none"),
    (2, 5, 2, "rows", True, 0.0, "mean"),
    (16, 64, 21, "image", True, 0.3, "mean"),
    (127, 40, 63, "rows", False, 0.5, "sum"),
    (128, 64, 64, "image", True, 0.0, "none"),
    (129, 72, 65, "odd", True, 0.2, "none"),
    (200, 33, 257, "steps", True, 0.1, "mean"),
    (300, 8, 150, "image-odd", False, 0.1, "none"),
    (1000, 64, 1030, "rows", True, 0.05, "mean"),
    (513, 200, 5003, "rows", True, 0.0, "sum"),
    (20000, 16, 21, "image", True, 0.3, "mean"),
    (64, 128, 40001, "rows", True, 0.0, "none"),
]


@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,K,V,order,bias,ignored,reduction", CE_CASES)
def test_linear_cross_entropy(M, K, V, order, bias, ignored, reduction, dt):
    _ce_check(*_ce_inputs(M, K, V, dt, order, bias, ignored, M + V), reduction)


@pytest.mark.parametrize("dt,M,V", [(F32, 30000, 4001), (F16, 40000, 9001), (BF16, 40000, 9001)],
                         ids=["f32", "f16", "bf16"])
def test_linear_cross_entropy_in_several_pieces(dt, M, V):
    # the gradient of the logits of this many rows does not exist at once
    _ce_check(*_ce_inputs(M, 24, V, dt, "rows", True, 0.1, 31), "mean")


@pytest.mark.parametrize("dt", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("M,K,V,order,reduction", [(4100, 300, 4100, "rows", "mean"), (3001, 130, 9999, "image", "none")])
def test_linear_cross_entropy_tiles_of_two_blocks(M, K, V, order, reduction, dt):
    _ce_check(*_ce_inputs(M, K, V, dt, order, True, 0.1, 32), reduction)


@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_linear_cross_entropy_large_logits(dt):
    # spread of 40: probabilities of 1 beside ones far below float16's range
    _ce_check(*_ce_inputs(200, 64, 500, dt, "rows", True, 0.0, 4, spread=40.0), "mean")


@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_linear_cross_entropy_masked_classes(dt):
    # -inf and the type's lowest value in the bias take classes out of the vocabulary
    x, w, b, t = _ce_inputs(140, 32, 300, dt, "rows", True, 0.1, 9)
    t = torch.where(t >= 0, t % 100, t)
    b[100:200] = float("-inf")
    b[200:] = torch.finfo(dt).min
    import volume_integration.heads as heads
    bl = b.clone().requires_grad_(True)
    loss = heads.linear_cross_entropy(x, w, t, bl)
    (db,) = torch.autograd.grad(loss, (bl,))
    want = hl.linear_ce(x, w[:100], b[:100], t, -100, "mean", torch.ones((), device="cuda"))
    hl.assert_within("loss", loss, want[0])
    hl.assert_within("dbias", db[:100], want[3])
    assert float(db[100:].abs().max()) == 0.0


@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_linear_cross_entropy_every_class_at_the_lowest_value(dt):
    # a row whose classes are all masked by the type's lowest value has them all equal
    import volume_integration.heads as heads
    V = 40
    x = torch.zeros(130, 16, device="cuda", dtype=dt)
    w = torch.ones(V, 16, device="cuda", dtype=dt)
    b = torch.full((V,), torch.finfo(dt).min, device="cuda", dtype=dt).requires_grad_(True)
    t = torch.arange(130, device="cuda") % V
    loss = heads.linear_cross_entropy(x, w, t, b, reduction="none")
    want = torch.full((130,), V, device="cuda", dtype=torch.float64).log()
    hl.assert_within("loss", loss, (want, 64 * hl.E * want))
    (db,) = torch.autograd.grad(loss.sum(), (b,))
    counts = torch.bincount(t, minlength=V).double()
    value = 130 / V - counts
    bound = (130 + 64) * hl.E * (130 / V + counts) + hl.half_step(dt) * (130 / V + counts)
    hl.assert_within("dbias", db, (value, bound + hl.last(dt, value.abs() + bound)))


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_linear_cross_entropy_ignored_rows_may_hold_anything(dt, reduction):
    x, w, b, t = _ce_inputs(150, 40, 33, dt, "rows", True, 0.0, 10)
    t[[0, 77, 149]] = -100
    x[0], x[77], x[149, 3] = float("nan"), float("inf"), float("-inf")
    _ce_check(x, w, b, t, reduction)


@pytest.mark.parametrize("dt", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_linear_cross_entropy_every_row_ignored(dt):
    import volume_integration.heads as heads
    x, w, b, t = _ce_inputs(100, 24, 50, dt, "rows", True, 0.0, 11)
    t[:] = 7
    for reduction in ("none", "sum", "mean"):
        leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
        loss = heads.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], ignore_index=7, reduction=reduction)
        if reduction == "mean":
            assert bool(torch.isnan(loss))
        else:
            assert float(loss.abs().sum()) == 0.0
        for g in torch.autograd.grad(loss.sum(), leaves):
            assert float(g.abs().max()) == 0.0


def test_linear_cross_entropy_target_outside_the_vocabulary():
    import volume_integration.heads as heads
    x, w, b, t = _ce_inputs(100, 24, 50, BF16, "rows", True, 0.0, 12)
    t[3], t[4], t[5] = 50, -1, 2 ** 40
    rows = heads.linear_cross_entropy(x, w, t, b, reduction="none")
    assert torch.isnan(rows).nonzero().flatten().tolist() == [3, 4, 5]
    assert bool(torch.isnan(heads.linear_cross_entropy(x, w, t, b)))
    xl = x.clone().requires_grad_(True)
    rows = heads.linear_cross_entropy(xl, w, t, b, reduction="none")
    (dx,) = torch.autograd.grad(rows.sum(), (xl,))
    assert torch.isnan(dx).any(1).nonzero().flatten().tolist() == [3, 4, 5]


def test_linear_cross_entropy_no_rows():
    import volume_integration.heads as heads
    x = torch.empty(0, 5, device="cuda", requires_grad=True)
    w = torch.ones(7, 5, device="cuda", requires_grad=True)
    t = torch.empty(0, device="cuda", dtype=torch.int64)
    assert heads.linear_cross_entropy(x, w, t, reduction="none").shape == (0,)
    assert bool(torch.isnan(heads.linear_cross_entropy(x, w, t)))
    loss = heads.linear_cross_entropy(x, w, t, reduction="sum")
    assert float(loss) == 0.0
    gx, gw = torch.autograd.grad(loss, (x, w))
    assert gx.shape == (0, 5) and float(gw.abs().max()) == 0.0


def test_linear_cross_entropy_shapes_and_a_row_of_infinite_gradient():
    import volume_integration.heads as heads
    x, w, b, t = _ce_inputs(60, 24, 50, BF16, "rows", True, 0.0, 13)
    loss = heads.linear_cross_entropy(x.view(3, 20, 24), w, t.view(3, 20), b, reduction="none")
    assert loss.shape == (3, 20)
    hl.assert_within("loss", loss.flatten(), hl.linear_ce(x, w, b, t, -100, "none")[0])
    # a row whose incoming gradient is infinite leaves the other rows' dx alone
    xl = x.clone().requires_grad_(True)
    g = torch.ones(60, device="cuda")
    (d0,) = torch.autograd.grad(heads.linear_cross_entropy(xl, w, t, b, reduction="none"), (xl,), g)
    g[7] = float("inf")
    (d1,) = torch.autograd.grad(heads.linear_cross_entropy(xl, w, t, b, reduction="none"), (xl,), g)
    keep = torch.arange(60, device="cuda") != 7
    assert torch.equal(d0[keep], d1[keep]) and not bool(torch.isfinite(d1[7]).all())


# ---------------------------------------------------------------------------
def _two_layers(x, w1, b1, w2, b2, w3, b3, t):
    import volume_integration.heads as heads
    h = heads.linear_act(x, w1, b1, activation="silu")
    h = heads.linear_act(h, w2, b2, residual=h, activation="gelu")
    return heads.linear_cross_entropy(h, w3, t, b3)


def _decoder(dt, g, M=500, K=4, H=64, V=37, order="image"):
    x = hl.matrix(M, K, dt, g, order)
    ws = [hl.matrix(H, K, dt, g, scale=0.5), hl.matrix(1, H, dt, g)[0], hl.matrix(H, H, dt, g, scale=0.1),
          hl.matrix(1, H, dt, g)[0], hl.matrix(V, H, dt, g, scale=0.3), hl.matrix(1, V, dt, g)[0]]
    t = torch.randint(0, V, (M,), generator=g, device="cuda")
    t[::5] = -100
    return x, ws, t


def _decoder64(x, ws, t):
    p = [v.detach().double().requires_grad_(True) for v in [x] + ws]
    z = p[0] @ p[1].t() + p[2]
    h = torch.nn.functional.silu(z)
    h = torch.nn.functional.gelu(h @ p[3].t() + p[4]) + h
    loss = torch.nn.functional.cross_entropy(h @ p[5].t() + p[6], t)
    return loss, torch.autograd.grad(loss, p)


def _close(got, want, rel):
    # relative to the norm: rounding errors of a chain of layers, each at most `rel` of its norm
    assert float((got.double() - want).norm()) <= rel * float(want.norm()), \
        float((got.double() - want).norm() / want.norm())


# a chain of six products and three stored activations, each rounded at most three times: 18 half steps
CHAIN = [(F32, 18 * 32 * 2.0 ** -24), (F16, 18 * 2.0 ** -11), (BF16, 18 * 2.0 ** -8)]


@pytest.mark.parametrize("dt,rel", CHAIN, ids=["f32", "f16", "bf16"])
def test_decoder_and_loss_together(dt, rel):
    x, ws, t = _decoder(dt, _gen(20))
    leaves = [v.detach().requires_grad_(True) for v in [x] + ws]
    loss = _two_layers(*leaves, t)
    grads = torch.autograd.grad(loss, leaves)
    l64, g64 = _decoder64(x, ws, t)
    _close(loss, l64, rel)
    for a, b in zip(grads, g64):
        _close(a, b, rel)


@pytest.mark.parametrize("want", [("x",), ("w",), ("b",), ("r",), ("w", "b"), ("x", "r")])
@pytest.mark.parametrize("order", ["rows", "image"])
def test_linear_act_some_gradients(want, order):
    import volume_integration.heads as heads
    for K in (4, 40):
        t = dict(zip("xwbr", _act_inputs(300, K, 24, BF16, order, True, True, 50)[:4]))
        dy = hl.matrix(300, 24, BF16, _gen(51), order)
        leaves = {k: (v.detach().requires_grad_(True) if k in want else v) for k, v in t.items()}
        y = heads.linear_act(leaves["x"], leaves["w"], leaves["b"], leaves["r"], "gelu")
        got = dict(zip(want, torch.autograd.grad(y, [leaves[k] for k in want], dy)))
        ref = dict(zip("xwb", hl.linear_act(t["x"], t["w"], t["b"], t["r"], "gelu", dy)[1:]))
        for k, g in got.items():
            if k == "r":
                assert torch.equal(g, dy)
            else:
                hl.assert_within(k, g, ref[k])
        # of a graph that could give all of them
        full = [v.detach().requires_grad_(True) for v in t.values()]
        y = heads.linear_act(*full, activation="gelu")
        for k, g in zip(want, torch.autograd.grad(y, [full["xwbr".index(k)] for k in want], dy)):
            assert torch.equal(g, got[k])


@pytest.mark.parametrize("want", [("x",), ("w",), ("b",), ("w", "b")])
def test_linear_cross_entropy_some_gradients(want):
    import volume_integration.heads as heads
    x, w, b, t = _ce_inputs(300, 40, 130, BF16, "rows", True, 0.2, 52)
    v = dict(zip("xwb", (x, w, b)))
    leaves = {k: (u.detach().requires_grad_(True) if k in want else u) for k, u in v.items()}
    loss = heads.linear_cross_entropy(leaves["x"], leaves["w"], t, leaves["b"])
    ref = dict(zip("xwb", hl.linear_ce(x, w, b, t, -100, "mean", torch.ones((), device="cuda"))[1:]))
    for k, g in zip(want, torch.autograd.grad(loss, [leaves[k] for k in want])):
        hl.assert_within(k, g, ref[k])


def test_no_second_derivative():
    import volume_integration.heads as heads
    x, w, b, t = _ce_inputs(30, 8, 9, F32, "rows", True, 0.0, 53)
    x.requires_grad_(True)
    for out in (heads.linear_act(x, w, b, activation="silu").sum(), heads.linear_cross_entropy(x, w, t, b)):
        (g,) = torch.autograd.grad(out, (x,), create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            g.sum().backward()


def test_another_stream_and_two_at_once():
    # two streams run the chain at the same time on inputs made on a third
    x, ws, t = _decoder(BF16, _gen(21), M=3000)
    leaves = [v.detach().requires_grad_(True) for v in [x] + ws]
    ref = torch.autograd.grad(_two_layers(*leaves, t), leaves)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    results = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                own = [v.detach().requires_grad_(True) for v in [x] + ws]
                results.append(torch.autograd.grad(_two_layers(*own, t), own))
    torch.cuda.synchronize()
    for r in results:
        for a, b in zip(r, ref):
            assert torch.equal(a, b)


def test_captured_and_replayed():
    x, ws, t = _decoder(BF16, _gen(22), M=700)
    static = [v.detach().clone().requires_grad_(True) for v in [x] + ws]

    def step():
        loss = _two_layers(*static, t)
        return [loss.detach()] + list(torch.autograd.grad(loss, static))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs with their own workspaces
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append(g)
        outs.append(out)
    for seed in (23, 24):
        x2, ws2, _ = _decoder(BF16, _gen(seed), M=700)
        with torch.no_grad():
            for a, b in zip(static, [x2] + ws2):
                a.copy_(b)
        eager = step()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for out in outs:
            for a, b in zip(out, eager):
                assert torch.equal(a, b)
    del graphs


def test_tiles_of_two_blocks_captured_and_on_two_streams():
    import volume_integration.heads as heads
    x, w, b, r, dy = _act_inputs(5000, 300, 1100, BF16, "rows", True, True, 54)
    static = [v.detach().clone().requires_grad_(True) for v in (x, w, b, r)]

    def step(leaves):
        y = heads.linear_act(*leaves, activation="silu")
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    want = step(static)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    torch.cuda.synchronize()
    results = []
    for _ in range(3):  # a replay beside two eager streams
        graph.replay()
        for s in (side, torch.cuda.Stream()):
            s.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(s):
                results.append(step([v.detach().requires_grad_(True) for v in (x, w, b, r)]))
    torch.cuda.synchronize()
    for res in results + [out]:
        for a, c in zip(res, want):
            assert torch.equal(a, c)
    del graph


def test_same_call_same_bits():
    x, w, b, t = _ce_inputs(3000, 64, 3001, BF16, "rows", True, 0.1, 25)
    import volume_integration.heads as heads

    def step():
        leaves = [v.detach().requires_grad_(True) for v in (x, w, b)]
        loss = heads.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])
        return [loss.detach()] + list(torch.autograd.grad(loss, leaves))
    first = step()
    for _ in range(4):
        for a, b2 in zip(step(), first):
            assert torch.equal(a, b2)


def test_offsets_beyond_32_bits():
    # rows 2^27 elements apart: the last row starts past element 2^33
    import volume_integration.heads as heads
    base = torch.empty(66 * 2 ** 27, dtype=F16, device="cuda")
    x = base.as_strided((66, 40), (2 ** 27, 1))
    g = _gen(26)
    x.copy_(hl.matrix(66, 40, F16, g))
    w = hl.matrix(48, 40, F16, g, scale=0.2)
    hl.assert_within("y", heads.linear_act(x, w, activation="silu"), hl.linear_act(x, w, None, None, "silu")[0])
    t = torch.randint(0, 48, (66,), generator=g, device="cuda")
    _ce_check(x, w, None, t, "none")


def test_a_wait_that_runs_out_is_reported(monkeypatch):
    # the first load is withheld and the waits are short: the kernel gives up and says so
    import volume_integration.heads as heads
    for M, K, N in ((300, 200, 100), (4100, 200, 1100)):  # tiles of one block, and of two
        x, w, _, _, _ = _act_inputs(M, K, N, BF16, "rows", False, False, 28)
        want = heads.linear_act(x, w)
        assert heads.device_status(reset=True) == 0
        monkeypatch.setenv("VI_HEADS_TEST_TIMEOUT", "1")
        heads.linear_act(x, w)
        assert heads.device_status(reset=True) == 8
        monkeypatch.delenv("VI_HEADS_TEST_TIMEOUT")
        assert torch.equal(heads.linear_act(x, w), want)  # and nothing is left behind
        assert heads.device_status() == 0


@pytest.mark.parametrize("M,K,N,dt,order", [
    (36_000_001, 16, 64, BF16, "image"),   # results beyond element 2^31, odd columns
    (9_000_000, 4, 256, F32, "image"),     # the narrow path's
    (2_200_000, 24, 1000, F16, "rows"),
])
def test_results_beyond_32_bits(M, K, N, dt, order):
    import volume_integration.heads as heads
    g = _gen(29)
    x, w, b = hl.matrix(M, K, dt, g, order), hl.matrix(N, K, dt, g, scale=0.2), hl.matrix(1, N, dt, g)[0]
    y = heads.linear_act(x, w, b, activation="silu")
    for rows in (slice(0, 300), slice(M // 2, M // 2 + 300), slice(M - 300, M)):
        hl.assert_within("y", y[rows], hl.linear_act(x[rows], w, b, None, "silu")[0])
    if dt == F16:
        t = torch.randint(0, N, (M,), generator=g, device="cuda")
        loss = heads.linear_cross_entropy(x, w, t, b, reduction="none")
        for rows in (slice(0, 300), slice(M - 300, M)):
            hl.assert_within("loss", loss[rows], hl.linear_ce(x[rows], w, b, t[rows], -100, "none")[0])


def test_gradients_reach_the_renderer():
    # features of a rendered view -> decoder -> label loss -> the scene's parameters
    import vi_testlib as tl
    import volume_integration as vi
    import volume_integration.heads as heads
    means, conf, s = tl.scene("tiny", device="cuda:0", table_range=1.0)
    g = _gen(27)
    table = s.feature_table.detach().clone().requires_grad_(True)
    conf = conf.detach().clone().requires_grad_(True)
    w1 = hl.matrix(32, s.output_feature_dim, F32, g).requires_grad_(True)
    w2 = hl.matrix(21, 32, F32, g).requires_grad_(True)
    _, feats, _ = vi.integrate_primitives(means, conf, table, s.linear_weights, s.linear_bias, s)
    t = torch.randint(0, 21, feats.shape[1:], generator=g, device="cuda")
    h = heads.linear_act(feats.permute(1, 2, 0), w1, activation="silu")
    loss = heads.linear_cross_entropy(h, w2, t)
    df, d1, d2, dt, dc = torch.autograd.grad(loss, (feats, w1, w2, table, conf), retain_graph=True)
    f64 = feats.detach().double().requires_grad_(True)
    a, b = w1.detach().double().requires_grad_(True), w2.detach().double().requires_grad_(True)
    z = torch.nn.functional.silu(f64.flatten(1).t() @ a.t()) @ b.t()
    ref = torch.nn.functional.cross_entropy(z, t.flatten())
    r = torch.autograd.grad(ref, (f64, a, b))
    rel = CHAIN[0][1]
    _close(loss.detach(), ref.detach(), rel)
    for x, y in zip((df, d1, d2), r):
        _close(x, y, rel)
    # the scene's gradients are the renderer's for exactly that incoming gradient
    ct, cc = torch.autograd.grad(feats, (table, conf), df)
    _close(dt, ct.double(), 1e-3)
    _close(dc, cc.double(), 1e-3)
    assert float(ct.abs().max()) > 0 and float(cc.abs().max()) > 0
