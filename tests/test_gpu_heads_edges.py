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
