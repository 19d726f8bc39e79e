"""CPU tests of the per-pixel heads: the Python layer's refusals, the C ABI's argument
checks, and the float64 forms that the GPU tests compare with (heads_lib) against
torch's autograd."""
import ctypes

import pytest
import torch

import heads_abi as ha
import heads_lib as hl


def _m(rows, cols, rs, cs, data=256):
    return ctypes.byref(ha.Matrix(data, rows, cols, rs, cs))


def test_python_refusals():
    import volume_integration.heads as heads
    x, w = torch.randn(6, 4), torch.randn(5, 4)
    t = torch.zeros(6, dtype=torch.int64)
    with pytest.raises(TypeError, match="CUDA"):
        heads.linear_act(x, w)
    with pytest.raises(TypeError, match="CUDA"):
        heads.linear_cross_entropy(x, w, t)
    with pytest.raises(ValueError, match="columns"):
        heads.linear_act(x, torch.randn(5, 3))
    with pytest.raises(ValueError, match="at least one"):
        heads.linear_act(torch.randn(6, 0), torch.randn(5, 0))
    with pytest.raises(ValueError, match="bias"):
        heads.linear_act(x, w, torch.randn(4))
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        heads.linear_act(x.double(), w.double())
    with pytest.raises(TypeError, match="weight must be"):
        heads.linear_act(x, w.half())
    with pytest.raises(TypeError, match="bias must be"):
        heads.linear_act(x, w, torch.randn(5).half())
    with pytest.raises(ValueError, match="weight"):
        heads.linear_act(x, torch.randn(4))
    for name, call in (("activation", lambda: heads.linear_act(x, w, activation="tanh")),
                       ("reduction", lambda: heads.linear_cross_entropy(x, w, t, reduction="avg"))):
        with pytest.raises((ValueError, TypeError)):
            call()


def test_c_abi_refusals():
    lib = ha.load()
    q = lib.vi_linear_act_forward_scratch_bytes
    x, w, y = _m(6, 4, 4, 1), _m(5, 4, 4, 1), _m(6, 5, 5, 1)
    assert q(2, 0, x, w, None, None, y, None) > 0
    for args, text in [
        ((7, 0, x, w, None, None, y, None), b"element type"),
        ((2, 9, x, w, None, None, y, None), b"activation"),
        ((2, 0, None, w, None, None, y, None), b"required"),
        ((2, 0, x, _m(5, 3, 3, 1), None, None, y, None), b"columns"),
        ((2, 0, _m(6, 0, 4, 1), _m(5, 0, 4, 1), None, None, y, None), b"at least one"),
        ((2, 0, x, w, None, None, None, None), b"y is required"),
        ((2, 0, x, w, None, None, _m(7, 5, 5, 1), None), b"y"),
        ((2, 0, x, w, None, None, _m(6, 5, 4, 1), None), b"dense"),
        ((2, 0, x, w, None, None, _m(6, 5, 0, 1), None), b"dense"),
        ((2, 0, x, w, None, _m(6, 4, 4, 1), y, None), b"residual"),
        ((2, 0, x, w, None, None, y, _m(6, 5, 6, 1)), b"strides"),
        ((2, 0, _m(6, 4, -4, 1), w, None, None, y, None), b"negative"),
        ((2, 0, _m(6, 4, 4, 1, 0), w, None, None, y, None), b"data"),
        ((2, 0, _m(2 ** 30 + 1, 4, 4, 1), w, None, None, y, None), b"2^30"),
        ((2, 0, _m(6, 4, 4, 1, 257), w, None, None, y, None), b"whole elements"),
        ((0, 0, x, _m(5, 4, 4, 1, 258), None, None, y, None), b"whole elements"),
        ((2, 0, x, w, ctypes.c_void_p(257), None, y, None), b"whole elements"),
        ((2, 0, x, w, None, _m(6, 5, 5, 1, 257), y, None), b"whole elements"),
        ((2, 0, x, w, None, None, _m(6, 5, 5, 1, 257), None), b"whole elements"),
    ]:
        assert q(*args) == 0 and text in lib.vi_last_error(), (args, lib.vi_last_error())
    # a call refuses what its query refuses, and scratch that is short or not aligned
    n = lib.vi_linear_ce_backward_scratch_bytes(2, x, w, None, _m(6, 4, 4, 1), _m(5, 4, 4, 1), None)
    assert n > 256
    p = ctypes.c_void_p
    args = (2, x, w, None, p(256), -100, 1, p(256), p(256), _m(6, 4, 4, 1), _m(5, 4, 4, 1), None)
    assert lib.vi_linear_ce_backward(*args, p(256), 64, None) == 1 and b"scratch" in lib.vi_last_error()
    assert lib.vi_linear_ce_backward(*args, p(264), n, None) == 1 and b"scratch" in lib.vi_last_error()
    assert lib.vi_linear_ce_backward(*args, None, n, None) == 1 and b"scratch" in lib.vi_last_error()
    assert lib.vi_linear_ce_forward(2, x, w, None, p(256), -100, 5, p(256), p(256), p(256), 1 << 20, None) == 1
    assert b"reduction" in lib.vi_last_error()
    assert lib.vi_linear_act_backward_scratch_bytes(2, 1, _m(6, 4, 4, 1), None, x, w, None, None, None, None) == 0
    assert lib.vi_linear_act_backward_scratch_bytes(2, 1, y, None, x, w, None, _m(6, 5, 5, 1), None, None) == 0
    assert lib.vi_linear_act_backward_scratch_bytes(2, 7, y, None, x, w, None, None, None, None) == 0
    # act' is kept, but for no activation and for images of few channels
    image, wide = _m(600, 4, 1, 600), _m(600, 9, 1, 600)
    assert [lib.vi_linear_act_keeps_dact(2, a, v, u) for a, v, u in (
        (1, x, w), (0, x, w), (1, image, w), (1, wide, _m(5, 9, 9, 1)), (1, image, _m(300, 4, 4, 1)))] == [1, 0, 0, 1, 1]
    assert lib.vi_linear_ce_backward_scratch_bytes(2, x, w, None, None, _m(5, 4, 2, 1), None) == 0


def test_scratch_covers_every_layout_step():
    # what a call lays out before its products has to be counted by its query: the masked
    # copy of x (whenever dweight is wanted), and operands the copies cannot read in place
    lib = ha.load()
    M, K, V = 8192, 256, 16384  # as many tiles of dweight as SMs: no pieces of its sum beside
    for dt, es in ((0, 6), (1, 2), (2, 2)):
        x, w = _m(M, K, K, 1), _m(V, K, K, 1)
        dx, dw = _m(M, K, K, 1), _m(V, K, K, 1)
        q = lib.vi_linear_ce_backward_scratch_bytes
        grad = M * V * es
        assert q(dt, x, w, None, None, dw, None) >= min(grad, 256 << 20) + M * K * es
        odd = _m(M, K, K + 1, 1)
        assert q(dt, odd, w, None, None, None, None) >= min(grad, 256 << 20) + M * K * es
        f = lib.vi_linear_act_forward_scratch_bytes
        y = _m(M, V, V, 1)
        assert f(dt, 0, odd, w, None, None, y, None) >= M * K * es
        assert f(dt, 0, _m(M, K, K, 1, 264), w, None, None, y, None) >= M * K * es
        b = lib.vi_linear_act_backward_scratch_bytes
        assert b(dt, 1, y, y, x, w, None, dx, dw, None) >= M * V * es


@pytest.mark.parametrize("act", hl.ACTS)
def test_float64_linear_act_against_autograd(act):
    g = torch.Generator().manual_seed(1)
    x, w, b, r, dy = [torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_(True)
                      for s in ((9, 5), (7, 5), (7,), (9, 7), (9, 7))]
    z = x @ w.t() + b
    f = {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu,
         "gelu": torch.nn.functional.gelu, "sigmoid": torch.sigmoid}[act]
    y = f(z) + r
    grads = torch.autograd.grad(y, (x, w, b), dy.detach())
    out = hl.linear_act(*[t.detach() for t in (x, w, b, r)], act, dy.detach())
    for (v, _), ref in zip(out, (y.detach(),) + grads):
        torch.testing.assert_close(v, ref, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_float64_linear_ce_against_autograd(reduction):
    g = torch.Generator().manual_seed(2)
    x, w, b = [torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_(True) for s in ((9, 5), (7, 5), (7,))]
    t = torch.tensor([0, 6, -100, 3, 2, -100, 1, 5, 4])
    loss = torch.nn.functional.cross_entropy(x @ w.t() + b, t, reduction=reduction)
    dl = torch.randn(loss.shape, generator=g, dtype=torch.float64)
    grads = torch.autograd.grad(loss, (x, w, b), dl)
    out = hl.linear_ce(x.detach(), w.detach(), b.detach(), t, -100, reduction, dl)
    for (v, _), ref in zip(out, (loss.detach(),) + grads):
        torch.testing.assert_close(v, ref, rtol=1e-12, atol=1e-12)


def test_a_value_outside_its_bound_is_found():
    x, w = torch.randn(20, 8), torch.randn(6, 8)
    value, bound = hl.linear_act(x, w, None, None, "silu")[0]
    got = value.float()
    hl.assert_within("y", got, (value, bound))
    got[3, 2] += 4 * float(bound[3, 2]) + 1e-6
    with pytest.raises(AssertionError, match="outside"):
        hl.assert_within("y", got, (value, bound))
    got[3, 2] = float("nan")
    with pytest.raises(AssertionError, match="outside"):
        hl.assert_within("y", got, (value, bound))
