"""CPU tests of layer_norm, quantize_rows, linear_act_int8 and sample_labels: refusals of the Python layer and of the C
ABI, and the float64 forms that the GPU tests compare with against torch's autograd and against differences."""
import ctypes

import pytest
import torch

import decoder_lib as dl
import heads_abi as ha

P, I, D = ctypes.c_void_p, ctypes.c_int64, ctypes.c_double


class Sampling(ctypes.Structure):
    _fields_ = [("temperature", D), ("top_p", D), ("min_p", D), ("top_k", I), ("temperatures", P), ("top_ks", P),
                ("top_ps", P), ("min_ps", P)]


def _m(rows, cols, rs, cs, data=256):
    return ctypes.byref(ha.Matrix(data, rows, cols, rs, cs))


def _lib():
    lib = ha.load()
    m, i, u64, f = ctypes.POINTER(ha.Matrix), ctypes.c_int, ctypes.c_uint64, ctypes.c_float
    lib.vi_layer_norm_forward.argtypes = [i, m, P, P, f, m, P, P]
    lib.vi_layer_norm_backward_scratch_bytes.argtypes = [i, m, m, P, m, P, P]
    lib.vi_layer_norm_backward_scratch_bytes.restype = u64
    lib.vi_layer_norm_backward.argtypes = [i, m, m, P, P, m, P, P, P, u64, P]
    lib.vi_quantize_rows.argtypes = [i, m, m, P, P]
    lib.vi_linear_act_int8_scratch_bytes.argtypes = [i, i, m, P, m, P, P, m, m]
    lib.vi_linear_act_int8_scratch_bytes.restype = u64
    lib.vi_linear_act_int8.argtypes = [i, i, m, P, m, P, P, m, m, P, u64, P]
    lib.vi_sample_labels_scratch_bytes.argtypes = [i, m, ctypes.POINTER(Sampling)]
    lib.vi_sample_labels_scratch_bytes.restype = u64
    lib.vi_sample_labels.argtypes = [i, m, P, ctypes.POINTER(Sampling), P, P, u64, P]
    return lib


def test_python_refusals_of_layer_norm():
    from volume_integration import heads
    x = torch.randn(6, 4)
    for error, text, call in (
            (TypeError, "CUDA", lambda: heads.layer_norm(x)),
            (TypeError, "float32, float16", lambda: heads.layer_norm(x.double())),
            (ValueError, "at least one", lambda: heads.layer_norm(torch.randn(6, 0))),
            (ValueError, "at least one", lambda: heads.layer_norm(torch.randn(()))),
            (ValueError, r"weight must be \[4\]", lambda: heads.layer_norm(x, torch.ones(5))),
            (ValueError, r"bias must be \[4\]", lambda: heads.layer_norm(x, None, torch.ones(4, 1))),
            (TypeError, "weight must be", lambda: heads.layer_norm(x, torch.ones(4).half())),
            (ValueError, "eps", lambda: heads.layer_norm(x, eps=-1.0)),
            (ValueError, "eps", lambda: heads.layer_norm(x, eps=float("nan")))):
        with pytest.raises(error, match=text):
            call()


def test_python_refusals_of_8_bit_layers():
    from volume_integration import heads
    x, pair = torch.randn(6, 4), (torch.zeros(5, 4, dtype=torch.int8), torch.ones(5))
    xq = (torch.zeros(6, 4, dtype=torch.int8), torch.ones(6))
    f = heads.linear_act_int8
    for error, text, call in (
            (TypeError, "CUDA", lambda: heads.quantize_rows(x)),
            (TypeError, "float32, float16", lambda: heads.quantize_rows(x.double())),
            (ValueError, "at least one", lambda: heads.quantize_rows(torch.randn(3, 0))),
            (TypeError, "CUDA", lambda: f(x, pair)),
            (ValueError, "pair", lambda: f(x, pair + pair)),
            (TypeError, "int8", lambda: f(x, (torch.zeros(5, 4), torch.ones(5)))),
            (TypeError, "float32", lambda: f(x, (pair[0], torch.ones(5).double()))),
            (ValueError, "scale", lambda: f(x, (pair[0], torch.ones(4)))),
            (ValueError, "weight must be", lambda: f(x, (torch.zeros(4, dtype=torch.int8), torch.ones(())))),
            (ValueError, "columns", lambda: f(torch.randn(6, 3), pair)),
            (TypeError, "or a pair", lambda: f(x.double(), pair)),
            (TypeError, "dtype", lambda: f(x, pair, dtype=torch.float16)),
            (ValueError, "dtype", lambda: f(xq, pair)),
            (TypeError, "dtype", lambda: f(xq, pair, dtype=torch.float64)),
            (ValueError, "activation", lambda: f(x, pair, activation="tanh")),
            (ValueError, "bias", lambda: f(x, pair, torch.ones(4))),
            (TypeError, "bias", lambda: f(x, pair, torch.ones(5).half())),
            (ValueError, "residual", lambda: f(x, pair, residual=torch.ones(6, 4))),
            (TypeError, "residual", lambda: f(x, pair, residual=torch.ones(6, 5).half()))):
        with pytest.raises(error, match=text):
            call()


def test_python_refusals_of_sample_labels():
    from volume_integration import heads
    z, u = torch.randn(6, 4), torch.rand(6)
    f = heads.sample_labels
    for error, text, call in (
            (TypeError, "CUDA", lambda: f(z, u)),
            (TypeError, "float32, float16", lambda: f(z.double(), u)),
            (TypeError, "u must be", lambda: f(z, u.double())),
            (ValueError, "u must be", lambda: f(z, u[:5])),
            (ValueError, "at least one", lambda: f(torch.randn(6, 0), u)),
            (ValueError, "temperature", lambda: f(z, u, temperature=-0.1)),
            (ValueError, "temperature", lambda: f(z, u, temperature=float("nan"))),
            (TypeError, "temperature", lambda: f(z, u, temperature=u.double())),
            (ValueError, "temperature", lambda: f(z, u, temperature=u[:3])),
            (ValueError, "top_k", lambda: f(z, u, top_k=-1)),
            (TypeError, "top_k", lambda: f(z, u, top_k=u)),
            (ValueError, "top_p", lambda: f(z, u, top_p=0.0)),
            (ValueError, "min_p", lambda: f(z, u, min_p=1.5))):
        with pytest.raises(error, match=text):
            call()


def test_c_abi_refusals():
    lib = _lib()
    x, y, vec = _m(6, 4, 4, 1), _m(6, 4, 4, 1), P(256)
    for args, text in [
        ((7, x, None, None, 1e-5, y, None, None), b"element type"),
        ((2, None, None, None, 1e-5, y, None, None), b"column"),
        ((2, _m(6, 0, 4, 1), None, None, 1e-5, y, None, None), b"column"),
        ((2, _m(2 ** 30 + 1, 4, 4, 1), None, None, 1e-5, y, None, None), b"2^30"),
        ((2, _m(6, 4, 4, 1, 0), None, None, 1e-5, y, None, None), b"data"),
        ((2, _m(6, 4, -4, 1), None, None, 1e-5, y, None, None), b"negative"),
        ((2, _m(6, 4, 4, 1, 257), None, None, 1e-5, y, None, None), b"whole elements"),
        ((2, x, P(257), None, 1e-5, y, None, None), b"whole elements"),
        ((2, x, None, P(257), 1e-5, y, None, None), b"whole elements"),
        ((2, x, None, None, -1.0, y, None, None), b"eps"),
        ((2, x, None, None, 1e-5, None, None, None), b"y is required"),
        ((2, x, None, None, 1e-5, _m(6, 5, 5, 1), None, None), b"dense"),
        ((2, x, None, None, 1e-5, _m(6, 4, 3, 1), None, None), b"dense"),
    ]:
        assert lib.vi_layer_norm_forward(*args) == 1 and text in lib.vi_last_error(), (args, lib.vi_last_error())
    q = lib.vi_layer_norm_backward_scratch_bytes
    assert q(2, y, x, vec, y, vec, vec) > 256 and q(2, y, x, vec, y, None, None) == 256
    assert q(2, None, x, vec, y, None, None) == 0 and b"dy" in lib.vi_last_error()
    assert q(2, y, x, vec, _m(6, 4, 2, 1), None, None) == 0 and b"dx" in lib.vi_last_error()
    assert q(2, y, x, vec, y, P(257), None) == 0 and b"whole elements" in lib.vi_last_error()
    assert lib.vi_layer_norm_backward(2, y, x, vec, vec, y, vec, None, vec, 16, None) == 1
    assert b"scratch" in lib.vi_last_error()
    # 8-bit rows
    for args, text in [
        ((5, x, y, vec, None), b"element type"),
        ((2, x, _m(6, 4, 3, 1), vec, None), b"contiguous"),
        ((2, x, _m(6, 5, 5, 1), vec, None), b"contiguous"),
        ((2, x, _m(6, 4, 1, 6), vec, None), b"contiguous"),
        ((2, x, y, None, None), b"required"),
        ((2, x, y, P(258), None), b"required"),
    ]:
        assert lib.vi_quantize_rows(*args) == 1 and text in lib.vi_last_error(), (args, lib.vi_last_error())
    f = lib.vi_linear_act_int8_scratch_bytes
    w, out = _m(5, 4, 16, 1), _m(6, 5, 5, 1)
    assert f(2, 0, x, None, w, vec, None, None, out) >= 6 * 16 + 6 * 4
    assert f(2, 0, _m(6, 4, 16, 1), vec, w, vec, None, None, out) == 256
    for args, text in [
        ((4, 0, x, None, w, vec, None, None, out), b"element type"),
        ((2, 7, x, None, w, vec, None, None, out), b"activation"),
        ((2, 0, x, None, _m(5, 3, 16, 1), vec, None, None, out), b"columns"),
        ((2, 0, _m(6, 2 ** 17 + 1, 1 << 18, 1), None, _m(5, 2 ** 17 + 1, 1 << 18, 1), vec, None, None, out), b"2^17"),
        ((2, 0, x, None, w, None, None, None, out), b"scale"),
        ((2, 0, _m(6, 4, 4, 1, 257), None, w, vec, None, None, out), b"whole elements"),
        ((2, 0, x, None, w, P(258), None, None, out), b"whole elements"),
        ((2, 0, x, None, w, vec, P(257), None, out), b"whole elements"),
        ((2, 0, x, None, w, vec, None, _m(6, 4, 4, 1), out), b"residual"),
        ((2, 0, x, None, w, vec, None, None, None), b"y is required"),
        ((2, 0, x, None, w, vec, None, None, _m(6, 5, 4, 1)), b"dense"),
        ((2, 0, _m(6, 4, 4, -1), None, w, vec, None, None, out), b"negative"),
    ]:
        assert f(*args) == 0 and text in lib.vi_last_error(), (args, lib.vi_last_error())
    # labels
    ok = dict(temperature=1.0, top_p=1.0, min_p=0.0, top_k=0)
    for dt, z, change, u, text in [
        (9, x, {}, vec, b"element type"), (2, None, {}, vec, b"required"), (2, _m(6, 0, 4, 1), {}, vec, b"column"),
        (2, _m(6, 4, -1, 1), {}, vec, b"negative"), (2, _m(6, 4, 4, 1, 257), {}, vec, b"whole elements"),
        (2, x, dict(temperature=-1.0), vec, b"temperature"), (2, x, dict(top_k=-1), vec, b"top_k"),
        (2, x, dict(top_p=0.0), vec, b"top_p"), (2, x, dict(min_p=2.0), vec, b"min_p"), (2, x, {}, None, b"need data"),
    ]:
        s = Sampling(**{**ok, **change})
        assert lib.vi_sample_labels(dt, z, u, ctypes.byref(s), vec, None, 0, None) == 1
        assert text in lib.vi_last_error(), (text, lib.vi_last_error())
        if u:
            assert lib.vi_sample_labels_scratch_bytes(dt, z, ctypes.byref(s)) == 0
    s = Sampling(**ok)
    assert lib.vi_sample_labels_scratch_bytes(2, x, ctypes.byref(s)) == 256
    long = _m(6, 60000, 60000, 1)
    n = lib.vi_sample_labels_scratch_bytes(2, long, ctypes.byref(s))
    assert n > 6 * 4096
    assert lib.vi_sample_labels(2, long, vec, ctypes.byref(s), vec, vec, n // 2, None) == 1
    assert b"scratch" in lib.vi_last_error()


@pytest.mark.parametrize("affine", [False, True])
def test_float64_layer_norm_against_autograd_and_differences(affine):
    g = torch.Generator().manual_seed(1)
    x, dy = (torch.randn(5, 7, generator=g, dtype=torch.float64) for _ in range(2))
    w, b = (torch.randn(7, generator=g, dtype=torch.float64) for _ in range(2)) if affine else (None, None)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b) if t is not None]
    y = torch.nn.functional.layer_norm(leaves[0], (7,), *(leaves[1:] if affine else ()), eps=1e-3)
    refs = [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    for (v, _), ref in zip(dl.layer_norm(x, w, b, 1e-3, dy), refs):
        torch.testing.assert_close(v, ref, rtol=1e-12, atol=1e-12)
    # the formula's gradient against central differences of its own value
    grads = dl.layer_norm(x, w, b, 1e-3, dy)[1:]
    step = 1e-5
    for which, t in enumerate(t for t in (x, w, b) if t is not None):
        move = torch.randn(t.shape, generator=g, dtype=torch.float64)
        at = []
        for sign in (1, -1):
            args = [v if v is not t else v + sign * step * move for v in (x, w, b)]
            at.append((dl.layer_norm(*args, 1e-3)[0][0] * dy).sum())
        torch.testing.assert_close((at[0] - at[1]) / (2 * step), (grads[which][0] * move).sum(), rtol=1e-7, atol=1e-8)


def test_float64_labels_follow_the_probabilities():
    # evenly spaced u: each label is drawn as often as its share of the kept mass says
    z = torch.tensor([[0.5, 2.0, -1.0, 2.0, float("-inf"), 0.0]]).expand(4000, 6)
    u = (torch.arange(4000) + 0.5) / 4000
    for settings in (dict(), dict(temperature=0.5), dict(top_k=3), dict(top_p=0.7), dict(min_p=0.2), dict(top_k=4, top_p=0.9)):
        t = settings.get("temperature", 1.0)
        p = torch.softmax(z[0].double() / t, 0)
        order = torch.sort(z[0], descending=True, stable=True).indices.tolist()
        if "top_k" in settings:
            order = order[:settings["top_k"]]
        if "top_p" in settings:
            mass, kept = sum(float(p[i]) for i in order), []
            for i in order:
                if sum(float(p[j]) for j in kept) < settings["top_p"] * mass:
                    kept.append(i)
            order = kept
        order = [i for i in order if float(p[i]) >= settings.get("min_p", 0.0) * float(p.max())]
        share = torch.zeros(6, dtype=torch.float64)
        share[order] = p[order] / p[order].sum()
        got = torch.bincount(dl.sample(z, u, **settings), minlength=6) / 4000
        assert float((got - share).abs().max()) <= 1 / 4000
