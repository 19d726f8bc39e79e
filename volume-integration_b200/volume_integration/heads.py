"""Per-pixel heads on rendered feature images (extension; no counterpart in the
reference, whose feature image goes to the user's own code: reference
``volume_integration/__init__.py:365-389``).

The renderer ends at ``out_features [F_out, H, W]``.  This module adds, on the
same CUDA library, the operators that feature and label fields put behind it:

* ``linear_act``: a dense layer, ``act(x W^T + b) + residual``;
* ``linear_cross_entropy``: the softmax cross entropy of a linear classifier over
  a vocabulary of labels or codes, without ever storing the logits;
* ``layer_norm``: each pixel's features normalised, before a dense layer;
* ``linear_act_int8``: the dense layer in 8-bit integers, for display; ``quantize_rows``
  makes its weights;
* ``sample_labels``: a label drawn from each pixel's logits, for display.

All take features of shape ``[..., K]`` in any strides, so the renderer's image
goes in as ``out_features.flatten(1).t()`` (rows are pixels) without a copy by
the caller, and answer in the same memory order.  float32,
float16 and bfloat16; one type per call; sums in float32.  Gradients flow to every
float input of the first three; the other two have none.

Sums are added in a fixed order: the same call gives the same bits.  There is no
CPU fallback: without the CUDA library the import fails.

The products run on the tensor cores; float32 operands as sums of three
bfloat16 parts, which keeps float32's precision: sums of any length are within 1e-6 of the norm of the
result (an infinite feature or weight gives NaN where float32 arithmetic might give an infinity).
"""
import torch

from . import _C

__all__ = ["ACTIVATIONS", "device_status", "layer_norm", "linear_act", "linear_act_int8", "linear_cross_entropy",
           "quantize_rows", "sample_labels"]

ACTIVATIONS = ("none", "relu", "silu", "gelu", "sigmoid")
REDUCTIONS = ("none", "mean", "sum")
_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _check_operands(x, weight, bias, what, out_name):
    if x.dim() < 1 or weight.dim() != 2:
        raise ValueError(f"{what}: x must be [..., K] and weight [{out_name}, K], "
                         f"got {tuple(x.shape)} and {tuple(weight.shape)}")
    if weight.shape[1] != x.shape[-1]:
        raise ValueError(f"{what}: weight has {weight.shape[1]} columns but x has {x.shape[-1]}")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"{what}: weight must have at least one row and one column, got {tuple(weight.shape)}")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f"{what}: bias must be [{weight.shape[0]}], got {tuple(bias.shape)}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{what}: x must be float32, float16 or bfloat16, got {x.dtype}")
    for name, t in (("weight", weight), ("bias", bias)):
        _check_like(x, t, what, name)
    if not x.is_cuda:
        raise TypeError(f"{what}: x must be a CUDA tensor, but device is {x.device}")


def _check_like(x, t, what, name):
    if t is not None and t.dtype != x.dtype:
        raise TypeError(f"{what}: {name} must be {x.dtype} like x, got {t.dtype}")
    if t is not None and t.device != x.device:
        raise ValueError(f"{what}: {name} is on {t.device} but x is on {x.device}")


def linear_act(x, weight, bias=None, residual=None, activation="none"):
    """``act(x @ weight.T + bias) + residual`` in one pass over the output.

    x: [..., K]; weight: [N, K]; bias: [N]; residual: [..., N]; ``activation`` one
    of ``ACTIVATIONS`` (gelu is the exact form, with the normal distribution
    function).  Returns [..., N] in x's type.  When x's rows lie next to each
    other in memory (a channel-first image seen as [pixels, K]) so do the result's.

    float16 and bfloat16 results are rounded once, from float32.  The backward
    keeps act' in 16 bits (float16: to 2^-12 of its value down to 2^-14, to 2^-26 absolute below;
    bfloat16: to 2^-11 of its value down to 2^-29, to 2^-40 absolute below) and, but for small products, rounds the product of dy
    and act' to the operands' type before the two matrix products.
    """
    _check_operands(x, weight, bias, "linear_act", "N")
    if activation not in ACTIVATIONS:
        raise ValueError(f"linear_act: activation must be one of {ACTIVATIONS}, got {activation!r}")
    n = weight.shape[0]
    lead = x.shape[:-1]
    if residual is not None:
        if residual.shape != lead + (n,):
            raise ValueError(f"linear_act: residual must be {tuple(lead + (n,))}, got {tuple(residual.shape)}")
        _check_like(x, residual, "linear_act", "residual")
    two_d = x.dim() == 2
    x2 = x if two_d else x.reshape(-1, x.shape[-1])
    r2 = residual if two_d or residual is None else residual.reshape(-1, n)
    y = _C.linear_act(x2, weight, bias, r2, ACTIVATIONS.index(activation))
    return y if two_d else y.reshape(lead + (n,))


def linear_cross_entropy(x, weight, target, bias=None, ignore_index=-100, reduction="mean"):
    """Softmax cross entropy of the logits ``x @ weight.T + bias`` against ``target``.

    x: [..., K]; weight: [V, K]; target: int64 [...], class indices; bias: [V].
    Rows whose target is ``ignore_index`` have loss 0 and take no part in the mean or in any
    gradient, whatever their features hold.  Any other target outside [0, V) makes its
    row's loss, and what it is summed into, NaN.  Returns float32: [...] for
    ``reduction="none"``, else a scalar (the mean over no row at all is NaN).

    The logits exist only as tiles on the chip; the backward computes them again
    in pieces of the vocabulary and keeps one piece of their gradient at a time,
    in x's type (weight's, bias's and x's gradients are sums of it in float32).  In float16 with
    ``reduction="none"`` the rows' incoming gradients share one scale: rows under 2^-26 of the
    largest lose their small probabilities.
    """
    _check_operands(x, weight, bias, "linear_cross_entropy", "V")
    if reduction not in REDUCTIONS:
        raise ValueError(f"linear_cross_entropy: reduction must be one of {REDUCTIONS}, got {reduction!r}")
    if target.dtype != torch.int64:
        raise TypeError(f"linear_cross_entropy: target must be int64, got {target.dtype}")
    if target.shape != x.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: target must be {tuple(x.shape[:-1])}, got {tuple(target.shape)}")
    if target.device != x.device:
        raise ValueError(f"linear_cross_entropy: target is on {target.device} but x is on {x.device}")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    t1 = target.reshape(-1).contiguous()
    loss = _C.linear_cross_entropy(x2, weight, bias, t1, int(ignore_index), REDUCTIONS.index(reduction))
    return loss.reshape(target.shape) if reduction == "none" else loss


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis, in one pass.

    x: [..., K]; weight, bias: [K], either may be None; var is the mean of
    (x - mean)^2.  Returns x's shape and type, rounded once, in x's memory order where its rows lie evenly
    spaced (a batch of images does not: row by row then).  Statistics and all sums are float32; each row's are kept for the backward (12 bytes a row).  A row's
    NaN or infinity stays in its row, in the result and in x's gradient.
    """
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm: x must be [..., K] with at least one column, got {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"layer_norm: x must be float32, float16 or bfloat16, got {x.dtype}")
    k = x.shape[-1]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != (k,):
            raise ValueError(f"layer_norm: {name} must be [{k}], got {tuple(t.shape)}")
        _check_like(x, t, "layer_norm", name)
    if not 0 <= eps < float("inf"):
        raise ValueError(f"layer_norm: eps must be a number of at least 0, got {eps!r}")
    if not x.is_cuda:
        raise TypeError(f"layer_norm: x must be a CUDA tensor, but device is {x.device}")
    if x.dim() == 2:
        return _C.layer_norm(x, weight, bias, eps)
    return _C.layer_norm(x.reshape(-1, k), weight, bias, eps).reshape(x.shape)


def quantize_rows(x):
    """x: [..., K] as 8-bit integers with a scale for each row: ``(q int8 [..., K], scale float32 [...])``.

    ``scale = max |x| / 127`` (rounded to float32) and q is ``x / scale`` rounded to the nearest whole number, ties
    to even, so x is about ``q * scale[..., None]``.  A row of zeros has scale 0; one with an infinity or a NaN has scale NaN and
    q 0.  q's rows lie a multiple of 16 bytes apart in memory.  Neither result carries gradients.
    """
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"quantize_rows: x must be [..., K] with at least one column, got {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"quantize_rows: x must be float32, float16 or bfloat16, got {x.dtype}")
    if not x.is_cuda:
        raise TypeError(f"quantize_rows: x must be a CUDA tensor, but device is {x.device}")
    if x.dim() == 2:
        return _C.quantize_rows(x)
    lead = x.shape[:-1]
    q, scale = _C.quantize_rows(x.reshape(-1, x.shape[-1]))
    return (q.unflatten(0, lead) if lead else q[0]), scale.reshape(lead)


def _check_pair(pair, what, name):
    if len(pair) != 2:
        raise ValueError(f"{what}: {name} must be the pair (q, scale) that quantize_rows returns")
    q, scale = pair
    if q.dtype != torch.int8 or scale.dtype != torch.float32:
        raise TypeError(f"{what}: {name} must be (int8, float32), got ({q.dtype}, {scale.dtype})")
    if q.dim() < 1 or scale.shape != q.shape[:-1]:
        raise ValueError(f"{what}: {name}'s scale must be {tuple(q.shape[:-1])}, got {tuple(scale.shape)}")
    return q, scale


def linear_act_int8(x, weight, bias=None, residual=None, activation="none", dtype=None):
    """``linear_act`` with the products in 8-bit integers: ``act(x W^T + bias) + residual``.

    weight: the pair ``quantize_rows`` makes of [N, K], one scale an output channel.  x: [..., K] of float32, float16
    or bfloat16, whose rows are quantised in the call, one scale a row; or such a pair, for several layers
    that read the same features: then ``dtype`` says the result's type.  bias: [N] and residual: [..., N] of the result's type
    (x's).  K is less than 2^17: sums are exact, then scaled in float32, and results are rounded once.  Rows or channels whose scale is
    NaN come out as NaN.  For display: there is no backward, and inputs that require gradients are refused
    where they are recorded.

    It pays where sums are long and outputs many (32768 x 1024 -> 4096 in float16: 180 us, linear_act 229), where several
    layers of 512 features and more read one pair, and for float32 x.  16-bit layers of up to 512 features take longer than in linear_act, as
    finding the scales costs a pass over x (1920 x 1080 x 64 -> 64: 324 us, linear_act 209).
    """
    what = "linear_act_int8"
    wq, ws = _check_pair(weight, what, "weight")
    if wq.dim() != 2:
        raise ValueError(f"{what}: weight must be [N, K], got {tuple(wq.shape)}")
    if isinstance(x, (tuple, list)):
        x, xs = _check_pair(x, what, "x")
        if dtype is None:
            raise ValueError(f"{what}: dtype, the result's type, is needed with an x in 8-bit integers")
    else:
        xs = None
        if x.dtype not in _DTYPES:
            raise TypeError(f"{what}: x must be float32, float16 or bfloat16, or a pair, got {x.dtype}")
        if dtype is not None and dtype != x.dtype:
            raise TypeError(f"{what}: dtype must be x's, {x.dtype}, got {dtype}")
        dtype = x.dtype
    if dtype not in _DTYPES:
        raise TypeError(f"{what}: dtype must be float32, float16 or bfloat16, got {dtype}")
    n, k = wq.shape
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"{what}: weight has {k} columns but x is {tuple(x.shape)}")
    if n < 1 or k < 1:
        raise ValueError(f"{what}: weight must have at least one row and one column, got {tuple(wq.shape)}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"{what}: activation must be one of {ACTIVATIONS}, got {activation!r}")
    lead = x.shape[:-1]
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError(f"{what}: bias must be [{n}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != lead + (n,):
        raise ValueError(f"{what}: residual must be {tuple(lead + (n,))}, got {tuple(residual.shape)}")
    for name, t in (("bias", bias), ("residual", residual)):
        if t is not None and t.dtype != dtype:
            raise TypeError(f"{what}: {name} must be {dtype} like the result, got {t.dtype}")
    for name, t in (("weight", wq), ("weight's scale", ws), ("x's scale", xs), ("bias", bias), ("residual", residual)):
        if t is not None and t.device != x.device:
            raise ValueError(f"{what}: {name} is on {t.device} but x is on {x.device}")
    if not x.is_cuda:
        raise TypeError(f"{what}: x must be a CUDA tensor, but device is {x.device}")
    index = ACTIVATIONS.index(activation)
    if x.dim() == 2:
        return _C.linear_act_int8(x, xs, wq, ws, bias, residual, index, dtype)
    return _C.linear_act_int8(x.reshape(-1, k), None if xs is None else xs.reshape(-1), wq, ws, bias,
                              None if residual is None else residual.reshape(-1, n), index, dtype).reshape(lead + (n,))


def _setting(value, default, dtype, logits, name, low, high, wants):
    """(number, tensor or None) of a setting that is one number or one value a row."""
    lead = logits.shape[:-1]
    if isinstance(value, torch.Tensor):
        if value.dtype != dtype:
            raise TypeError(f"sample_labels: {name} must be a number or {dtype}, got {value.dtype}")
        if value.shape != lead:
            raise ValueError(f"sample_labels: {name} must be a number or {tuple(lead)}, got {tuple(value.shape)}")
        if value.device != logits.device:
            raise ValueError(f"sample_labels: {name} is on {value.device} but logits is on {logits.device}")
        return default, value.reshape(-1)
    if not low <= value <= high:
        raise ValueError(f"sample_labels: {name} must be {wants}, got {value!r}")
    return value, None


def sample_labels(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """A label drawn from each row of logits by the random number u: int64 [...].

    logits: [..., V]; u: float32 [...], in [0, 1).  With w = exp((z - max z) / temperature), and the labels in the order
    of falling z (equal ones: lowest first): ``top_k`` keeps the first k (0: all); ``top_p`` those of them in front of which
    lies less than that share of their mass (1: all), the first always; ``min_p`` those with w >= min_p.  The answer is the
    first label, in index order, at which the running sum of the kept w exceeds u times the whole.
    ``temperature`` 0 takes the first of the largest.

    Each setting is a number, or a tensor [...] with one value a row (top_k int64, the others float32; a row's
    temperature of 0 or less is 0, one that is NaN answers -1, a top_k under 1 is off, a top_p of 0 or less keeps the
    first, a min_p above 1 is 1; a top_p or min_p that is NaN is off).  Logits of -inf are never drawn; a row without
    any other, or with a NaN, answers -1; +inf takes all mass.  Weights (from 2^-1000 on) and sums are 64 bits wide
    where they decide, so the answer is the definition's but where u falls within about 1e-10 of a border.

    Fast on images (channel-first logits) of up to 256 labels without top_k and top_p; with one of them an image is read
    with strides (800 x 800 x 150 in float16: 78 us with min_p, 2 ms with top_p).
    """
    what = "sample_labels"
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: logits must be [..., V] with at least one column, got {tuple(logits.shape)}")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"{what}: logits must be float32, float16 or bfloat16, got {logits.dtype}")
    if u.dtype != torch.float32:
        raise TypeError(f"{what}: u must be float32, got {u.dtype}")
    lead = logits.shape[:-1]
    if u.shape != lead:
        raise ValueError(f"{what}: u must be {tuple(lead)}, got {tuple(u.shape)}")
    if u.device != logits.device:
        raise ValueError(f"{what}: u is on {u.device} but logits is on {logits.device}")
    inf = float("inf")
    t, ts = _setting(temperature, 1.0, torch.float32, logits, "temperature", 0, inf, "at least 0")
    k, ks = _setting(top_k, 0, torch.int64, logits, "top_k", 0, 2 ** 62, "at least 0")
    p, ps = _setting(top_p, 1.0, torch.float32, logits, "top_p", 5e-324, inf, "above 0")
    m, ms = _setting(min_p, 0.0, torch.float32, logits, "min_p", 0, 1, "between 0 and 1")
    if not logits.is_cuda:
        raise TypeError(f"{what}: logits must be a CUDA tensor, but device is {logits.device}")
    z = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    label = _C.sample_labels(z, u.reshape(-1), t, ts, k, ks, p, ps, m, ms)
    return label if logits.dim() == 2 else label.reshape(lead)


def device_status(device=None, reset=False):
    """Status word of the heads' kernels on a device: 0, or ``VI_DEVICE_HEAD_TIMEOUT`` (8) when a
    bounded wait gave up in one of them (that call's results are unspecified).  Waits
    for the current stream; ``reset`` clears the word.
    """
    index = torch.device("cuda" if device is None else device).index
    return _C.heads_status(torch.cuda.current_device() if index is None else index, reset)
