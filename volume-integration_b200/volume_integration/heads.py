"""Per-pixel heads on rendered feature images (extension; no counterpart in the
reference, whose feature image goes to the user's own code: reference
``volume_integration/__init__.py:365-389``).

The renderer ends at ``out_features [F_out, H, W]``.  This module adds, on the
same CUDA library, the two operators that feature and label fields put behind it:

* ``linear_act``: a dense layer, ``act(x W^T + b) + residual``;
* ``linear_cross_entropy``: the softmax cross entropy of a linear classifier over
  a vocabulary of labels or codes, without ever storing the logits.

Both take features of shape ``[..., K]`` in any strides, so the renderer's image
goes in as ``out_features.flatten(1).t()`` (rows are pixels) without a copy by
the caller, and ``linear_act`` answers in the same memory order.  float32,
float16 and bfloat16; one type per call; sums in float32.  Gradients flow to every
float input.

Sums are added in a fixed order: the same call gives the same bits.  There is no
CPU fallback: without the CUDA library the import fails.

The products run on the tensor cores; float32 operands as sums of three
bfloat16 parts, which keeps float32's precision: sums of any length are within 1e-6 of the norm of the
result (an infinite feature or weight gives NaN where float32 arithmetic might give an infinity).
"""
import torch

from . import _C

__all__ = ["ACTIVATIONS", "device_status", "linear_act", "linear_cross_entropy"]

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


def device_status(device=None, reset=False):
    """Status word of the heads' kernels on a device: 0, or ``VI_DEVICE_HEAD_TIMEOUT`` (8) when a
    bounded wait gave up in one of them (that call's results are unspecified).  Waits
    for the current stream; ``reset`` clears the word.
    """
    index = torch.device("cuda" if device is None else device).index
    return _C.heads_status(torch.cuda.current_device() if index is None else index, reset)
