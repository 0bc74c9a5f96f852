"""Operators of a network that reads long signals and gives theta.

``gated_recurrence`` (a scan over the samples, with its backward) and ``rms_norm``
(with the residual's addition, and an 8-bit output).  Both are HIP kernels behind
the C ABI, called from native functions (csrc/torch_sequence.cpp); there is no torch
or CPU fallback.  No counterpart in the reference, whose networks are torch modules
(``stn/demos/*.py``).
"""
import torch

from ._native import torch_binding
from ._tracing import recorded

__all__ = ["gated_recurrence", "rms_norm"]


def gated_recurrence(x, f, g=None, h0=None, lengths=None):
    """A gated linear recurrence over each row's samples.

    With a = sigmoid(f) for each sample and channel,

        h_t = a_t h_{t-1} + (1 - a_t) x_t,    y_t = h_t g_t sigmoid(g_t)

    (``y = h`` without ``g``).  The state is held in 32 bits.

    Arguments:
        x, f, g: [B, T, C] float32 or bfloat16 of one type; slices of one
            projection's output and [T, B, C] in memory are read where they lie (any
            strides over B and T, while the samples of a tile, up to 1024, span less than 2^31
            bytes; others, and channels that are not neighbours, are copied first)
        h0: [B, C] float32, the state before the first sample (default: zeros)
        lengths: [B] int32 or int64, samples in each row (default: T; clamped to
            [0, T]).  Behind a row's end y is 0 and the state stays; what the inputs
            hold there is not used
    Output:
        (y [B, T, C] of x's type, h [B, C] float32: the state after each row's last
        sample, ``h0`` of the samples that follow)
    """
    return recorded(_native_recurrence, x, f, g, h0, lengths)


def _native_recurrence(x, f, g, h0, lengths):
    return tuple(torch_binding().recurrence(x, f, g, h0, lengths))


def rms_norm(x, weight, residual=None, eps=1e-6, out_dtype=None):
    """Root-mean-square norm over the last dimension, the residual added before it.

    With r = x + residual: ``y = r / sqrt(mean(r^2) + eps) * weight``.

    Arguments:
        x: [..., C] float32 or bfloat16
        weight: [C] float32 or bfloat16
        residual: [..., C] of x's type or float32 (default: none)
        eps: float
        out_dtype: None for x's type, or torch.float8_e4m3fn: y in 8 bits with a
            scale per row, max |y| / 448 (no gradient: under ``torch.no_grad()``)
    Output:
        y, or (y, r) with a residual, r of the residual's type; in 8 bits
        (y, scale) or (y, scale, r), scale [...] float32: ``y.float() * scale[..., None]``
        is the norm's value
    """
    assert out_dtype in (None, x.dtype, torch.float8_e4m3fn), \
        'out_dtype must be None, the type of x, or torch.float8_e4m3fn'
    return recorded(_native_rms_norm, x, weight, residual, float(eps),
                    out_dtype == torch.float8_e4m3fn)


def _native_rms_norm(x, weight, residual, eps, eight):
    out = torch_binding().rms_norm(x, weight, residual, eps, eight)
    return out[0] if len(out) == 1 else tuple(out)
