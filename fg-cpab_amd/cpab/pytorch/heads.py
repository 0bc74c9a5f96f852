"""Operators over heads, of a network that reads long signals and gives theta.

``qk_norm`` (the norms of queries and keys by head, rotated by the position).  HIP
kernels behind the C ABI, called from native functions (csrc/torch_heads.cpp); there is no
torch or CPU fallback.  No counterpart in the reference, whose networks are torch modules
(``stn/demos/*.py``).
"""
from ._native import torch_binding
from ._tracing import recorded

__all__ = ["qk_norm"]


def qk_norm(q, k, q_weight, k_weight, freqs=None, positions=None, neighbours=False, eps=1e-6):
    """Root-mean-square norms of queries and keys by head, rotated by the position.

    For each head's values x: ``y = x / sqrt(mean(x^2) + eps) * weight``; with ``freqs``
    the first ``2 len(freqs)`` of them, as pairs (a, b), turn by the angle
    p = position * freqs[pair]: ``(a cos p - b sin p, b cos p + a sin p)``.

    Arguments:
        q: [B, T, heads, width] float32 or bfloat16, width at most 512; slices of one
            projection's output are read where they lie (any strides over B, T and the
            heads; width of other strides is copied first)
        k: [B, T, key heads, width] of q's type
        q_weight, k_weight: [width] float32 or bfloat16, both of one type
        freqs: float32, radians for each unit of position, at most width / 2 of them; no
            gradient (default: nothing turns)
        positions: [B, T] (or what broadcasts to it: [T], [B, 1]) int32, int64 or float32,
            the samples' places or times; no gradient (default: 0 to T - 1)
        neighbours: bool, pairs are two values side by side, (0, 1), (2, 3), ...; else
            len(freqs) apart, (0, n), (1, n + 1), ...
        eps: float
    Output:
        (q, k) of the inputs' shapes and type
    """
    return recorded(_native_qk_norm, q, k, q_weight, k_weight, freqs, positions, bool(neighbours),
                    float(eps))


def _native_qk_norm(q, k, q_weight, k_weight, freqs, positions, neighbours, eps):
    return tuple(torch_binding().qk_norm(q, k, q_weight, k_weight, freqs, positions, neighbours, eps))
