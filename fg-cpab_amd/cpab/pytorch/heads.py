"""Operators over heads, of a network that reads long signals and gives theta.

``gated_delta_rule`` (a scan with a matrix of state for each head, with its backward) and
``qk_norm`` (the norms of queries and keys by head, rotated by the position).  HIP kernels behind the C ABI, called from native functions (csrc/torch_heads.cpp); there is no
torch or CPU fallback.  No counterpart in the reference, whose networks are torch modules
(``stn/demos/*.py``).
"""
from ._native import torch_binding
from ._tracing import recorded

__all__ = ["gated_delta_rule", "qk_norm"]


def gated_delta_rule(q, k, v, decay, beta, h0=None, lengths=None, scale=None):
    """The gated delta rule over each row's samples: a state S [dk, dv] for each head
    that a sample's key and value correct, and its query reads.

        S' = exp(decay_t) S_{t-1},   S_t = S' + beta_t k_t (v_t - S'^T k_t)^T,
        o_t = scale S_t^T q_t

    The state is held in 32 bits, and so is what passes between samples.  Products take it
    to 24 bits; those whose result is rounded to bfloat16 to 17 (outputs of bfloat16 inputs,
    and their gradients where decay and beta are bfloat16 too): within 1e-5 of the whole
    before that rounding.  What is not finite in a sample reaches its row's head from the 64
    samples around it on (the formula's own reach is from the sample on), and, as a head's
    key or query, the heads that share it; no other row and no other head.

    Arguments:
        q, k: [B, T, key heads, dk] of v's type, dk from 1 to 128.  Keys longer than 1 can
            make the state grow without bound, as they do in the formula
        v: [B, T, heads, dv] float32 or bfloat16; heads is a multiple of the key heads,
            neighbouring ones share a query and a key.  Slices of one projection's output
            are read where they lie (any strides over B, T and the heads; others are
            copied first)
        decay: [B, T, heads] float32 or bfloat16, the decay's logarithm, at most 0 (-inf
            clears the state; below -128 it counts as -128, which is the same)
        beta: [B, T, heads] of decay's type, how much of the difference is written
        h0: [B, heads, dk, dv] float32, the state before the first sample (default: zeros)
        lengths: [B] int32 or int64, samples in each row (default: T; clamped to
            [0, T]).  Behind a row's end o is 0 and the state stays; what the inputs
            hold there is not used
        scale: float, of the output (default: 1 / sqrt(dk))
    Output:
        (o [B, T, heads, dv] of v's type, h [B, heads, dk, dv] float32: the state after
        each row's last sample, ``h0`` of the samples that follow)
    """
    return recorded(_native_delta_rule, q, k, v, decay, beta, h0, lengths,
                    None if scale is None else float(scale))


def _native_delta_rule(q, k, v, decay, beta, h0, lengths, scale):
    return tuple(torch_binding().delta_rule(q, k, v, decay, beta, h0, lengths, scale))


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
            gradient (default, or no values: nothing turns)
        positions: [B, T] (or what broadcasts to it: [T], [B, 1]) int32, int64 or float32,
            the samples' places or times; no gradient (default: 0 to T - 1).  They are not
            taken without freqs; freqs of no values leave them unread
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
