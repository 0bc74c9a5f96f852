"""Gradients of a norm whose residual has 16 bits: they are those of the sum itself, not of
the sum rounded to the residual's type.

Bounds, from the arithmetic (u = 2^-24): the sum of two 16-bit values carries a unit u in 32
bits, the mean of its squares (C / 64 + 20) u at most, so n = r s carries e = (C / 128 + 16) u
of its value; a term of the weight's gradient 8 u besides, `rows` of them added in some
order rows u of the sum of their sizes; the mean of u n (C / 64 + 40) u of the mean of
|u n| and 2 e.  What is stored in 16 bits carries half a unit of its last place, at most
2^-8 of the value.  A sum rounded to 16 bits would add 2^-8 of each term."""
import pytest
import torch

import cpab
import sequence_oracle as so

pytestmark = pytest.mark.gpu
U, BF16 = so.U, torch.bfloat16
HALF = 2.0 ** -8 * 1.01


@pytest.mark.parametrize("wtype", [BF16, torch.float32])
@pytest.mark.parametrize("rows,C", [(1, 7), (1, 1000), (3, 1024), (2, 4200), (2, 20000), (1, 40001), (300, 64)])
def test_gradients_of_the_sum_itself(cuda, wtype, rows, C):
    gen = torch.Generator().manual_seed(rows * 31 + C)
    x, res, dy = (torch.randn(rows, C, generator=gen).to(BF16).to(cuda) for _ in range(3))
    w = (1 + 0.3 * torch.randn(C, generator=gen)).to(wtype).to(cuda)
    leaves = [t.requires_grad_() for t in (x, w, res)]
    y, r = cpab.rms_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    X, W, R, DY = (so.f64(t) for t in (x, w, res, dy))
    want = so.rms_norm_grads(X, W, R, 1e-6, DY, None)
    _, rr, s = so.rms_norm(X, W, R)
    n, v, e = rr * s, (DY * W).abs(), (C / 128 + 16) * U
    size = (DY * n).abs().sum(0)
    unit = HALF if wtype == BF16 else 0.0
    over = (so.f64(grads[1]) - want[1]).abs() - (((rows + 8) * U + e) * size + (unit + U) * want[1].abs())
    assert over.max() <= 0, ("grad weight", float(over.max()))
    mean = (v * n.abs()).mean(-1, keepdim=True)
    bound = s * ((e + 8 * U) * v + n.abs() * mean * ((C / 64 + 40) * U + 2 * e))
    for got, exact in ((grads[0], want[0]), (grads[2], want[2])):
        over = (so.f64(got) - exact).abs() - (bound * 1.001 + (HALF + 4 * U) * exact.abs())
        assert over.max() <= 0, ("grad", float(over.max()))
