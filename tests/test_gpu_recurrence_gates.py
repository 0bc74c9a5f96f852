"""The recurrence's gradient through gates that are closed, or nearly: a loss on the last
state alone, whose gradient comes to a sample through the gates behind it and no other way,
so that a bound on each value's own size holds.

Bounds, from the arithmetic (u = 2^-24).  A gate and its complement carry |f| u from the
scaling of exp's argument and 4 u from exp, the sum, the reciprocal and the difference: r =
(|f| + 4) u of the value.  With l = dh times the gates behind a sample, each gate brings its r
and 2 u for its products: R = the sum of those.  So grad x = (1 - a) l carries R + r + 2 u
of its value, grad h0 = l over all gates R + 2 u, and grad f = l (h - x) a (1 - a) R + 2 r + 4 u
and what h is off, at most 18 u N M with M the largest size and N the samples that a gate remembers.
bfloat16 results carry half a unit of their last place, at most 2^-8 of the value, besides; what
lies below the normal numbers is not asked for."""
import pytest
import torch

import cpab
import sequence_oracle as so

pytestmark = pytest.mark.gpu
U = so.U


def compare(cuda, dtype, x, f, g, h0, dh, lengths=None):
    B, T, C = x.shape
    x, f = x.to(dtype).to(cuda), f.to(dtype).to(cuda)
    leaves = [t.requires_grad_() for t in (x, f, h0.to(cuda))]
    n = None if lengths is None else torch.tensor(lengths)
    _, h = cpab.gated_recurrence(leaves[0], leaves[1], g if g is None else g.to(dtype).to(cuda), leaves[2],
                                 n if n is None else n.to(cuda))
    gx, gf, gh = torch.autograd.grad(h, leaves, dh.to(cuda))
    X, F, H0, DH = (so.f64(t) for t in (*leaves, dh))
    want = so.recurrence_grads(X, F, None, H0, n, torch.zeros_like(X), DH)
    states = so.recurrence(X, F, None, H0, n)[2]
    a, k = torch.sigmoid(F), torch.sigmoid(-F)
    r = (F.abs() + 4) * U
    live = torch.ones(B, T, 1, dtype=torch.float64)
    if n is not None:
        live = (torch.arange(T)[None, :] < n[:, None])[..., None].double()
    R = ((r + 2 * U) * live).flip(1).cumsum(1).flip(1)     # of the gates from a sample on
    after = torch.cat([R[:, 1:], torch.zeros(B, 1, C, dtype=torch.float64)], 1)
    unit = 0.0 if dtype == torch.float32 else so.UNIT[dtype]
    off = 18 * U * so.recurrence_memory(F, T) * float(max(X.abs().max(), H0.abs().max()))
    # by the formula: differentiating sigmoid(-f) itself as s (1 - s) loses a small 1 - s in 64 bits too
    l = want["x"] / k
    want["f"] = l * (states[:, :T] - X) * a * k
    for what, got, exact, bound in (
            ("grad h0", gh, want["h0"], (R[:, 0] + 2 * U) * want["h0"].abs()),
            ("grad x", gx, want["x"], (after + r + 2 * U + unit) * want["x"].abs()),
            ("grad f", gf, want["f"], (after + 2 * r + 4 * U + unit) * want["f"].abs()
             + l.abs() * a * k * (off + U * (states[:, :T] - X).abs()))):
        over = (so.f64(got) - exact).abs() - bound * 1.01 - 1e-38
        at = over.argmax()
        assert over.max() <= 0, (what, float(exact.reshape(-1)[at]), float(so.f64(got).reshape(-1)[at]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mean", [-60.0, -30.0, -18.0, -14.0, -10.0, -6.0, 0.0, 14.0])
@pytest.mark.parametrize("gate", [False, True])
def test_one_sample(cuda, dtype, mean, gate):
    gen = torch.Generator().manual_seed(int(mean) + 100)
    x, f, g = (torch.randn(3, 1, 130, generator=gen) for _ in range(3))
    h0, dh = (torch.randn(3, 130, generator=gen) for _ in range(2))
    compare(cuda, dtype, x, mean + 0.5 * f, g if gate else None, h0, dh)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [2, 5, 16, 17, 40])
def test_closed_all_along(cuda, dtype, T):
    gen = torch.Generator().manual_seed(T)
    x, f = (torch.randn(2, T, 37, generator=gen) for _ in range(2))
    h0, dh = (torch.randn(2, 37, generator=gen) for _ in range(2))
    compare(cuda, dtype, x, -60.0 / T + f.clamp(-1, 1), None, h0, dh)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,C", [(60, 33), (300, 40), (1300, 8), (2500, 70)])
def test_closed_now_and_then(cuda, dtype, T, C):
    # open gates, and three closed ones for each channel, at any place of a tile
    gen = torch.Generator().manual_seed(T + C)
    x = torch.randn(2, T, C, generator=gen)
    f = 8 + 0.5 * torch.randn(2, T, C, generator=gen).clamp(-1, 1)
    at = torch.randint(0, T // 2, (2, 3, C), generator=gen)
    f.scatter_(1, at, -18 + 5 * torch.rand(2, 3, C, generator=gen))
    h0, dh = (torch.randn(2, C, generator=gen) for _ in range(2))
    compare(cuda, dtype, x, f, None, h0, dh)
    compare(cuda, dtype, x, f, None, h0, dh, lengths=[T - T // 4, T])
