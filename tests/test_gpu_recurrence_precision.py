"""Gates of 32-bit inputs carry a few units in their last place, however far they are closed.

Bounds, from the arithmetic (u = 2^-24): exp2 of the rounded argument 2 u, what the rounding
takes back 1 u, the sum 1 u, the reciprocal 2 u, the product 1 u: 7 u of the smaller of a gate
and its complement, which is the gate's error too where it is the larger and half a unit
more.  A state that is one such product, or one and an addition of 0, carries 9 u, with the
output gate's 7 u and two products 20 u."""
import pytest
import torch

import cpab
import sequence_oracle as so

pytestmark = pytest.mark.gpu
U = so.U


def off(got, want):
    return float(((so.f64(got) - want).abs() / want.abs()).max()) / U


@pytest.mark.parametrize("T", [1, 3, 40])
def test_gates_of_any_size(cuda, T):
    # sample 0 of each row is the one that is looked at, the others hold the state
    gen = torch.Generator().manual_seed(T)
    f = torch.full((2, T, 4001), 300.0)
    f[:, 0] = torch.linspace(-85, 85, 4001) + torch.rand(2, 4001, generator=gen) * 0.04
    f = f.to(cuda)
    F = so.f64(f[:, 0])
    zero, one = torch.zeros(2, T, 4001, device=cuda), torch.ones(2, T, 4001, device=cuda)
    h0 = torch.ones(2, 4001, device=cuda, requires_grad=True)
    y, h = cpab.gated_recurrence(zero, f, h0=h0)
    assert off(h, torch.sigmoid(F)) <= 9 and off(y[:, 0], torch.sigmoid(F)) <= 9
    assert off(torch.autograd.grad(h, h0, torch.ones_like(h))[0], torch.sigmoid(F)) <= 9
    x = one.clone().requires_grad_()
    _, h = cpab.gated_recurrence(x, f)
    assert off(h, torch.sigmoid(-F)) <= 9
    assert off(torch.autograd.grad(h, x, torch.ones_like(h))[0][:, 0], torch.sigmoid(-F)) <= 9
    y, _ = cpab.gated_recurrence(one, torch.full_like(f, -300.0), f)
    assert off(y[:, 0], F * torch.sigmoid(F)) <= 20


def test_ends_of_the_type(cuda):
    h0 = torch.tensor([[2.0]], device=cuda)
    for size in (120.0, 1e6, 2e38, 3e38, float("inf")):
        for sign, want in ((1, 2.0), (-1, 3.0)):
            f = torch.full((1, 1, 1), sign * size, device=cuda, requires_grad=True)
            x = torch.full((1, 1, 1), 3.0, device=cuda)
            _, h = cpab.gated_recurrence(x, f, h0=h0)
            assert float(h.detach()) == want
            assert float(torch.autograd.grad(h.sum(), f)[0]) == 0
    f = torch.full((1, 1, 1), float("nan"), device=cuda)
    assert torch.isnan(cpab.gated_recurrence(x, f, h0=h0)[1]).all()
