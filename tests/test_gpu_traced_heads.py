"""The operators over heads in a module that torch.jit.trace has recorded: other inputs and
lengths than the trace's, their gradients, and torch.no_grad()."""
import pytest
import torch

import cpab

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::DeprecationWarning")]
B, T, H, K, D = 2, 70, 4, 2, 16


class Heads(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.inward = torch.nn.Linear(24, (2 * K + H) * D + 2 * H)
        self.q_weight, self.k_weight = (torch.nn.Parameter(D ** -0.5 * torch.ones(D)) for _ in range(2))
        self.register_buffer("freqs", torch.linspace(1.0, 0.1, D // 2))

    def forward(self, x, lengths):
        q, k, v, decay, beta = self.inward(x).split([K * D, K * D, H * D, H, H], -1)
        q, k = cpab.qk_norm(q.unflatten(-1, (K, D)), k.unflatten(-1, (K, D)), self.q_weight, self.k_weight, self.freqs)
        return cpab.gated_delta_rule(q, k, v.unflatten(-1, (H, D)), -torch.nn.functional.softplus(decay),
                                     torch.sigmoid(beta), None, lengths)


def test_traced(cuda):
    torch.manual_seed(0)
    net = Heads().to(cuda)
    x, z = (torch.randn(B, T, 24, device=cuda) for _ in range(2))
    traced = torch.jit.trace(net, (x, torch.tensor([T, 5], device=cuda)))
    n = torch.tensor([31, T], device=cuda)
    z.requires_grad_()
    got, want = traced(z, n), net(z, n)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    ups = [torch.randn_like(t) for t in want]
    for a, b in zip(torch.autograd.grad(got, (z, *traced.parameters()), ups),
                    torch.autograd.grad(want, (z, *net.parameters()), ups)):
        assert torch.equal(a, b)
    with torch.no_grad():
        out = traced(z, n)
        assert not out[0].requires_grad and all(torch.equal(a, b) for a, b in zip(out, net(z, n)))
