"""The norm in modules that torch.jit.trace has recorded: its 8-bit output under
torch.no_grad(), and both outputs with their gradients."""
import pytest
import torch

import cpab

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::DeprecationWarning")]
E4M3 = torch.float8_e4m3fn


class Norm(torch.nn.Module):
    def __init__(self, kind):
        super().__init__()
        self.weight = torch.nn.Parameter(1 + 0.3 * torch.randn(48))
        self.kind = kind

    def forward(self, x, residual):
        return cpab.rms_norm(2 * x, self.weight, residual, out_dtype=self.kind)


def test_8_bits_without_gradients(cuda):
    net = Norm(E4M3).to(cuda)
    x, r, z, t = (torch.randn(5, 48, device=cuda) for _ in range(4))
    with torch.no_grad():
        m = torch.jit.trace(net, (x, r), check_trace=False)   # the check knows no 8-bit comparison
        got, want = m(z, t), net(z, t)
    assert got[0].dtype == E4M3 and torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8))
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    with pytest.raises(RuntimeError, match="no gradient"):
        m(z, t)


def test_both_outputs(cuda):
    net = Norm(None).to(cuda)
    x, r, z, t, dy, ds = (torch.randn(5, 48, device=cuda) for _ in range(6))
    m = torch.jit.trace(net, (x, r))
    z.requires_grad_(), t.requires_grad_()
    got, want = m(z, t), net(z, t)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for a, b in zip(torch.autograd.grad(got, (z, t, m.weight), (dy, ds)),
                    torch.autograd.grad(want, (z, t, net.weight), (dy, ds))):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert not m(z, t)[0].requires_grad
