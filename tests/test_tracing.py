"""Calls kept by torch.jit.trace, with a function on the CPU in a native one's place: they
run in the caller's gradient mode, while the trace is recorded and when it runs again."""
import pytest
import torch

from cpab.pytorch import _tracing

pytestmark = pytest.mark.filterwarnings("ignore::DeprecationWarning")
modes = []


def pair(x, w, refuses):
    """Two outputs; like a function without a gradient it may refuse inputs that ask for one."""
    modes.append(torch.is_grad_enabled() and any(t.requires_grad for t in (x, w)))
    if refuses and modes[-1]:
        raise RuntimeError("no gradient; call it under torch.no_grad()")
    return x * w, (x + w).sum()


def single(x, w):
    return pair(x, w, False)[0]


class Net(torch.nn.Module):
    def __init__(self, function, *more):
        super().__init__()
        self.w = torch.nn.Parameter(torch.randn(3))
        self.call = lambda x: _tracing.recorded(function, x, self.w, *more)

    def forward(self, x):
        return self.call(2 * x)


def test_without_gradients_under_no_grad():
    x, net = torch.randn(3), Net(pair, True)
    with torch.no_grad():
        m = torch.jit.trace(net, (x,))
        a, b = m(torch.ones(3))
    assert torch.equal(a, 2 * net.w) and torch.equal(b, (2 + net.w).sum())
    assert not a.requires_grad and not b.requires_grad
    # with gradients on it is refused, as it is without a trace
    with pytest.raises(RuntimeError, match="no_grad"):
        torch.jit.trace(net, (x,))
    with pytest.raises(RuntimeError, match="no_grad"):
        m(x)


def test_the_mode_of_each_run():
    # recorded without gradients and run with them, and the other way round
    x, net = torch.randn(3), Net(single)
    with torch.no_grad():
        m = torch.jit.trace(net, (x,))
    del modes[:]
    grad, = torch.autograd.grad(m(x).sum(), m.w)
    assert modes == [True]
    torch.testing.assert_close(grad, 2 * x)
    m = torch.jit.trace(net, (x,))
    del modes[:]
    with torch.no_grad():
        assert torch.equal(m(x), 2 * x * net.w) and not m(x).requires_grad
    assert modes == [False, False]      # and so keeps nothing for a backward
    grad, = torch.autograd.grad(m(x).sum(), m.w)
    torch.testing.assert_close(grad, 2 * x)


def test_several_outputs():
    x, net = torch.randn(3), Net(pair, False)
    m = torch.jit.trace(net, (x,))
    a, b = m(x)
    grad, = torch.autograd.grad(a.sum() + 3 * b, m.w)
    torch.testing.assert_close(grad, 2 * x + 3)
    a, b = m(x)
    torch.testing.assert_close(torch.autograd.grad(b, m.w)[0], torch.ones(3))
