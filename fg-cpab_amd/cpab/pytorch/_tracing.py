"""The native autograd functions under ``torch.jit.trace``.

The tracer does not see a native autograd function: it records the allocation of
its output and none of the work, so that a traced call would return memory that
nothing wrote.  While a trace is recorded the call goes through a Python autograd
function instead, which the tracer keeps as one operation and runs again with the
traced module's inputs (and which ``torch.jit.save`` refuses to export).
"""
import threading

import torch

__all__ = ["recorded"]


def recorded(function, *args):
    """``function(*args)``, kept as one operation by a trace in progress.

    The tracer compares a call's arguments by their text when it checks a trace:
    ``function`` is a module's, with everything it needs in ``args``.
    """
    if torch.jit.is_tracing():
        return _Recorded.apply(function, *args)
    return function(*args)


class _Recorded(torch.autograd.Function):
    """A native function with a graph of its own, held from forward to backward, where the
    caller's gradients are on (``needs_input_grad`` does not tell: a parameter asks for one
    under ``torch.no_grad()`` too)."""

    _caller = threading.local()

    @classmethod
    def apply(cls, *args):
        # what a trace runs again as well, each time in its caller's mode
        cls._caller.grad = torch.is_grad_enabled()
        return super().apply(*args)

    @staticmethod
    def forward(ctx, function, *args):
        grad = _Recorded._caller.grad
        with torch.set_grad_enabled(grad):
            ctx.args = [a.detach().requires_grad_(grad and need) if isinstance(a, torch.Tensor) else a
                        for a, need in zip(args, ctx.needs_input_grad[1:])]
            ctx.out = function(*ctx.args)
        if isinstance(ctx.out, torch.Tensor):
            return ctx.out.detach()
        return tuple(o.detach() for o in ctx.out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        wanted = [i for i, need in enumerate(ctx.needs_input_grad[1:]) if need]
        outs = (ctx.out,) if isinstance(ctx.out, torch.Tensor) else ctx.out
        kept = [(o, g) for o, g in zip(outs, grads) if o.requires_grad]
        grads = torch.autograd.grad([o for o, _ in kept], [ctx.args[i] for i in wanted],
                                    [g for _, g in kept], retain_graph=True, allow_unused=True)
        found = dict(zip(wanted, grads))
        return (None, *(found.get(i) for i in range(len(ctx.args))))
