"""Aligns a set of signals: a network reads each one and gives the theta that warps it.

    PYTHONPATH=fg-cpab_amd python examples/align_signals.py

The network is a stack of gated recurrences (``cpab.gated_recurrence``) with
root-mean-square norms that add the residual (``cpab.rms_norm``); its theta warps the
signal through ``Cpab.transform_data``; the loss is the variance of the warped signals
around their mean, and ``cpab.AdamW`` moves the weights, its states in 8 bits.  Trained,
the network is also run as signals arrive, sample by sample, and with 8-bit norms.
"""
import argparse

import torch
from torch import nn

import cpab
from cpab import Cpab


class Block(nn.Module):
    def __init__(self, width):
        super().__init__()
        self.norm = nn.Parameter(torch.ones(width))
        self.into = nn.Linear(width, 3 * width)
        self.out = nn.Linear(width, width)
        with torch.no_grad():   # gates that remember from a few samples to hundreds
            self.into.bias[width:2 * width] = torch.linspace(0, 6, width)


class Encoder(nn.Module):
    """Signals [B, T] to theta [B, d]."""

    def __init__(self, d, width=64, layers=3):
        super().__init__()
        self.embed = nn.Linear(1, width)
        self.blocks = nn.ModuleList(Block(width) for _ in range(layers))
        self.norm = nn.Parameter(torch.ones(width))
        self.head = nn.Linear(width, d)
        nn.init.normal_(self.head.weight, std=1e-3)
        nn.init.zeros_(self.head.bias)

    def forward(self, signals, lengths=None, states=None, eight=False):
        """(theta, the state after each signal's last sample).  `states`: those of the
        samples before.  `eight`: norms in 8 bits, without gradients."""
        x, residual, after = self.embed(signals[..., None]), None, []
        for k, block in enumerate(self.blocks):
            y, residual = self._norm(x, block.norm, residual, eight)
            a, f, g = self._product(y, block.into, eight).chunk(3, -1)
            y, h = cpab.gated_recurrence(a, f, g, None if states is None else states[k], lengths)
            after.append(h)
            x = block.out(y)
        y, _ = self._norm(x, self.norm, residual, eight)
        y = self._product(y, self.head, eight)
        if lengths is None:
            return y[:, -1], after
        last = (lengths.long() - 1).clamp(min=0)
        return y[torch.arange(len(y), device=y.device), last], after

    @staticmethod
    def _norm(x, weight, residual, eight):
        kind = torch.float8_e4m3fn if eight else None
        if residual is None:
            y = cpab.rms_norm(x, weight, out_dtype=kind)
            return y, x
        *y, r = cpab.rms_norm(x, weight, residual=residual, out_dtype=kind)
        return (tuple(y) if eight else y[0]), r

    @staticmethod
    def _product(y, linear, eight):
        if not eight:
            return linear(y)
        q, scale = y
        return (q.to(linear.weight.dtype) @ linear.weight.t()) * scale[..., None] + linear.bias


def make_signals(T, n, samples, device):
    """n smooth signals of one class, each moved by a warp of its own."""
    t = torch.linspace(0, 1, samples, device=device)
    base = torch.exp(-((t - 0.3) / 0.06) ** 2) - 0.7 * torch.exp(-((t - 0.65) / 0.1) ** 2)
    theta = 0.5 * T.sample_transformation(n)
    with torch.no_grad():
        return T.transform_data(base.expand(n, 1, samples).contiguous(), theta, [samples])[:, 0]


def spread(warped):
    """Variance of the signals around their mean."""
    return ((warped - warped.mean(0)) ** 2).mean()


def train(signals, T, steps=60, lr=3e-3, state_bits=8, log=None):
    """(the trained encoder, the losses)."""
    n, samples = signals.shape
    net = Encoder(T.get_theta_dim()).to(signals.device)
    opt = cpab.AdamW(net.parameters(), lr=lr, state_bits=state_bits)
    losses = []
    for step in range(steps):
        theta, _ = net(signals)
        warped = T.transform_data(signals[:, None], theta, [samples])[:, 0]
        loss = spread(warped) + 1e-4 * theta.square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        if log and step % 10 == 0:
            log(f"step {step}: loss {float(losses[-1]):.5f}")
    return net, torch.stack(losses).tolist()


def stream(net, signals):
    """theta after the last sample, the signals read one sample at a time."""
    states = None
    with torch.no_grad():
        for t in range(signals.shape[1]):
            theta, states = net(signals[:, t:t + 1], states=states)
    return theta


def main():
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--signals", type=int, default=32)
    parser.add_argument("--samples", type=int, default=1000)
    parser.add_argument("--steps", type=int, default=60)
    args = parser.parse_args()
    torch.manual_seed(0)
    T = Cpab([16])
    signals = make_signals(T, args.signals, args.samples, torch.device("cuda"))
    net, losses = train(signals, T, args.steps, log=print)
    print(f"variance before {float(spread(signals)):.5f}, loss after {losses[-1]:.5f}")
    with torch.no_grad():
        theta, _ = net(signals)
        eight, _ = net(signals, eight=True)
    print(f"theta sample by sample: off by {float((stream(net, signals) - theta).abs().max()):.2g}")
    print(f"theta with 8-bit norms: off by {float((eight - theta).abs().max()):.2g} of {float(theta.abs().max()):.2g}")


if __name__ == "__main__":
    main()
