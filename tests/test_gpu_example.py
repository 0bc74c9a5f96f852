"""The example that runs the operators around the transform together: a network reads
signals and gives theta, trained through the transform, then run sample by sample."""
import importlib.util
import os

import pytest
import torch

from cpab import Cpab

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(__file__))), "examples",
                    "align_signals.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("align_signals", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("bits", [8, 32])
def test_training_aligns(cuda, example, bits):
    torch.manual_seed(0)
    T = Cpab([16])
    signals = example.make_signals(T, 16, 400, cuda)
    net, losses = example.train(signals, T, steps=40, state_bits=bits)
    assert losses[-1] < 0.6 * losses[0]
    with torch.no_grad():
        theta, _ = net(signals)
        eight, _ = net(signals, eight=True)
    # sample by sample the same network in another order of rounding: each layer's
    # result to a few 2^-24 of its terms, some hundreds of them
    scale = float(theta.abs().max())
    assert float((example.stream(net, signals) - theta).abs().max()) <= 1e-4 * scale + 1e-6
    # an 8-bit norm is off by up to 2^-4 of a value, at random over a product's 64 terms
    # and four norms in a row
    assert float((eight - theta).abs().max()) <= 0.25 * scale


def test_ragged_signals_as_if_alone(cuda, example):
    torch.manual_seed(1)
    T = Cpab([8])
    net = example.Encoder(T.get_theta_dim(), width=24, layers=2).to(cuda)
    torch.nn.init.normal_(net.head.weight)
    signals = example.make_signals(T, 4, 300, cuda)
    lengths = torch.tensor([300, 17, 128, 1], device=cuda)
    with torch.no_grad():
        whole, states = net(signals, lengths)
        for b, n in enumerate(lengths.tolist()):
            alone, own = net(signals[b:b + 1, :n])
            torch.testing.assert_close(whole[b:b + 1], alone, rtol=1e-4, atol=1e-4)
            for s, o in zip(states, own):
                torch.testing.assert_close(s[b:b + 1], o, rtol=1e-4, atol=1e-4)
