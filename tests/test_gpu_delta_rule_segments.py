"""Gated delta rule where a head's axis is cut into segments: ragged rows, no state before,
widths that are padded; what a cleared state leaves; and how near bfloat16 results come.

The bounds of single values and of a result's whole are test_gpu_delta_rule.py's.  A
bfloat16 result w, rounded once from what is within 1e-5 of the whole, is off by what its
rounding leaves, evenly spread over a unit u of its last place: u^2 / 12 in the mean square,
u^4 / 180 in that square's variance.  Over n values the squares' sum is so within 8 roots of
the variances' sum of their mean (Chebyshev: 64 to 1 for any spread, and far rarer for a sum of many), and the whole within its root and 1e-5 of
the norm: near 1.6e-3, where a second rounding to 16 bits would leave 2.2e-3."""
import pytest
import torch

import cpab
import heads_oracle as ho
from test_gpu_delta_rule import NAMES, compare, make, zeroed

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


# With 256 compute units a call's heads are cut from 16 chunks on: 1100 samples of these into
# four segments of 320, 2100 into seven of 320.  On a card of another size they are cut
# elsewhere or not at all, and the results are the same.
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [1024, 1100, 2100])
@pytest.mark.parametrize("start", [True, False])
def test_ragged_rows(cuda, dtype, T, start):
    lengths = [T, 0, 70, T // 2, 320, 321, 640, T - 1, 1, 64]
    args, n = make(cuda, dtype, len(lengths), T, 2, 1, 20, 12, lengths=lengths, seed=41, start=start)
    compare(cuda, dtype, len(lengths), T, 2, 1, 20, 12, given=(args, n))


@pytest.mark.parametrize("dtype,gates", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("dk,dv", [(20, 40), (33, 21), (100, 8), (128, 70)])
def test_widths_and_no_start(cuda, dtype, gates, dk, dv):
    for start in (True, False):
        compare(cuda, dtype, 1, 1100, 2, 2, dk, dv, gates=gates, seed=42, start=start)


def test_rows_behind_their_end(cuda):
    # zeros behind every row's end, in each segment, and nothing of the inputs there is used
    T, lengths = 2100, [2100, 0, 70, 320, 321, 1000]
    args, n = make(cuda, F32, len(lengths), T, 2, 2, 16, 16, lengths=lengths, seed=43)

    def run(given):
        leaves = [t.detach().requires_grad_() for t in given]
        o, h = cpab.gated_delta_rule(*leaves, n)
        with torch.no_grad():
            alone = cpab.gated_delta_rule(*given, n)
        return (o, h, *alone, *torch.autograd.grad((o, h), leaves, (torch.ones_like(o), torch.ones_like(h))))
    got = run(args)
    clean = run([zeroed(t, n).to(cuda, t.dtype) for t in args[:5]] + [args[5]])
    assert all(torch.equal(a, b) for a, b in zip(got, clean))
    o, h, o_alone, h_alone, *grads = got
    assert torch.equal(o, o_alone) and torch.equal(h, h_alone)
    for b, k in enumerate(lengths):
        assert (o[b, k:] == 0).all()
        for g in grads[:5]:
            assert (g[b, k:] == 0).all()
        if k == 0:
            assert torch.equal(h[b], args[5][b]) and (grads[5][b] == 1).all()


@pytest.mark.parametrize("wanted", [(0,), (2,), (5,), (1, 3, 4)])
def test_parts_of_the_gradient(cuda, wanted):
    T, lengths = 1100, [1100, 0, 321]
    args, n = make(cuda, F32, 3, T, 2, 1, 20, 12, lengths=lengths, seed=44)
    ups = [torch.randn(3, T, 2, 12, device=cuda), torch.randn(3, 2, 20, 12, device=cuda)]

    def run(which, outs=(0, 1)):
        leaves = [t.detach().requires_grad_(i in which) for i, t in enumerate(args)]
        out = cpab.gated_delta_rule(*leaves, n)
        return torch.autograd.grad([out[k] for k in outs], [leaves[i] for i in which], [ups[k] for k in outs])
    full = run(range(6))
    assert all(torch.equal(g, full[i]) for g, i in zip(run(wanted), wanted))
    for k in (0, 1):   # of one output alone: the two add up
        ups[k].zero_()
        want = run(wanted)
        assert all(torch.equal(a, b) for a, b in zip(run(wanted, (1 - k,)), want))
        ups[k].normal_()


def test_graph_replays(cuda):
    args, n = make(cuda, BF16, 3, 1100, 2, 1, 32, 40, lengths=[1100, 0, 321], seed=45)

    def passes(given):
        leaves = [t.detach().requires_grad_() for t in given]
        out = cpab.gated_delta_rule(*leaves, n)
        with torch.no_grad():
            alone = cpab.gated_delta_rule(*given, n)
        return (*out, *alone, *torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes(args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = passes(args)
    for seed in range(46, 49):
        new, other = make(cuda, BF16, 3, 1100, 2, 1, 32, 40, lengths=[1100 - seed, seed, 640], seed=seed)
        n.copy_(other)
        for a, b in zip(args, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, passes(new)))


@pytest.mark.parametrize("T", [9, 150, 1100])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_what_a_cleared_state_leaves(cuda, dtype, T):
    # the samples from a cleared state on are those of a call that begins there, of another
    # state: the products' order in the chunks differs, and no more
    args, _ = make(cuda, dtype, 2, T, 2, 1, 24, 16, seed=47)
    q, k, v, decay, beta, h0 = args
    at = T // 2
    cleared = decay.clone()
    cleared[:, at] = -float("inf")
    o, h = cpab.gated_delta_rule(q, k, v, cleared, beta, 100 * h0)
    rest = [t[:, at:] for t in (q, k, v, decay, beta)]
    ro, rh = ho.delta_rule(*(ho.f64(t) for t in rest[:3]), ho.f64(rest[3]).index_fill(1, torch.tensor([0]), -1e4),
                           ho.f64(rest[4]))
    unit = 2.0 ** -8 if dtype == BF16 else 0.0
    for got, want in ((o[:, at:], ro), (h, rh), (cpab.gated_delta_rule(*rest)[0], ro)):
        out = 1e-5 + (unit if got.dtype == BF16 else 0.0)
        assert float((ho.f64(got) - want).norm()) <= out * float(want.norm())


def within_rounding(got, want, what):
    got, want = ho.f64(got).flatten(), want.flatten()
    unit = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=1e-30))) - 7)
    most = ((unit ** 2 / 12).sum() + 8 * (unit ** 4 / 180).sum().sqrt()).sqrt() + 1e-5 * want.norm()
    off = (got - want).norm()
    assert off <= most, f"{what}: {float(off / want.norm()):.3g} of the whole, {float(most / want.norm()):.3g} from rounding"


@pytest.mark.parametrize("gates", [BF16, F32])
@pytest.mark.parametrize("B,T,H,K,dk,dv", [(2, 300, 4, 2, 64, 64), (1, 1100, 2, 2, 128, 128), (3, 130, 3, 1, 40, 72)])
def test_bfloat16_results_are_rounded_once(cuda, gates, B, T, H, K, dk, dv):
    args, _ = make(cuda, BF16, B, T, H, K, dk, dv, gates=gates, seed=48)
    leaves = [t.detach().requires_grad_() for t in args]
    o, h = cpab.gated_delta_rule(*leaves)
    gen = torch.Generator().manual_seed(49)
    do, dh = torch.randn(o.shape, generator=gen).to(cuda, BF16), torch.randn(h.shape, generator=gen).to(cuda)
    grads = dict(zip(NAMES, torch.autograd.grad((o, h), leaves, (do, dh))))
    ref = [ho.f64(t) for t in args]
    want, _ = ho.delta_rule_grads(*ref, None, None, ho.f64(do), ho.f64(dh))
    want["o"] = ho.delta_rule(*ref)[0]
    with torch.no_grad():
        grads.update(o=o, alone=cpab.gated_delta_rule(*args)[0])
    want["alone"] = want["o"]
    for name, got in grads.items():
        if got.dtype == BF16:
            within_rounding(got, want[name], name)
