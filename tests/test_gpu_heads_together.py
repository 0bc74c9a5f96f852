"""Norms of queries and keys, the gated delta rule and Muon's step in a run, as a network
that reads signals has them, against their formulas in 64 bits.

Bound of the gradients and outputs: each of the run's steps (projection, norm, rule and the
product behind it, forwards and backwards) is off by at most 1e-5 of its result's norm, as
the steps' own tests hold it; the norm's rows come at a size near 1 and the rule's keys at
length 1 with beta below 1, so that no step grows what comes in by more than a small factor.
Eight steps, of which four at most (the rule's and the norm's, both ways) may double what
comes in: 2^4 x 8 x 1e-5 = 1.3e-3 in the worst case, where all errors point one way; as
independent ones, 2^4 x 8^(1/2) x 1e-5, 5e-4.  What a wrong formula or a stale value gives
is of the order of 1.  The captured step repeats the eager one's sums in the same order."""
import pytest
import torch

import cpab
import heads_oracle as ho

pytestmark = pytest.mark.gpu
F32 = torch.float32
H, K, D, W, OUT = 4, 2, 16, 24, 5
SIZES = {"wq": (K * D, W), "wk": (K * D, W), "wv": (H * D, W), "wg": (2 * H, W), "wo": (OUT, H * D)}


def weights(cuda, seed=0):
    gen = torch.Generator().manual_seed(seed)
    out = {n: torch.randn(s, generator=gen) * s[1] ** -0.5 for n, s in SIZES.items()}
    out["qn"], out["kn"] = (D ** -0.5 * (1 + 0.1 * torch.randn(D, generator=gen)) for _ in range(2))
    return {n: t.to(cuda).requires_grad_() for n, t in out.items()}


def network(w, x, norm, rule, freqs, positions=None, h0=None, lengths=None):
    B, T = x.shape[:2]
    q = (x @ w["wq"].T).view(B, T, K, D)
    k = (x @ w["wk"].T).view(B, T, K, D)
    v = (x @ w["wv"].T).view(B, T, H, D)
    gates = x @ w["wg"].T
    decay, beta = -torch.nn.functional.softplus(gates[..., :H]), torch.sigmoid(gates[..., H:])
    q, k = norm(q, k, w["qn"], w["kn"], freqs, positions)
    o, h = rule(q, k, v, decay, beta, h0, lengths)
    return o.reshape(B, T, H * D) @ w["wo"].T, h


def data(cuda, B, T, seed=1):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(B, T, W, generator=gen).to(cuda), torch.randn(B, T, OUT, generator=gen).to(cuda),
            torch.linspace(1.0, 0.01, D // 2).to(cuda))


def close(got, want, by=5e-4):
    got, want = ho.f64(got), ho.f64(want)
    assert torch.isfinite(got).all() and float((got - want).norm()) <= by * float(want.norm())


@pytest.mark.parametrize("B,T", [(3, 1), (2, 50), (2, 333)])
@pytest.mark.parametrize("ragged", [False, True])
def test_training_step(cuda, B, T, ragged):
    w = weights(cuda)
    x, up, freqs = data(cuda, B, T)
    lengths = torch.arange(T, T - B, -1, device=cuda).clamp(min=0) if ragged else None
    y, h = network(w, x, cpab.qk_norm, cpab.gated_delta_rule, freqs, lengths=lengths)
    (y * up).sum().backward()
    we = {n: ho.f64(t).requires_grad_() for n, t in w.items()}
    ye, he = network(we, ho.f64(x), ho.qk_norm, ho.delta_rule, ho.f64(freqs), lengths=None if lengths is None else lengths.cpu())
    (ye * ho.f64(up)).sum().backward()
    close(y, ye)
    close(h, he)
    for n in w:
        close(w[n].grad, we[n].grad)
    # the matrices move by Muon, the norms' weights by AdamW
    before = {n: (ho.f64(t), ho.f64(t.grad)) for n, t in w.items()}
    matrices = [t for t in w.values() if t.dim() == 2]
    muon = cpab.Muon(matrices, lr=0.02, weight_decay=0.1)
    adam = cpab.AdamW([w["qn"], w["kn"]], lr=0.02)
    muon.step()
    adam.step()
    for n, (p, g) in before.items():
        if p.dim() == 2:
            rows, cols = p.shape
            want, _ = ho.muon(p, g, torch.zeros_like(p), 0.02, 0.1, 0.95, True, (3.4445, -4.775, 2.0315), 1e-7, 5,
                              0.02 * max(1.0, rows / cols) ** 0.5)
            # the bound of the step's own test, on what moves
            assert float((ho.f64(w[n]) - want).norm()) <= 1e-5 * float((want - p).norm()) + 2.0 ** -22 * float(p.norm())
        else:
            assert not torch.equal(ho.f64(w[n]), p)
    again, _ = network(w, x, cpab.qk_norm, cpab.gated_delta_rule, freqs, lengths=lengths)
    close(again, network({n: ho.f64(t) for n, t in w.items()}, ho.f64(x), ho.qk_norm, ho.delta_rule, ho.f64(freqs),
                         lengths=None if lengths is None else lengths.cpu())[0])


def test_sample_by_sample_and_in_pieces(cuda):
    w = weights(cuda)
    B, T = 2, 90
    x, _, freqs = data(cuda, B, T)
    with torch.no_grad():
        whole, last = network(w, x, cpab.qk_norm, cpab.gated_delta_rule, freqs)
        # a prompt in one piece, then each sample as it comes
        parts, h, at = [], None, 0
        for n in (40, 17, *[1] * 33):
            where = torch.arange(at, at + n, device=cuda).expand(B, n)
            y, h = network(w, x[:, at:at + n], cpab.qk_norm, cpab.gated_delta_rule, freqs, where, h)
            parts.append(y)
            at += n
    assert at == T
    close(torch.cat(parts, 1), whole)
    close(h, last)


def test_a_captured_training_step(cuda):
    x, up, freqs = data(cuda, 2, 100)

    def start():
        w = weights(cuda)
        return w, [t for t in w.values() if t.dim() == 2], [torch.zeros_like(t) for t in w.values() if t.dim() == 2]

    def step(w, matrices, momenta):
        y, _ = network(w, x, cpab.qk_norm, cpab.gated_delta_rule, freqs)
        grads = torch.autograd.grad((y * up).sum(), list(w.values()))
        with torch.no_grad():
            cpab.muon_step(matrices, [g for g in grads if g.dim() == 2], momenta, lr=0.02)
        return y.detach()

    want, state = [], start()
    for _ in range(4):
        want.append((step(*state).clone(), [t.detach().clone() for t in state[1]]))
    state = start()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*state)
    torch.cuda.current_stream().wait_stream(side)
    first = start()
    with torch.no_grad():
        for to, of in zip([*state[0].values(), *state[2]], [*first[0].values(), *first[2]]):
            to.copy_(of)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(*state)
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        close(y, want[k][0], 1e-4)
        for a, b in zip(state[1], want[k][1]):
            close(a, b, 1e-4)
        eager = start()   # the program's own work between the replays
        assert torch.equal(step(*eager), want[0][0])
