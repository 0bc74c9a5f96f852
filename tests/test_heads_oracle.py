"""The oracle's own formulas of the operators over heads, on the CPU: gradients written out
against automatic ones, and the chunks' formulas against the definition."""
import pytest
import torch

import heads_oracle as ho


def sample(B=2, T=9, H=4, K=2, dk=5, dv=3, seed=0):
    gen = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(B, T, K, dk, generator=gen).double() for _ in range(2))
    k = k / k.norm(dim=-1, keepdim=True)
    v = torch.randn(B, T, H, dv, generator=gen).double()
    decay = -torch.rand(B, T, H, generator=gen).double()
    beta = torch.rand(B, T, H, generator=gen).double()
    return q, k, v, decay, beta, torch.randn(B, H, dk, dv, generator=gen).double()


@pytest.mark.parametrize("lengths", [None, torch.tensor([4, 0]), torch.tensor([9, 12])])
def test_delta_rule_gradients(lengths):
    given = [t.requires_grad_() for t in sample()]
    o, h = ho.delta_rule(*given, lengths=lengths)
    do, dh = torch.randn_like(o), torch.randn_like(h)
    want = torch.autograd.grad((o, h), given, (do, dh))
    got, size = ho.delta_rule_grads(*(t.detach() for t in given), lengths, None, do, dh)
    for name, w in zip(("q", "k", "v", "decay", "beta", "h0"), want):
        assert torch.allclose(got[name], w, rtol=1e-10, atol=1e-12), name
    assert size["S"] > 0 and size["L"] > 0


def test_chunk_formulas():
    # X = (I - M beta) R, U = beta X, and the state after, against the definition
    T = 9
    q, k, v, decay, beta, h0 = (t[:1, :, :1] if t.dim() < 4 or t.shape[1] == T else t[:1, :1] for t in sample(H=1, K=1))
    o, h = ho.delta_rule(q, k, v, decay, beta, h0)
    q, k, v, decay, beta, S = q[0, :, 0], k[0, :, 0], v[0, :, 0], decay[0, :, 0], beta[0, :, 0], h0[0, 0]
    G = decay.cumsum(0)
    D = torch.exp(G[:, None] - G[None]).tril()
    A, P = (D * (k @ k.T)).tril(-1), 5 ** -0.5 * D * (q @ k.T)
    M = A @ torch.linalg.inv(torch.eye(T).double() + beta[:, None] * A)
    R = v - G.exp()[:, None] * (k @ S)
    U = beta[:, None] * (R - M @ (beta[:, None] * R))
    assert torch.allclose(5 ** -0.5 * G.exp()[:, None] * (q @ S) + P @ U, o[0, :, 0])
    after = G[-1].exp() * S + k.T @ ((G[-1] - G).exp()[:, None] * U)
    assert torch.allclose(after, h[0, 0])


def test_turning_is_a_rotation():
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(2, 5, 3, 8, generator=gen).double()
    freqs = torch.tensor([1.0, 0.5, 0.1]).double()
    for neighbours in (False, True):
        y = ho.turned(x, freqs, None, neighbours)
        assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1)) and torch.equal(y[..., 6:], x[..., 6:])
        assert torch.allclose(ho.turned(y, freqs, None, neighbours, -1.0), x)
        # position 0 turns nothing
        assert torch.equal(y[:, 0], x[:, 0])


def test_muon_of_both_shapes():
    # a matrix and its transposed one take the same step, transposed; and the singular values
    # of the step are near 1
    gen = torch.Generator().manual_seed(2)
    g, m = torch.randn(6, 11, generator=gen).double(), torch.randn(6, 11, generator=gen).double()
    p = torch.zeros(6, 11).double()
    args = (0.1, 0.0, 0.9, True, (3.4445, -4.775, 2.0315), 1e-7, 5, 1.0)
    a, b = ho.muon(p, g, m, *args)[0], ho.muon(p.T, g.T, m.T, *args)[0]
    assert torch.allclose(a, b.T)
    s = torch.linalg.svdvals(a)
    assert 0.6 < s.min() and s.max() < 1.3
