"""A step that cpab.AdamW refuses is not counted: the next one is what it would have been."""
import pytest
import torch

import cpab

pytestmark = pytest.mark.gpu


def pair(cuda):
    gen = torch.Generator().manual_seed(1)
    return [torch.nn.Parameter(torch.randn(n, 4, generator=gen).to(cuda)) for n in (5, 6)]


def test_sparse_gradient(cuda):
    # the second parameter's gradient is refused: neither is stepped, neither counted
    p, q = pair(cuda)
    a, b = pair(cuda)
    mine, ref = cpab.AdamW([p, q], lr=0.1), cpab.AdamW([a, b], lr=0.1)
    for k in range(3):
        g = torch.ones_like(p) * (k + 1)
        p.grad, a.grad = g, g.clone()
        q.grad = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.ones(1, 4), (6, 4)).to(cuda)
        with pytest.raises(AssertionError, match="sparse"):
            mine.step()
        q.grad, b.grad = torch.ones_like(q), torch.ones_like(b)
        mine.step()
        ref.step()
        assert torch.equal(p, a) and torch.equal(q, b)
    assert [mine.state[t]["step"] for t in (p, q)] == [3, 3]


def test_type_that_is_not_taken(cuda):
    # a float64 parameter has a call of its own, and that one is refused
    p, _ = pair(cuda)
    d = torch.nn.Parameter(torch.randn(7, dtype=torch.float64, device=cuda))
    opt = cpab.AdamW([p, d], lr=0.1)
    for _ in range(3):
        p.grad, d.grad = torch.ones_like(p), torch.ones_like(d)
        with pytest.raises(RuntimeError, match="bfloat16"):
            opt.step()
    assert opt.state[p]["step"] == 3 and opt.state[d]["step"] == 0


def test_state_that_does_not_fit(cuda):
    p, q = pair(cuda)
    opt = cpab.AdamW([p, q], lr=0.1)
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    opt.step()
    before = p.detach().clone()
    kept = opt.state[q]["exp_avg"]
    opt.state[q]["exp_avg"] = kept[:3]
    with pytest.raises(RuntimeError, match="exp_avg of parameter 1"):
        opt.step()
    assert torch.equal(p, before) and [opt.state[t]["step"] for t in (p, q)] == [1, 1]
    opt.state[q]["exp_avg"] = kept
    opt.step()
    assert [opt.state[t]["step"] for t in (p, q)] == [2, 2]
