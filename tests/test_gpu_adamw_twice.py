"""adamw_step refuses a tensor that comes twice; the optimiser steps a parameter that a group
holds twice in turn, as torch's does."""
import pytest
import torch

import cpab

pytestmark = pytest.mark.gpu


def test_refusals(cuda):
    p, q, g, m, n, v, w = (torch.zeros(8, device=cuda) for _ in range(7))
    for lists in (([p, p], [m, n], [v, w]), ([p, q], [m, m], [v, w]), ([p, q], [m, n], [v, v]),
                  ([p, q], [m, n], [m, w]), ([p, q], [p, n], [v, w]), ([p, p.view(2, 4)], [m, n.view(2, 4)],
                                                                      [v, w.view(2, 4)])):
        grads = [g.view(t.shape) for t in lists[0]]
        with pytest.raises(RuntimeError, match="twice"):
            cpab.adamw_step(lists[0], grads, lists[1], lists[2], 1)
    assert all((t == 0).all() for t in (p, q, m, n, v, w))
    # one gradient for two parameters is read twice, and empty ones share their place
    e = torch.zeros(0, device=cuda)
    cpab.adamw_step([p, q, e, e], [g + 1, g + 1, e, e], [m, n, e, e], [v, w, e, e], 1)
    cpab.adamw_step([p, q], [g, g], [m, n], [v, w], 2)
    assert torch.equal(p, q) and (p < 0).all()


@pytest.mark.filterwarnings("ignore:optimizer contains a parameter group with duplicate parameters")
def test_a_group_with_a_parameter_twice(cuda):
    start = torch.randn(33, generator=torch.Generator().manual_seed(0)).to(cuda)
    a, b = (torch.nn.Parameter(start.clone()) for _ in range(2))
    mine = cpab.AdamW([a, a], lr=1e-2)
    ref = cpab.AdamW([b], lr=1e-2)
    for _ in range(3):
        a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
        mine.step()
        ref.step()
        ref.step()
    assert torch.equal(a, b)
