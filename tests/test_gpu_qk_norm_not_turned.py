"""Norms of heads of which nothing turns, in a program that has the samples' places in hand:
no frequencies and no positions, or frequencies of no values with them."""
import os
import sys

import pytest
import torch

import cpab
import heads_oracle as ho

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
sys.path.append(os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(__file__))), "perf"))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [1, 16, 33])
@pytest.mark.parametrize("neighbours", [False, True])
def test_frequencies_of_no_values(cuda, dtype, D, neighbours):
    gen = torch.Generator().manual_seed(D)
    args = [torch.randn(2, 9, n, D, generator=gen).to(cuda, dtype) for n in (3, 2)]
    args += [(1 + 0.1 * torch.randn(D, generator=gen)).to(cuda, dtype) for _ in range(2)]
    none = torch.zeros(0, device=cuda)
    ups = [torch.randn(t.shape, generator=gen).to(cuda, dtype) for t in args[:2]]

    def passes(*turn):
        leaves = [t.detach().requires_grad_() for t in args]
        out = cpab.qk_norm(*leaves, *turn, neighbours=neighbours)
        return (*out, *torch.autograd.grad(out, leaves, ups))
    want = passes()
    for at in (None, torch.arange(9, device=cuda), torch.arange(18, device=cuda).view(2, 9) + (1 << 40),
               torch.full((2, 1), float("nan"), device=cuda)):
        assert all(torch.equal(a, b) for a, b in zip(passes(none, at), want))


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_case_of_the_benchmark(cuda, train, dtype):
    # as they are drawn: places are in hand, whatever turns
    import more_operators as cases
    assert not cases.own
    for turned in (0, 8):
        case = cases._qk(dtype, 2, 7, 4, 2, 17, turned, train, given=True)
        state = cases.prepare(case, 3)
        assert "positions" in state
        cases.own = True
        try:
            got = cases.run(state)
        finally:
            cases.own = False
        want = cases.exact(case, 3)
        assert set(got) == set(want)
        for name, w in want.items():
            # a result's rounding, and in 32 bits 60 units of a row's and 14 rows' sums
            off = float((ho.f64(got[name]) - w.cpu()).norm()) / float(w.norm())
            assert off <= ho.UNIT[got[name].dtype] + 74 * ho.U, (turned, name, off)
