"""Tensors made under torch.inference_mode() may not be changed outside it: adamw_step refuses
them before anything moves."""
import pytest
import torch

import cpab

pytestmark = pytest.mark.gpu
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


@pytest.mark.parametrize("which", range(6))
def test_inference_tensors(cuda, which):
    def make(inside, kind=torch.float32, n=40):
        with torch.inference_mode(inside):
            t = torch.ones(n, dtype=torch.uint8 if kind in (E4M3, E8M0) else kind, device=cuda)
            return t.view(kind) if kind in (E4M3, E8M0) else t

    kinds = (torch.float32, E4M3, E4M3, E8M0, E8M0, torch.float32)
    sizes = (40, 40, 40, 2, 2, 40)

    def tensors(inside):
        return [make(inside and k == which, kind, n) for k, (kind, n) in enumerate(zip(kinds, sizes))]

    def step(p, m, v, ms, vs, w):
        cpab.adamw_step([p], [torch.ones(40, device=cuda)], [m], [v], 1, exp_avg_scales=[ms],
                        exp_avg_sq_scales=[vs], masters=[w])

    bad = tensors(True)
    with pytest.raises(RuntimeError, match="inference"):
        step(*bad)
    for t, same in zip(bad, tensors(False)):
        assert torch.equal(t.view(torch.uint8), same.view(torch.uint8))
    with torch.inference_mode():
        step(*bad)
    good = tensors(False)
    step(*good)
    for t, same in zip(bad, good):
        assert torch.equal(t.view(torch.uint8), same.view(torch.uint8))
    # a gradient is only read
    p, m, v = (make(False) for _ in range(3))
    cpab.adamw_step([p], [make(True)], [m], [v], 1)
