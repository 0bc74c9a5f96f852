"""A Muon step of more matrices than one launch takes, in tiles, on one workspace: each is
what it is alone, and the formula's."""
import pytest
import torch

import cpab
from test_gpu_muon import compare, make

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("dtype,masters", [(F32, False), (BF16, True)])
def test_against_the_formula(cuda, dtype, masters):
    # tiles of up to 64, 128 and 256, 40 to a launch
    compare(cuda, dtype, [(70, 70), (66, 130), (130, 66)] * 30, masters=masters, seed=21)
    compare(cuda, dtype, [(300, 300)] * 41 + [(60, 60)] * 41, masters=masters, seed=22)


def test_large_tiles_against_each_alone(cuda):
    shapes = [(1030, 1040)] * 42
    all_, alone = (make(cuda, BF16, shapes, seed=23, masters=True) for _ in range(2))
    before = [t.double() for t in alone["masters"]]
    cpab.muon_step(all_["params"], all_["grads"], all_["momenta"], masters=all_["masters"])
    for k in (0, 1, 39, 40, 41):
        cpab.muon_step(*(alone[n][k:k + 1] for n in ("params", "grads", "momenta")), masters=alone["masters"][k:k + 1])
        # the tiles go by how many there are: a product's sums in another order, within the
        # step's own bound of the move on each side, and the masters' roundings
        a, b = all_["masters"][k].double(), alone["masters"][k].double()
        assert float((a - b).norm()) <= 2e-5 * float((b - before[k]).norm()) + 2.0 ** -22 * float(b.norm())
        assert torch.equal(all_["momenta"][k], alone["momenta"][k])
    assert all(torch.equal(p, m.to(BF16)) for p, m in zip(all_["params"], all_["masters"]))
