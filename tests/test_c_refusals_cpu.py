"""Arguments with which the C entries of the training operators would leave the arrays: refused before any launch."""
import pytest

from mlp_splatting_b200 import _lib as L
from mlp_splatting_b200 import muon

FAKE = 0x1000      # never dereferenced: the calls stop at their argument checks
NS = (5, *muon.COEFFICIENTS, 1e-7)


def step(*sizes, active=FAKE):
    tensors = (L.MuonTensor * len(sizes))(*((FAKE, FAKE, FAKE, n, 32, 72, 1.0, 0, 0) for n in sizes))
    return L.load().mlpsp_muon_step(tensors, len(sizes), active, 0.1, 0.9, 1, 0.0, *NS, None, None)


@pytest.mark.parametrize("sizes", [(3, 4), (4, 3), (3, 0), (5, 5, 6)])
def test_one_mask_for_stacks_of_one_length(sizes):
    assert step(*sizes) == -1 and b"as many matrices" in L.load().mlpsp_last_error()


def test_a_mask_of_nothing():
    assert step(0, 0) == 0
