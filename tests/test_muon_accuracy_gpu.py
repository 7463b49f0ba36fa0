"""How near the Newton-Schulz kernels are to 64-bit arithmetic: nearer than the iteration in plain FP32, which is what keeping diagonals apart
in FP32 and adding long sums panel by panel is for.  Without either the error is several times as large (4e-6 of the result for 128 rows).

Bound: the plain iteration's error on the same Gaussian matrices times 1.2, since that error is itself a sample.  It depends on how a CPU orders its
sums, and over a few single matrices it scatters by about a tenth."""
import pytest
import torch

from mlp_splatting_b200 import muon
from tests.test_muon_gpu import iteration

pytestmark = pytest.mark.gpu


# warp (tiles of 16 and of 32 rows, long rows), pair (short and long rows), cluster (one CTA, several, long rows of few)
@pytest.mark.parametrize("n,r,c", [(400, 4, 32), (200, 16, 72), (200, 32, 72), (1200, 16, 1000), (700, 32, 800), (100, 64, 72), (400, 64, 384),
                                   (8, 128, 256), (6, 128, 1152), (4, 128, 2048), (6, 1152, 128), (8, 40, 1500), (60, 128, 700)])
def test_nearer_than_plain_fp32(n, r, c):
    u = torch.randn(n, r, c, generator=torch.Generator().manual_seed(n + r + c))
    want = iteration(u.double())
    plain = float((iteration(u).double() - want).norm() / want.norm())
    got = float((muon.orthogonalize(u.cuda()).cpu().double() - want).norm() / want.norm())
    print(f"{n} x {r} x {c}: {got:.2e}, plain FP32 {plain:.2e}")
    assert got <= 1.2 * plain
