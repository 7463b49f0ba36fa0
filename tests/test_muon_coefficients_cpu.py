"""Which coefficients mlpsp_orthogonalize refuses: those under which a singular value within [0, 1] leaves [0, 4] in some step, or b s^2 + c s^4
leaves [-32, 32].  Against both polynomials on a fine grid."""
import numpy as np
import pytest

from mlp_splatting_b200 import _lib as L


def accepted(a, b, c, steps):
    return L.load().mlpsp_orthogonalize(None, 0, 0, 4, 4, steps, a, b, c, 1e-7, None, None, None) == 0


def extremes(a, b, c, steps, margin=1.0):
    """The largest |singular value| / 4 and |polynomial| / 32 over all steps, each of whose ranges is widened by `margin`."""
    top, worst = 1.0, 0.0
    for _ in range(steps):
        s = np.linspace(0.0, top, 20001)
        p = b * s ** 2 + c * s ** 4
        y = (a + p) * s
        worst = max(worst, np.abs(y).max() / 4, np.abs(p).max() / 32)
        if worst > 4:
            break
        top = np.abs(y).max() * margin
    return worst


# 10 s - 8 s^3 has its maximum of 4.3 at s^2 = 5/12 and ends at 2: what a tiny c does not change
@pytest.mark.parametrize("c", [0.0, 1e-300, -1e-300, 1e-17, -1e-17, 1e-12, -1e-12, 1e-6, -1e-3])
def test_a_maximum_inside_is_found_whatever_the_last_coefficient(c):
    assert not accepted(10.0, -8.0, c, 1)
    assert accepted(8.0, -6.0, c, 1)          # 3.56


def test_against_a_grid():
    g = np.random.default_rng(0)
    seen = [0, 0]
    for _ in range(4000):
        a, b, c = g.normal(size=3) * (3.0, 6.0, 6.0) * 10.0 ** -g.choice([0, 0, 0, 3, 9, 15], size=3)
        steps = int(g.integers(1, 4))
        # the check widens a step's range by 0.1 %, which the next step multiplies up to 25-fold, (|a| + 3 |b| + 5 |c|) / 4, and the one
        # behind it again: what holds without any margin and fails with twice that one may go either way (and 1e-4 for the grid)
        if extremes(a, b, c, steps) > 1.0001:
            assert not accepted(a, b, c, steps), (a, b, c, steps)
            seen[0] += 1
        elif extremes(a, b, c, steps, 1.002) < 0.9999:
            assert accepted(a, b, c, steps), (a, b, c, steps)
            seen[1] += 1
    assert min(seen) > 300
