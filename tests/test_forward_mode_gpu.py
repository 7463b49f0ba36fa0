"""Inputs on the GPU that carry a forward-mode tangent are refused; under torch.func too."""
import pytest
import torch
from torch.autograd import forward_ad

from mlp_splatting_b200 import muon
from mlp_splatting_b200 import primitive_csr as pc
from tests.test_forward_mode_cpu import calls

pytestmark = pytest.mark.gpu


def test_tangents_are_refused():
    route = pc.route_records(torch.zeros(2, 2, dtype=torch.int32, device="cuda"), 1)
    x, y, w = (torch.ones(s, device="cuda") for s in ((2, 3), (4, 3), (4,)))
    with forward_ad.dual_level():
        duals = [forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, y, w)]
        for call, _name in calls(*duals, route)[:6]:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert torch.equal(pc.dispatch_rows(x, route), torch.ones(4, 3, device="cuda"))      # others go on
    for f in (lambda t: pc.combine_rows(t, route), lambda t: muon.orthogonalize(t)):
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.jvp(f, (y,), (y,))
