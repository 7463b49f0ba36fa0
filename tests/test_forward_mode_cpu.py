"""Operators without a forward-mode derivative refuse inputs that carry a tangent: nothing is found on the device."""
import pytest
import torch
from torch.autograd import forward_ad

from mlp_splatting_b200 import muon
from mlp_splatting_b200 import primitive_csr as pc


def calls(x, y, w, route):
    return [(lambda: pc.dispatch_rows(x, route), "dispatch_rows"), (lambda: pc.dispatch_rows_gradient(y, route), "dispatch_rows_gradient"),
            (lambda: pc.combine_rows(y, route), "combine_rows"), (lambda: pc.combine_rows(y.detach(), route, w), "combine_rows"),
            (lambda: pc.combine_rows_gradients(x, y, route), "combine_rows_gradients"),
            (lambda: muon.orthogonalize(y), "orthogonalize"), (lambda: muon.orthogonalize(torch.ones(4, 3), out=y), "orthogonalize"),
            (lambda: muon.muon_step(torch.ones(4, 3), y, torch.ones(4, 3), lr=0.1), "muon_step")]


def test_tangents_are_refused():
    route = pc.RecordRoute(torch.zeros(2, dtype=torch.int64), torch.zeros(4, dtype=torch.int32), 2, 2)
    with forward_ad.dual_level():
        x, y, w = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (torch.ones(2, 3), torch.ones(4, 3), torch.ones(4)))
        for call, name in calls(x, y, w, route):
            with pytest.raises(NotImplementedError, match=f"^{name} has no forward-mode derivative"):
                call()
        for call, _name in calls(torch.ones(2, 3), torch.ones(4, 3), torch.ones(4), route):      # no tangent: what is wrong is the device
            with pytest.raises(ValueError, match="one CUDA device"):
                call()
