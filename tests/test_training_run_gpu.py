"""The training operators one behind the other as a step uses them: records -> route_records -> dispatch_rows -> grouped_forward ->
combine_rows -> loss -> combine_rows_gradients -> grouped_weight_gradients -> muon_step, and dispatch_rows_gradient of a loss on the
dispatched rows.  Every call takes what the one before it gave."""
import math

import numpy as np
import pytest
import torch

from mlp_splatting_b200 import muon
from mlp_splatting_b200 import primitive_csr as pc
from tests.helpers import WKEYS, oracle_frame, small_case

pytestmark = pytest.mark.gpu


def test_records_to_weights():
    from mlp_splatting_b200.cumodel import render_tiles_training_records
    from mlp_splatting_b200.engine import PackedScene, normalize_rows
    from mlp_splatting_b200.primitive_gemm import grouped_forward, grouped_weight_gradients
    from oracle import oracle as orc
    W, H = 53, 39
    scene, cam = small_case(n=500, W=W, H=H, mu=-2.6, seed=5)
    f = oracle_frame(scene, cam, 5e-3, precision=0)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()      # noqa: E731
    weights = [t(scene[k]) for k in WKEYS]
    freq, att, rays = t(scene["freq"]), t(scene["att"]), t(f["rays_d_unit"])
    rgb, _alpha, ids, x6, raw, masks, _gates, offsets = render_tiles_training_records(
        [t(cam["rays_o"]), rays, t(scene["positions"]), t(scene["log_scales"]), normalize_rows(t(scene["quats"])), t(f["tile_prims"]),
         t(f["tile_offsets"]), freq, att, *weights], W, H, 8, 5e-3, 1.5, 2.0)
    N, R, P = 500, int(ids.numel()), W * H

    def packed(w):
        return PackedScene(scene["positions"], scene["log_scales"], scene["quats"], *w, scene["freq"], scene["att"], device=torch.device("cuda", 0))

    route = pc.route_records(ids, N, offsets)
    order = torch.empty(R, dtype=torch.int64, device="cuda")
    order[route.slots.long()] = torch.arange(R, device="cuda")
    rows = torch.cat([pc.dispatch_rows(rays, route), x6[order, 3:]], dim=1)        # a record's ray is its pixel's, the rest its own
    assert torch.equal(rows, x6[order])
    share = raw[:, 4] * raw[:, 5]                # of a record in its pixel: transmittance before it times its opacity, kept fixed here
    goal = torch.rand(P, 3, generator=torch.Generator().manual_seed(2)).cuda()

    def colours(scene_of):
        y = grouped_forward(route.offsets, rows, scene_of, dtype=torch.float32)[:, :3].contiguous()
        return y, pc.combine_rows(y, route, share)

    def loss(image):
        return 0.5 * float((image - goal).double().square().sum())

    y, image = colours(packed(weights))
    assert float((image - rgb).abs().max()) <= 2e-5        # the FP32 evaluator's tolerance on images
    grad_y, grad_share = pc.combine_rows_gradients(image - goal, y, route, share)
    pixel = torch.repeat_interleave(torch.arange(P, device="cuda"), offsets[1:] - offsets[:-1])
    terms = (image - goal).double()[pixel] * y.double()[route.slots.long()]
    assert bool(((grad_share.double() - terms.sum(1)).abs() <= 4 * 2.0 ** -24 * terms.abs().sum(1)).all())

    # through the sigmoid of the colours; the densities, whose share is kept, get no gradient
    d4 = torch.cat([grad_y * y * (1 - y), torch.zeros(R, 1, device="cuda")], dim=1).contiguous()
    csr = pc.PrimitiveCSR(route.offsets, order, rows, d4, masks[order].contiguous())
    grads = grouped_weight_gradients(csr, freq, att, weights, dtype=torch.float32)
    cpu = lambda a: a.detach().cpu().numpy()      # noqa: E731
    model = orc.grouped_weight_gradients_model(cpu(csr.offsets), cpu(rows), cpu(d4), cpu(csr.relu_masks), cpu(freq), cpu(att), [cpu(w) for w in weights],
                                               dtype="float32")
    for got, want in zip(grads, model):      # some 300 sums and products of 2^-24 each, cancellation of the sums by about five
        assert float(np.linalg.norm(cpu(got) - want)) <= 1e-4 * float(np.linalg.norm(want))
    # against differences along the gradient of the last layer, in which the loss is smooth: the slope is the gradient's square; the third
    # derivative adds some h^2, and the images' roundings, 1e-7 of 6,000 values of one, divided by 2 h
    direction, h = grads[4] / grads[4].abs().max(), 1e-2
    ends = [loss(colours(packed([*weights[:4], weights[4] + s * h * direction, weights[5]]))[1]) for s in (1, -1)]
    slope = float((grads[4].double() * direction.double()).sum())
    assert abs((ends[0] - ends[1]) / (2 * h) - slope) <= 1e-2 * slope

    # the step: its direction is a descent direction
    matrices, updates = [weights[0], weights[2], weights[4]], [grads[0], grads[2], grads[4]]
    momenta = [torch.zeros_like(w) for w in matrices]
    seen = route.offsets[1:] != route.offsets[:-1]
    before = [w.clone() for w in matrices]
    muon.muon_step(matrices, updates, momenta, lr=1e-3, active=seen)
    for b, w, u in zip(before, matrices, updates):
        assert torch.equal(w[~seen], b[~seen]) and float(((w - b).double() * u.double()).sum()) < 0
        moved = (b - w)[seen] / (1e-3 * math.sqrt(max(1.0, w.shape[1] / w.shape[2])))
        # the weights' rounding over the step
        want = muon.orthogonalize(u[seen].contiguous())      # the first step's update is the gradient times a number
        assert float((moved - want).double().norm()) <= 2.0 ** -23 / 1e-3 * float(b[seen].double().norm()) + 1e-4 * float(want.double().norm())

    # a loss on the dispatched rows: its gradient comes back to the pixels
    at_primitives = pc.dispatch_rows(rays, route)
    back = pc.dispatch_rows_gradient(at_primitives, route)
    count = (offsets[1:] - offsets[:-1])[:, None]
    assert bool(((back.double() - count * rays.double()).abs() <= count * 2.0 ** -24 * count * rays.double().abs()).all())
