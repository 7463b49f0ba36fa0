"""The training operators together, on the records of a rendered image: routing, evaluation, compositing as a weighted sum, its gradients,
weight gradients, and a step on the weights."""
import math
import threading

import numpy as np
import pytest
import torch

from mlp_splatting_b200 import muon
from mlp_splatting_b200 import primitive_csr as pc
from tests.helpers import WKEYS, oracle_frame, small_case

pytestmark = pytest.mark.gpu


def _records(seed):
    from mlp_splatting_b200.cumodel import render_tiles_training_records
    from mlp_splatting_b200.engine import PackedScene, normalize_rows
    scene, cam = small_case(n=600, W=61, H=43, mu=-2.6, seed=seed)
    f = oracle_frame(scene, cam, 5e-3, precision=0)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()      # noqa: E731
    tensors = [t(cam["rays_o"]), t(f["rays_d_unit"]), t(scene["positions"]), t(scene["log_scales"]), normalize_rows(t(scene["quats"])),
               t(f["tile_prims"]), t(f["tile_offsets"]), t(scene["freq"]), t(scene["att"])] + [t(scene[k]) for k in WKEYS]
    packed = PackedScene(scene["positions"], scene["log_scales"], scene["quats"], *[scene[k] for k in WKEYS], scene["freq"], scene["att"],
                         device=torch.device("cuda", 0))
    return tensors, packed, render_tiles_training_records(tensors, 61, 43, 8, 5e-3, 1.5, 2.0)


def test_a_step_from_records_to_weights():
    from mlp_splatting_b200 import muon
    from mlp_splatting_b200 import primitive_csr as pc
    from mlp_splatting_b200.primitive_gemm import grouped_forward, grouped_weight_gradients
    tensors, packed, (rgb, _alpha, ids, x6, raw, masks, _gates, offsets) = _records(3)
    N, R, P = packed.n, int(ids.numel()), 61 * 43
    assert R > 5 * P // 2

    # the route and the grouping sort agree; a pixel's row reaches its records
    route = pc.route_records(ids, N, offsets)
    csr = pc.group_records(ids, x6, raw[:, :4].contiguous(), N, masks)
    assert torch.equal(route.offsets, csr.offsets)
    assert torch.equal(csr.record_indices[route.slots.long()], torch.arange(R, device="cuda"))
    pixel = torch.repeat_interleave(torch.arange(P, device="cuda"), offsets[1:] - offsets[:-1])
    rays = tensors[1]
    at_primitives = pc.dispatch_rows(rays, route)
    assert torch.equal(at_primitives, rays[pixel][csr.record_indices])
    assert torch.equal(at_primitives, csr.x6[:, :3])      # a record's ray direction is its pixel's

    # evaluation at the primitives, colours back to the pixels: the rendered image
    y = grouped_forward(csr.offsets, csr.x6, packed, dtype=torch.float32)
    weights = (raw[:, 4] * raw[:, 5]).contiguous()        # transmittance before the record times its opacity
    image = pc.combine_rows(y[:, :3].contiguous(), route, weights)
    assert float((image - rgb).abs().max()) <= 2e-5       # the FP32 evaluator's tolerance on images

    # gradients of the colours: those of the reverse compositing, which multiplies by the output activation's slope
    g = torch.randn(P, 3, generator=torch.Generator().manual_seed(1)).cuda()
    grad_y, grad_w = pc.combine_rows_gradients(g, y[:, :3].contiguous(), route, weights)
    d4 = pc.primitive_records_reverse(ids, offsets, x6, raw, tensors[3], tensors[4], g, torch.zeros(P, device="cuda"))[0]
    colour = grad_y[route.slots.long()] * raw[:, :3] * (1 - raw[:, :3])
    # three more roundings than grad_y on each side
    assert bool(((colour - d4[:, :3]).abs() <= 8 * 2.0 ** -24 * d4[:, :3].abs() + 1e-12).all())
    terms = g.double()[pixel] * y[:, :3].double()[route.slots.long()]
    assert bool(((grad_w.double() - terms.sum(1)).abs() <= 4 * 2.0 ** -24 * terms.abs().sum(1)).all())      # three products and sums

    # weight gradients of the grouped records, and a step on the primitives that have any
    csr = pc.group_records(ids, x6, d4, N, masks)
    w = tensors[9:15]
    grads = grouped_weight_gradients(csr, tensors[7], tensors[8], w, dtype=torch.float32)
    matrices, updates = [w[0], w[2], w[4]], [grads[0], grads[2], grads[4]]
    momenta = [torch.zeros_like(t) for t in matrices]
    active = csr.offsets[1:] > csr.offsets[:-1]
    assert 0 < int(active.sum()) < N
    before = [t.clone() for t in matrices]
    muon.muon_step(matrices, updates, momenta, lr=0.02, momentum=0.9, active=active)
    for b, t, u, m in zip(before, matrices, updates, momenta):
        assert torch.equal(t[~active], b[~active]) and not bool(m[~active].any())
        direction = u[active] + 0.9 * (m[active] - u[active])
        moved = (b - t)[active].double() / (0.02 * math.sqrt(max(1.0, t.shape[1] / t.shape[2])))
        want = muon.orthogonalize(direction).double()
        # w's rounding over the step, and the direction's
        assert float((moved - want).norm()) <= 2.0 ** -23 / 0.02 * float(b[active].double().norm()) + 1e-4 * float(want.norm())
        seen = direction.flatten(1).norm(dim=1) > 0
        size = torch.linalg.matrix_norm(moved[seen], ord=2)
        assert bool((size < 1.3).all()) and bool((size > 0.3).all())      # singular values towards one


def test_calls_of_two_threads():
    """Each on its own stream, with calls that wait for an answer: neither sees the other's."""
    def work(seed, out):
        g = torch.Generator().manual_seed(seed)
        with torch.cuda.stream(torch.cuda.Stream()):
            for i in range(20):
                first = torch.tensor([0, 900, 2_000, 70_000 + i])
                ids = torch.randint(-1, 700, (70_000 + i,), generator=g, dtype=torch.int32)
                if (seed + i) % 3 == 0:
                    first[1] = 80_000
                u = torch.randn(2, 128, 300, generator=g)
                w, m = torch.randn(5, 64, 400, generator=g).cuda(), torch.zeros(5, 64, 400, device="cuda")
                grads = torch.randn(5, 64, 400, generator=g).cuda()
                try:
                    route = pc.route_records(ids.cuda(), 700, first.cuda())
                    x = torch.randn(3, 65, generator=g).cuda()
                    out.append(pc.combine_rows(pc.dispatch_rows(x, route), route).cpu())
                    out.append(route.slots.cpu())
                except ValueError as e:
                    out.append(str(e))
                out.append(muon.orthogonalize(u.cuda()).cpu())
                muon.muon_step(w, grads, m, lr=0.1)
                out.append(w.cpu())

    want, got = [[], []], [[], []]
    for k in range(2):
        work(k, want[k])
    threads = [threading.Thread(target=work, args=(k, got[k])) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(want[0] + want[1], got[0] + got[1]):
        assert a == b if isinstance(a, str) else torch.equal(a, b)
    assert [len(a) for a in want] == [len(b) for b in got] and any(isinstance(a, str) for a in want[0])
