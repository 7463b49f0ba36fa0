"""Orthogonalised updates (muon.orthogonalize, muon.muon_step) against the iteration in 64 bits.

Tolerance of the iteration.  Its error is linear in the unit of the operands: to first order every step adds a multiple of it and
passes on what came before, whatever the arithmetic.  The kernels' operands carry 22 bits and their products are summed in FP32, a
plain FP32 iteration's carry 24, so the kernels may be off by 2^-22 / 2^-24 = 4 times what that one is (in the 2-norm over a stack),
and by eight roundings of the result itself, for stacks so small that FP32 happens to be exact."""
import math

import pytest
import torch

from mlp_splatting_b200 import muon

pytestmark = pytest.mark.gpu
DTYPES = (torch.float32, torch.float16, torch.bfloat16)
SMALL = [(1, 1, 1), (3, 1, 7), (5, 2, 3), (17, 3, 5), (33, 4, 32), (70, 5, 9), (7, 16, 72), (9, 17, 18), (40, 32, 72), (11, 32, 32),
         (3, 72, 32), (3, 31, 95), (2, 32, 96), (5, 8, 48), (6, 96, 12), (2000, 4, 32), (2, 30, 42)]
MIDDLE = [(3, 33, 33), (3, 64, 72), (5, 64, 64), (2, 40, 96), (3, 72, 64), (3, 49, 61), (4, 96, 48), (2, 64, 50), (3, 57, 81), (700, 64, 72),
          (2, 33, 256), (3, 200, 40), (400, 64, 270), (2, 41, 512), (3, 12, 97), (5, 1, 512), (2, 32, 500), (300, 31, 520), (900, 5, 700)]
LARGE = [(3, 33, 133), (2, 64, 72), (3, 64, 64), (5, 4, 128), (2, 128, 128), (1, 128, 1152), (2, 512, 128), (1, 100, 300), (1, 2048, 128),
         (1, 128, 2048), (1, 1, 2048), (3, 65, 70), (2, 33, 97), (1, 97, 33), (3, 128, 129), (3, 50, 260), (400, 64, 64), (1, 6, 1030)]


def stack(n, r, c, seed, dtype=torch.float32, scale=1e-3):
    g = torch.Generator().manual_seed(seed)
    u = torch.randn(n, r, c, generator=g) + 1.5 * torch.randn(n, r, 1, generator=g) * torch.randn(n, 1, c, generator=g)
    return (scale * u).to(dtype)


def iteration(u, steps=5, coefficients=muon.COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = u.mT if u.shape[1] > u.shape[2] else u
    x = x / torch.linalg.vector_norm(x, dim=(1, 2), keepdim=True).clamp(min=eps)
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if u.shape[1] > u.shape[2] else x


def allowed(u, **how):
    """(the 64-bit result, the 2-norm by which the kernels' may differ before rounding to a narrower type)"""
    want = iteration(u.double(), **how)
    plain = iteration(u.float(), **how).double()
    return want, 4 * float((plain - want).norm()) + 8 * 2.0 ** -22 * float(want.norm())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,r,c", SMALL + MIDDLE + LARGE)
def test_iteration(n, r, c, dtype):
    u = stack(n, r, c, seed=n + r + c, dtype=dtype)
    want, tol = allowed(u)
    out = muon.orthogonalize(u.cuda())
    assert out.dtype == dtype and out.shape == u.shape
    if dtype != torch.float32:      # one rounding at the end, binary16 below its normal range included
        tol += torch.finfo(dtype).eps / 2 * float(want.norm()) + 2.0 ** -25 * math.sqrt(want.numel())
    assert float((out.cpu().double() - want).norm()) <= tol
    again = muon.orthogonalize(u.cuda())
    assert torch.equal(again, out)
    one = muon.orthogonalize(u[0].cuda())
    assert one.shape == (r, c)
    if min(r, c) > 64 or max(r, c) <= 256:      # other shapes go to another kernel when there are many
        assert torch.equal(one, out[0])
    want, tol = allowed(u[:1])
    if dtype != torch.float32:
        tol += torch.finfo(dtype).eps / 2 * float(want.norm()) + 2.0 ** -25 * math.sqrt(want.numel())
    assert float((one.cpu().double() - want[0]).norm()) <= tol


# more matrices than the GPU takes at once, at the borders between the kernels and between their splits of a matrix
MANY = [(1300, 5, 700), (1200, 16, 1000), (1200, 16, 1024), (320, 1030, 16), (700, 32, 800), (700, 32, 801), (400, 64, 384), (300, 64, 385), (250, 40, 300),
        (60, 128, 700), (40, 97, 1500), (20, 128, 2048), (150, 128, 256), (160, 128, 257), (3, 128, 256), (3, 70, 144), (2, 1300, 90)]


@pytest.mark.parametrize("n,r,c", MANY)
def test_many_long_matrices(n, r, c):
    u = stack(n, r, c, seed=n + r + c)
    want, tol = allowed(u)
    out = muon.orthogonalize(u.cuda())
    assert float((out.cpu().double() - want).norm()) <= tol
    # an inactive matrix and its neighbours
    active = torch.arange(n) % 5 != 2
    w, m = stack(n, r, c, seed=1).cuda(), torch.zeros(n, r, c, device="cuda")
    before = w.clone()
    muon.muon_step(w, u.cuda(), m, lr=1.0, momentum=0.0, active=active.cuda())
    assert torch.equal(w[~active], before[~active]) and not m[~active].any()
    # w - scale X, with an FP32 rounding of the product and of the difference each
    scale = math.sqrt(max(1.0, r / c))
    step = before.cpu().double() - scale * want
    tol = scale * tol + 2.0 ** -23 * (float(before.double().norm()) + 2 * scale * float(want.norm()))
    assert float((w.cpu().double() - step)[active].norm()) <= tol


@pytest.mark.parametrize("how", [dict(steps=1), dict(steps=12), dict(coefficients=(1.5, -0.5, 0.0), steps=9),
                                 dict(coefficients=(1.875, -1.25, 0.375), steps=7), dict(eps=1.0, steps=3)])
@pytest.mark.parametrize("n,r,c", [(9, 32, 72), (5, 4, 32), (3, 64, 72), (1, 128, 300)])
def test_steps_and_coefficients(n, r, c, how):
    u = stack(n, r, c, seed=3)
    want, tol = allowed(u, **how)
    assert float((muon.orthogonalize(u.cuda(), **how).cpu().double() - want).norm()) <= tol


@pytest.mark.parametrize("n,r,c", [(9, 32, 72), (6, 4, 32), (3, 64, 72), (1, 128, 300)])
def test_low_rank_updates(n, r, c):
    """Few records: gradients of rank two and rank one.  What rounding puts into the empty directions grows 485-fold."""
    g = torch.Generator().manual_seed(8)
    for rank in (1, 2):
        u = torch.randn(n, r, rank, generator=g) @ torch.randn(n, rank, c, generator=g)
        want, tol = allowed(u)
        assert float((muon.orthogonalize(u.cuda()).cpu().double() - want).norm()) <= tol


@pytest.mark.parametrize("n,r,c", [(13, 4, 32), (9, 32, 72), (5, 64, 64), (3, 128, 300), (9, 7, 5)])
def test_extreme_matrices_stay_apart(n, r, c):
    """Zeros, an infinity, a NaN, values whose squares overflow or underflow, next to ordinary matrices."""
    u = stack(n, r, c, seed=4)
    plain = muon.orthogonalize(u.cuda())
    v = u.clone()
    v[0] = 0.0
    v[1, r // 2, c // 2] = float("inf")
    v[2, 0, c - 1] = float("nan")
    got = muon.orthogonalize(v.cuda())
    assert not bool(got[0].any()) and bool(got[1].isnan().all()) and bool(got[2].isnan().all())
    assert torch.equal(got[3:], plain[3:])
    for scale in (2.0 ** 100, 2.0 ** 60, 2.0 ** -10):      # 2^-10 with the entries of 1e-3 keeps the norm above eps
        v = u.clone()
        v[1] *= scale
        got = muon.orthogonalize(v.cuda())
        want, tol = allowed(u[1:2])
        assert float((got[1:2].cpu().double() - want).norm()) <= tol
        assert torch.equal(got[0], plain[0]) and torch.equal(got[2:], plain[2:])
    tiny = u[1:2] * 2.0 ** -90      # the norm is far below eps: X0 = U / eps, and every step multiplies it by a
    want = iteration(tiny.double())
    assert float((muon.orthogonalize(tiny.cuda()).cpu().double() - want).norm()) <= 16 * 2.0 ** -24 * float(want.norm())
    many = u * torch.exp(torch.arange(n) * 2.0 - 8.0)[:, None, None]
    want, tol = allowed(many)
    assert float((muon.orthogonalize(many.cuda()).cpu().double() - want).norm()) <= tol


@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("n,r,c", [(5, 32, 72), (5, 4, 32), (2, 64, 72), (1, 128, 300)])
def test_any_alignment_and_in_place(n, r, c, shift):
    u = stack(n, r, c, seed=6)
    want = muon.orthogonalize(u.cuda())
    for dtype in (torch.float32, torch.bfloat16):
        flat = torch.zeros(n * r * c + 8, dtype=dtype, device="cuda")
        view = flat[shift:shift + n * r * c].view(n, r, c)
        view.copy_(u)
        expected = want if dtype == torch.float32 else muon.orthogonalize(view.clone())
        assert muon.orthogonalize(view, out=view) is view
        assert torch.equal(view, expected)
        assert not bool(flat[:shift].any()) and not bool(flat[shift + n * r * c:].any())      # neighbours as they were


STEP_SHAPES = [(50, 32, 72), (50, 32, 32), (50, 4, 32), (50, 64, 72), (50, 7, 5), (50, 40, 33)]


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masked", [False, True])
def test_steps_of_a_stack(dtype, masked, nesterov):
    """Two steps on a list of stacks.  Momentum: one fused operation on a difference, 2 * 2^-24 of |g| + |m|.  Weights: three
    roundings of 2^-24, and lr times the tolerance of the iteration, which the second step takes of its own momentum."""
    g = torch.Generator().manual_seed(9)
    active = (torch.rand(50, generator=g) < 0.6) if masked else None
    w = [torch.randn(s, generator=g) for s in STEP_SHAPES]
    m = [torch.zeros(s) for s in STEP_SHAPES]
    wd, md = [t.cuda() for t in w], [t.cuda() for t in m]
    on = torch.ones(50, dtype=torch.bool) if active is None else active
    for step in range(2):
        grads = [stack(*s, seed=step * 10 + i, dtype=dtype) for i, s in enumerate(STEP_SHAPES)]
        grads[0][3] = 0.0
        gd = [t.cuda() for t in grads]
        if masked:
            for t in gd:
                t[~active.cuda()] = float("nan")      # gradients of inactive primitives are not read
        before = [t.cpu() for t in wd]
        old = [t.cpu() for t in md]
        muon.muon_step(wd, gd, md, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1,
                       active=None if active is None else active.cuda())
        for i, (r, c) in enumerate(s[1:] for s in STEP_SHAPES):
            gi, mi = grads[i].double(), old[i].double()
            new = mi + (1 - 0.9) * (gi - mi)
            got_m = md[i].cpu()
            assert bool(((got_m.double() - new).abs() <= 4 * 2.0 ** -24 * (gi.abs() + mi.abs()))[on].all())
            u = gi + 0.9 * (got_m.double() - gi) if nesterov else got_m.double()
            want, tol = allowed(u[on].float())      # rounding u to FP32 is one unit more, well within the four
            want = before[i].double()[on] * (1 - 0.02 * 0.1) - 0.02 * math.sqrt(max(1.0, r / c)) * want
            off = (wd[i].cpu().double()[on] - want).norm()
            assert float(off) <= 3 * 2.0 ** -24 * float(want.norm()) + 0.02 * math.sqrt(max(1.0, r / c)) * tol
            assert torch.equal(wd[i].cpu()[~on], before[i][~on]) and torch.equal(got_m[~on], old[i][~on])


def test_step_of_the_decoder_layers():
    """Single matrices, one tensor instead of a list, and no weight decay."""
    g = torch.Generator().manual_seed(2)
    for shape in ((128, 128), (128, 1152), (512, 128), (16, 40)):
        w, grad = torch.randn(shape, generator=g), stack(1, *shape, seed=1)[0]
        wd, md = w.cuda(), torch.zeros(shape, device="cuda")
        muon.muon_step(wd, grad.cuda(), md, lr=0.5, momentum=0.0)
        assert torch.equal(md.cpu(), grad)
        want, tol = allowed(grad[None])
        scale = 0.5 * math.sqrt(max(1.0, shape[0] / shape[1]))
        want = w.double() - scale * want[0]
        assert float((wd.cpu().double() - want).norm()) <= 3 * 2.0 ** -24 * float(want.norm()) + scale * tol


def test_nothing_active_and_nothing_at_all():
    w, m = torch.ones(6, 32, 72, device="cuda"), torch.ones(6, 32, 72, device="cuda")
    muon.muon_step(w, torch.full_like(w, float("nan")), m, lr=1.0, active=torch.zeros(6, dtype=torch.bool, device="cuda"))
    assert bool((w == 1).all()) and bool((m == 1).all())
    assert muon.orthogonalize(torch.zeros(0, 32, 72, device="cuda")).shape == (0, 32, 72)
    muon.muon_step(torch.zeros(0, 64, 72, device="cuda"), torch.zeros(0, 64, 72, device="cuda"), torch.zeros(0, 64, 72, device="cuda"), lr=1.0)


def test_what_was_packed_from_old_weights_is_packed_anew():
    """In-place steps count as such: the renderer's packed scene, and autograd's check of saved tensors."""
    from mlp_splatting_b200.cumodel import NeuralPrimitiveSceneTileCUDA
    model = NeuralPrimitiveSceneTileCUDA(num_primitives=20).cuda()
    packed = model.packed_scene()
    assert model.packed_scene() is packed
    layers = [model.W1, model.W2, model.W3]
    momenta = [torch.zeros_like(w) for w in layers]
    saved = (model.W2 * model.W2).sum()
    muon.muon_step(layers, [torch.randn_like(w) for w in layers], momenta, lr=0.1)
    again = model.packed_scene()
    assert again is not packed and torch.equal(again.W1, model.W1.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
    out = torch.zeros(3, 4, device="cuda")
    version = out._version
    muon.orthogonalize(torch.ones(3, 4, device="cuda"), out=out)
    assert out._version > version


def test_other_streams_and_replayed_graphs():
    """A step captured on small and large matrices and replayed on new gradients; two graphs over the same tensors."""
    shapes = [(20, 32, 72), (3, 64, 64), (1, 128, 300)]
    w = [torch.zeros(s, device="cuda") for s in shapes]
    m = [torch.zeros(s, device="cuda") for s in shapes]
    g = [stack(*s, seed=1).cuda() for s in shapes]
    start = [stack(*s, seed=2, scale=1.0).cuda() for s in shapes]

    def step():
        muon.muon_step(w, g, m, lr=0.1, weight_decay=0.01, check=False)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for graph in graphs:
        with torch.cuda.graph(graph):
            step()

    def run(calls):
        for t, s in zip(w, start):
            t.copy_(s)
        for t in m:
            t.zero_()
        for i, call in enumerate(calls):
            for t, s in zip(g, shapes):
                t.copy_(stack(*s, seed=20 + i))
            call()
        torch.cuda.synchronize()
        return [t.clone() for t in w + m]

    for a, b in zip(run([step, step, step]), run([graphs[0].replay, graphs[1].replay, graphs[0].replay])):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="check=False inside a graph capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            muon.orthogonalize(w[2])


def test_refusals():
    u = torch.ones(4, 32, 72, device="cuda")
    half, flags = u.half(), torch.ones(4, dtype=torch.bool, device="cuda")
    cases = [
        (lambda: muon.orthogonalize(u[0, 0]), "a matrix"),
        (lambda: muon.orthogonalize(torch.ones(129, 129, device="cuda")), "shorter side"),
        (lambda: muon.orthogonalize(torch.ones(8, 2049, device="cuda")), "shorter side"),
        (lambda: muon.orthogonalize(torch.ones(0, 8, device="cuda")), "shorter side"),
        (lambda: muon.orthogonalize(u.double()), "float32, float16 or bfloat16"),
        (lambda: muon.orthogonalize(u.mT), "contiguous"),
        (lambda: muon.orthogonalize(u.cpu()), "one CUDA device"),
        (lambda: muon.orthogonalize(u, out=half), "shape and type"),
        (lambda: muon.orthogonalize(u[:2], out=u[1:3]), "lie apart"),
        (lambda: muon.orthogonalize(u, steps=0), "steps"),
        (lambda: muon.orthogonalize(u, steps=True), "steps"),
        (lambda: muon.orthogonalize(u, eps=0.0), "eps"),
        (lambda: muon.muon_step(u, u, u.clone(), lr=0.1, momentum=1.0), "momentum"),
        (lambda: muon.muon_step(u, u.clone(), u.clone(), lr=float("nan")), "lr"),
        (lambda: muon.muon_step(u, u.clone(), u, lr=0.1), "overlap"),
        (lambda: muon.muon_step([u, u], [u.clone()] * 2, [u.clone(), u.clone()], lr=0.1), "overlap"),
        (lambda: muon.muon_step(half, half, half.clone(), lr=0.1), "FP32"),
        (lambda: muon.muon_step(u, u[:3], u.clone(), lr=0.1), "one shape"),
        (lambda: muon.muon_step([u], [u, u], [u.clone()], lr=0.1), "as many"),
        (lambda: muon.muon_step([], [], [], lr=0.1), "at least one"),
        (lambda: muon.muon_step(u, u.clone(), u.clone(), lr=0.1, active=flags[:3]), "active"),
        (lambda: muon.muon_step(u[0], u[1], u[2], lr=0.1, active=flags), "active"),
        (lambda: muon.muon_step(u, u.clone(), u.clone(), lr=0.1, active=flags.int()), "active"),
    ]
    for call, text in cases:
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(RuntimeError, match="singular values leave"):
        muon.orthogonalize(u, coefficients=(5.0, 1.0, 1.0))
    assert bool((u == 1).all())


@pytest.mark.parametrize("n,r,c", [(932_100, 32, 72), (4_200_000, 16, 32), (524_400, 64, 64), (131_200, 128, 128)])
def test_stacks_beyond_32_bits(n, r, c):
    """More than 2^31 elements: the last matrices come out as they do alone, in place."""
    u = torch.empty(n, r, c, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(n))
    assert u.numel() > 2 ** 31
    tail, head = u[-8:].clone(), u[:8].clone()
    assert muon.orthogonalize(u, out=u) is u
    assert torch.equal(u[-8:], muon.orthogonalize(tail)) and torch.equal(u[:8], muon.orthogonalize(head))


def test_a_step_beyond_32_bits():
    n, r, c = 932_100, 32, 72
    g = torch.empty(n, r, c, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(3))
    w, m = torch.ones(n, r, c, device="cuda"), torch.zeros(n, r, c, device="cuda")
    last = [t[-5:].clone() for t in (w, g, m)]
    muon.muon_step(w, g, m, lr=0.1)
    muon.muon_step(*last, lr=0.1)
    assert torch.equal(w[-5:], last[0]) and torch.equal(m[-5:], last[2])
