"""Rows of pixels to primitives and back (primitive_csr.route_records, dispatch_rows, combine_rows and their gradients)
against plain 64-bit statements."""
import pytest
import torch

from mlp_splatting_b200 import primitive_csr as pc

pytestmark = pytest.mark.gpu
DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def ids_of(T, N, fan, seed, drop=0.1):
    g = torch.Generator().manual_seed(seed)
    if fan:
        ids = torch.randint(0, max(N, 1), (T, fan), generator=g)
        lists = None
        R = T * fan
    else:
        counts = torch.randint(0, 12, (T,), generator=g) * (torch.rand(T, generator=g) < 0.8)
        lists = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(counts, 0)])
        R = int(lists[-1])
        ids = torch.randint(0, max(N, 1), (R,), generator=g)
    gone = torch.rand(ids.shape, generator=g) < drop
    ids = torch.where(gone, torch.where(torch.rand(ids.shape, generator=g) < 0.5, -1, N + 3), ids)
    if N == 0:
        ids = torch.full_like(ids, -1)
    return ids, lists


def plain_route(ids, N):
    key = torch.where((ids < 0) | (ids >= N), N, ids).reshape(-1)
    order = torch.sort(key, stable=True)[1]
    slots = torch.empty(key.numel(), dtype=torch.int64)
    slots[order] = torch.arange(key.numel())
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(torch.bincount(key, minlength=N + 1)[:N], 0)])
    return offsets, slots


def pixel_of(T, fan, lists, R):
    if fan:
        return torch.arange(R) // fan
    return torch.bucketize(torch.arange(R), lists[1:], right=True)


def make(T, N, fan, seed, drop=0.1):
    ids, lists = ids_of(T, N, fan, seed, drop)
    route = pc.route_records(ids.to(torch.int32).cuda(), N, None if lists is None else lists.cuda())
    offsets, slots = plain_route(ids, N)
    return route, offsets, slots, pixel_of(T, fan, lists, ids.numel()), int(offsets[-1])


SHAPES = [(1, 1, 1), (1, 64, 8), (7, 3, 2), (257, 5, 4), (4099, 256, 2), (1000, 70_000, 3), (3001, 300, 0), (64, 1, 0), (5, 0, 2)]


@pytest.mark.parametrize("T,N,fan", SHAPES + [(40_000, 100_000, 0), (300, 17_000_000, 4)])
@pytest.mark.parametrize("wide", [False, True])
def test_route_is_a_stable_grouping(T, N, fan, wide):
    ids, lists = ids_of(T, N, fan, seed=T + N)
    ids = ids.to(torch.int64 if wide else torch.int32)
    if wide and ids.numel():
        ids.view(-1)[0] = 2 ** 32      # out of range, not primitive 0
    route = pc.route_records(ids.cuda(), N, None if lists is None else lists.cuda())
    offsets, slots = plain_route(ids.to(torch.int64), N)
    assert torch.equal(route.offsets.cpu(), offsets) and torch.equal(route.slots.cpu().long(), slots)
    assert route.pixels == T and route.fan == fan and route.records == ids.numel()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [1, 3, 4, 6, 7, 8, 33, 96, 513, 2056])
@pytest.mark.parametrize("T,N,fan", [(1, 64, 8), (257, 5, 4), (401, 300, 0)])
def test_rows_there_and_back(T, N, fan, D, dtype):
    """dispatch copies exactly; a sum of K products in FP32 is off by at most K steps of 2^-24 times the sum of the
    magnitudes (weights and rows enter exactly), plus half a step of the output's type."""
    route, offsets, slots, pix, kept = make(T, N, fan, seed=D)
    g = torch.Generator().manual_seed(D)
    R, half = slots.numel(), torch.finfo(dtype).eps / 2
    x, y = torch.randn(T, D, generator=g).to(dtype), torch.randn(R, D, generator=g).to(dtype)
    w, dout = torch.rand(R, generator=g), torch.randn(T, D, generator=g).to(dtype)
    want = torch.zeros(R, D, dtype=dtype)
    want[slots] = x[pix]
    want[kept:] = 0
    assert torch.equal(pc.dispatch_rows(x.cuda(), route).cpu(), want)
    y_dev = y.clone()
    y_dev[kept:] = float("nan")      # rows of dropped records are never read
    live = (slots < kept).double()[:, None]
    rows = y.double()[slots] * live
    longest = int(torch.bincount(pix, minlength=T).max()) if R else 0

    def close(got, terms):
        sums = torch.zeros(T, D, dtype=torch.float64).index_add_(0, pix, terms)
        size = torch.zeros(T, D, dtype=torch.float64).index_add_(0, pix, terms.abs())
        tol = longest * 2.0 ** -24 * size
        tol = tol + half * (sums.abs() + tol) + 2.0 ** -25      # binary16 below its normal range: half of 2^-24
        assert got.dtype == dtype and bool(((got.cpu().double() - sums).abs() <= tol).all())

    close(pc.combine_rows(y_dev.cuda(), route, w.cuda()), w.double()[:, None] * rows)
    close(pc.combine_rows(y_dev.cuda(), route), rows)
    close(pc.dispatch_rows_gradient(y_dev.cuda(), route), rows)
    shape = (T, fan) if fan else (R,)
    dy, dw = pc.combine_rows_gradients(dout.cuda(), y_dev.cuda(), route, w.view(shape).cuda())
    want_y = torch.zeros(R, D, dtype=torch.float64)
    want_y[slots] = w.double()[:, None] * dout.double()[pix] * live
    tol_y = (half + 2.0 ** -24) * 1.01 * want_y.abs() + 2.0 ** -25
    assert dy.dtype == dtype and bool(((dy.cpu().double() - want_y).abs() <= tol_y).all()) and not bool(dy[kept:].any())
    products = rows * dout.double()[pix]
    tol_w = (D + 5) * 2.0 ** -24 * products.abs().sum(1) + 1e-30
    assert dw.shape == shape and bool(((dw.cpu().double().view(-1) - products.sum(1)).abs() <= tol_w).all())
    assert pc.combine_rows_gradients(dout.cuda(), y_dev.cuda(), route)[1] is None


@pytest.mark.parametrize("T,N,fan,D,dtype", [(30_000, 300, 0, D, t) for D in (6, 13, 33) for t in DTYPES]
                         + [(4_000, 70, 3, D, t) for D in (130, 513) for t in DTYPES]
                         + [(45_000, 300, 0, 128, torch.float32), (20_000, 9, 4, 260, torch.float16), (9_000, 400, 0, 256, torch.bfloat16)])
def test_many_rows_there_and_back(T, N, fan, D, dtype):
    """Enough of them for the kernels' other shapes: threads with two pieces, narrow groups, y beyond the L2."""
    test_rows_there_and_back(T, N, fan, D, dtype)


@pytest.mark.parametrize("fan", [3, 0])
def test_autograd_is_the_gradient(fan):
    """Through autograd, with an expanded gradient, against the same program in 64 bits; and against differences."""
    T, N, D = 97, 20, 5
    route, offsets, slots, pix, kept = make(T, N, fan, seed=5)
    g = torch.Generator().manual_seed(1)
    R = slots.numel()
    x, w = torch.randn(T, D, generator=g), torch.rand(R, generator=g)
    scale = torch.randn(R, D, generator=g)

    def plain(x, w):
        rows = torch.zeros(R, D, dtype=torch.float64).index_copy(0, slots, x[pix])
        rows = rows * (torch.arange(R) < kept)[:, None] * scale.double()
        rows = rows * rows
        return torch.zeros(T, D, dtype=torch.float64).index_add(0, pix, w[:, None] * rows[slots])

    xd, wd = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    rows = pc.dispatch_rows(xd, route) * scale.cuda()
    out = pc.combine_rows(rows * rows, route, wd)
    gx, gw = torch.autograd.grad(out.sum(), (xd, wd))
    x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
    total = plain(x64, w64).sum()
    ex, ew = torch.autograd.grad(total, (x64, w64))
    # a dozen roundings of 2^-24 on each of at most twelve terms per pixel, five per record
    assert bool(((gx.cpu().double() - ex).abs() <= 24 * 2.0 ** -24 * (ex.abs() + 40.0)).all())
    assert bool(((gw.cpu().double() - ew).abs() <= 24 * 2.0 ** -24 * (ew.abs() + 1e-3)).all())
    with torch.no_grad():
        dx, dw, h = torch.randn(T, D, generator=g).double(), torch.randn(R, generator=g).double(), 1e-6
        slope = (plain(x64 + h * dx, w64 + h * dw).sum() - plain(x64 - h * dx, w64 - h * dw).sum()) / (2 * h)
        along = (gx.cpu().double() * dx).sum() + (gw.cpu().double() * dw).sum()
        assert abs(float(slope - along)) <= 1e-4 * float((gx.cpu().double() * dx).abs().sum() + (gw.cpu().double() * dw).abs().sum())
    only = pc.combine_rows(torch.ones(R, D, device="cuda"), route, wd)
    assert torch.autograd.grad(only.sum(), wd)[0].shape == wd.shape
    late = pc.dispatch_rows(xd, route).sum()
    route.slots.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(late, xd)


def test_long_and_empty_lists():
    """A pixel of 100,000 records between empty ones; all records dropped; no records; no pixels."""
    first = torch.tensor([0, 0, 100_000, 100_000])
    ids = torch.arange(100_000, dtype=torch.int32) % 7
    route = pc.route_records(ids.cuda(), 7, first.cuda())
    y = torch.ones(100_000, 3, device="cuda")
    assert torch.equal(pc.combine_rows(y, route).cpu(), torch.tensor([[0.0] * 3, [1e5] * 3, [0.0] * 3]))
    gone = pc.route_records(torch.full((4, 2), -1, dtype=torch.int32, device="cuda"), 9)
    assert int(gone.offsets[-1]) == 0 and gone.slots.tolist() == list(range(8))
    assert not bool(pc.combine_rows(torch.full((8, 5), float("inf"), device="cuda"), gone).any())
    assert not bool(pc.dispatch_rows(torch.full((4, 5), float("inf"), device="cuda"), gone).any())
    dy, dw = pc.combine_rows_gradients(torch.full((4, 5), float("nan"), device="cuda"), torch.zeros(8, 5, device="cuda"), gone,
                                       torch.ones(4, 2, device="cuda"))
    assert not bool(dy.any()) and not bool(dw.any())
    none = pc.route_records(torch.zeros(0, dtype=torch.int32, device="cuda"), 3, torch.zeros(5, dtype=torch.int64, device="cuda"))
    assert none.offsets.tolist() == [0] * 4
    assert pc.dispatch_rows(torch.ones(4, 2, device="cuda"), none).shape == (0, 2)
    assert not bool(pc.combine_rows(torch.ones(0, 2, device="cuda"), none).any())
    empty = pc.route_records(torch.zeros(0, 4, dtype=torch.int32, device="cuda"), 3)
    assert pc.combine_rows(torch.ones(0, 2, device="cuda"), empty, torch.ones(0, 4, device="cuda")).shape == (0, 2)


def test_unaligned_rows_and_other_streams():
    """Rows that start off a 16-byte boundary, on a stream that is not the current default, twice with the same bits."""
    route, offsets, slots, pix, kept = make(500, 40, 0, seed=2)
    R = slots.numel()
    base = torch.randn(R * 8 + 3, generator=torch.Generator().manual_seed(0)).cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    results = []
    with torch.cuda.stream(stream):
        for shift in (0, 1, 2):
            y = base[shift:shift + R * 8].view(R, 8)
            results.append([pc.combine_rows(y, route).cpu() for _ in range(2)])
            assert torch.equal(*results[-1])
            want = torch.zeros(500, 8, dtype=torch.float64)
            want.index_add_(0, pix, y.cpu().double()[slots] * (slots < kept)[:, None])
            torch.testing.assert_close(results[-1][0].double(), want, rtol=1e-5, atol=1e-5)


def test_captured_and_replayed():
    """Routing, both ways and the gradients in one graph, replayed on new inputs."""
    T, N, D = 300, 50, 12
    ids = torch.zeros(T, 2, dtype=torch.int32, device="cuda")
    x, w, dout = torch.zeros(T, D, device="cuda"), torch.zeros(T, 2, device="cuda"), torch.zeros(T, D, device="cuda")

    def step():
        route = pc.route_records(ids, N)
        rows = pc.dispatch_rows(x, route)
        return route.slots, rows, pc.combine_rows(rows, route, w), *pc.combine_rows_gradients(dout, rows, route, w)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (1, 2):
        torch.manual_seed(seed)
        ids.copy_(torch.randint(-1, N, (T, 2)))
        for t in (x, w, dout):
            t.copy_(torch.randn(t.shape))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, step()):
            assert torch.equal(got, want)
    first = torch.arange(0, 2 * T + 1, 2, device="cuda")
    with pytest.raises(RuntimeError, match="check=False inside a graph capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            pc.route_records(ids.view(-1), N, first)


def test_refusals():
    route, *_ = make(10, 4, 2, seed=1)
    x = torch.ones(10, 4, device="cuda")
    y = torch.ones(20, 4, device="cuda")
    for bad in ([1, 2, 3], [0, 2, 1, 3], [0, 1, 2]):
        with pytest.raises(ValueError, match="start at zero, end at the record count and be monotone"):
            pc.route_records(torch.zeros(3, dtype=torch.int32, device="cuda"), 4, torch.tensor(bad, device="cuda"))
    cases = [
        (lambda: pc.dispatch_rows(x.t(), route), "contiguous"),
        (lambda: pc.dispatch_rows(x.cpu(), route), "one CUDA device"),
        (lambda: pc.dispatch_rows(x.double(), route), "float32, float16 or bfloat16"),
        (lambda: pc.dispatch_rows(y, route), "must have shape"),
        (lambda: pc.dispatch_rows(torch.ones(10, 0, device="cuda"), route), "must have shape"),
        (lambda: pc.combine_rows(x, route), "must have shape"),
        (lambda: pc.combine_rows(y, route, torch.ones(19, device="cuda")), "one for every record"),
        (lambda: pc.combine_rows(y, route, torch.ones(20, device="cuda").half()), "one for every record"),
        (lambda: pc.combine_rows_gradients(x.half(), y, route), "one element type"),
        (lambda: pc.combine_rows(y, pc.RecordRoute(route.offsets, route.slots, 9, 2)), "pixels x fan"),
        (lambda: pc.combine_rows(y, pc.RecordRoute(route.offsets, route.slots.long(), 10, 2)), "slots must be int32"),
        (lambda: pc.combine_rows(y, pc.RecordRoute(route.offsets, route.slots, 10, 0, torch.zeros(3, dtype=torch.int64, device="cuda"))),
         "one entry more than pixels"),
        (lambda: pc.route_records(torch.zeros(3, dtype=torch.int32, device="cuda"), 4), "with pixel_offsets"),
        (lambda: pc.route_records(torch.zeros(3, 1, device="cuda"), 4), "int32 or int64"),
        (lambda: pc.route_records(torch.zeros(3, 1, dtype=torch.int32, device="cuda"), -1), "below 2\\^31"),
    ]
    for call, text in cases:
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(TypeError, match="RecordRoute"):
        pc.dispatch_rows(x, (route.offsets, route.slots))


def test_wrong_routes_stay_inside_their_tensors():
    """Slots and offsets that no call of route_records gives (bounds are checked in the kernels): defined where the rules
    hold, nothing outside the outputs is touched."""
    slots = torch.tensor([5, -1, 2, 99, 0, 1], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 4], device="cuda")
    first = torch.tensor([-3, 2, 1, 50], device="cuda")
    route = pc.RecordRoute(offsets, slots, 3, 0, first)
    y = torch.arange(12.0, device="cuda").view(6, 2)
    guard = torch.full((6 + 2, 2), 7.0, device="cuda")
    out = pc.combine_rows(y, route)
    assert out.shape == (3, 2) and torch.equal(out[0], torch.zeros(2, device="cuda"))
    rows = pc.dispatch_rows(torch.ones(3, 2, device="cuda"), route)
    assert rows.shape == (6, 2) and not bool(rows[5].any())
    pc.combine_rows_gradients(torch.ones(3, 2, device="cuda"), y, route, torch.ones(6, device="cuda"))
    torch.cuda.synchronize()
    assert bool((guard == 7.0).all())


@pytest.mark.parametrize("N", [1, 2, 510, 511, 512, 600, 262_143, 262_144])
@pytest.mark.parametrize("R", [1, 31, 4096, 4097, 65_536, 65_537, 300_001])
def test_route_at_the_borders_of_its_passes(N, R):
    ids = torch.randint(-1, N + 1, (R, 1), generator=torch.Generator().manual_seed(N + R))
    route = pc.route_records(ids.to(torch.int32).cuda(), N)
    offsets, slots = plain_route(ids, N)
    assert torch.equal(route.offsets.cpu(), offsets) and torch.equal(route.slots.cpu().long(), slots)


@pytest.mark.parametrize("R", [1, 5000, 70_000])
def test_no_primitives_at_all(R):
    route = pc.route_records(torch.zeros(R, 1, dtype=torch.int32, device="cuda"), 0)
    assert route.offsets.tolist() == [0] and torch.equal(route.slots.cpu().long(), torch.arange(R))
    x = torch.ones(R, 3, device="cuda")
    assert not pc.dispatch_rows(x, route).any() and not pc.combine_rows(x * float("nan"), route).any()


def test_rows_beyond_32_bits():
    """2^31 elements and more on both sides; a permutation of rows and its way back."""
    T, D, N = 33_000, 65_536, 500
    ids = torch.randint(0, N, (T, 1), generator=torch.Generator().manual_seed(1), dtype=torch.int32).cuda()
    route = pc.route_records(ids, N)
    x = torch.empty(T, D, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(2))
    assert x.numel() > 2 ** 31
    rows = pc.dispatch_rows(x, route)
    slots = route.slots.long()
    for at in (0, T // 2, T - 2, T - 1):
        assert torch.equal(rows[slots[at]], x[at])
    back = pc.combine_rows(rows, route)
    assert torch.equal(back, x)
    del back
    two = torch.full((T, 1), 2.0, device="cuda")
    grad, grad_w = pc.combine_rows_gradients(x, rows, route, two)
    assert torch.equal(grad[slots[T - 1]], 2 * x[T - 1]) and torch.equal(grad[slots[0]], 2 * x[0])
    # <x, x> of 65,536 squares, each sum of products off by at most 2^-24 of the terms so far per step, in at most 2^12 steps
    for at in (0, T - 1):
        assert abs(float(grad_w[at, 0]) - float(x[at].double().square().sum())) <= 2.0 ** -12 * D * 2
