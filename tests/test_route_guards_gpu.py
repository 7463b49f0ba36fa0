"""What the row kernels write: with slots that no route has (kernels check every one against the records), nothing beside the outputs, and of the
outputs exactly the rows that the slots name.  Through the C entries, with outputs in the middle of larger arrays."""
import pytest
import torch

from mlp_splatting_b200 import _lib as L

pytestmark = pytest.mark.gpu
TYPES = {torch.float32: L.PRECISION_F32, torch.float16: L.PRECISION_F16, torch.bfloat16: L.PRECISION_BF16}
MARK, MARGIN = 7.0, 4096


class Inside:
    """`shape` elements in the middle of MARKs, `shift` elements off the start's alignment."""

    def __init__(self, shape, dtype, shift):
        self.n = torch.Size(shape).numel()
        self.flat = torch.full((self.n + 2 * MARGIN,), MARK, dtype=dtype, device="cuda")
        self.first = MARGIN + shift
        self.view = self.flat[self.first:self.first + self.n].view(shape)

    def margins(self):
        return bool((self.flat[:self.first] == MARK).all()) and bool((self.flat[self.first + self.n:] == MARK).all())


def lists(fan, T, kind):
    if fan:
        return None, T * fan, torch.arange(T * fan) // fan
    counts = torch.arange(T) * 7 % 5
    first = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
    return first, int(first[-1]), torch.repeat_interleave(torch.arange(T), counts)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D", [1, 2, 6, 8, 33, 64, 264, 2056])
@pytest.mark.parametrize("fan", [3, 0])
@pytest.mark.parametrize("shift", [0, 1])
def test_rows_of_wrong_slots(dtype, D, fan, shift):
    lib, T = L.load(), 301 if D < 256 else 40
    stream = torch.cuda.current_stream().cuda_stream
    g = torch.Generator().manual_seed(D)
    first, R, pixel = lists(fan, T, 0)
    kept = R - R // 5
    slots = torch.randperm(R, generator=g).to(torch.int32)
    bad = torch.rand(R, generator=g) < 0.3
    wrong = torch.tensor([-1, R, R + 1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    slots[bad] = wrong[torch.randint(0, 5, (int(bad.sum()),), generator=g)]
    lives = ~bad & (slots < kept)
    x, dout = (torch.randn(T, D, generator=g).to(dtype) for _ in range(2))
    y, w = torch.randn(R, D, generator=g).to(dtype), torch.rand(R, generator=g)
    xd, dd, yd, wd, sd = x.cuda(), dout.cuda(), y.cuda(), w.cuda(), slots.cuda()
    kd, fd = torch.tensor([kept], device="cuda"), None if first is None else first.cuda()
    where = (T, fan, L.ptr(fd), sd.data_ptr(), R, kd.data_ptr())
    out, back, dy = Inside((R, D), dtype, shift), Inside((T, D), dtype, shift), Inside((R, D), dtype, shift)
    dw = Inside((R,), torch.float32, shift)
    assert lib.mlpsp_dispatch_rows(xd.data_ptr(), TYPES[dtype], D, *where, out.view.data_ptr(), stream) == 0
    assert lib.mlpsp_combine_rows(yd.data_ptr(), TYPES[dtype], D, wd.data_ptr(), *where, back.view.data_ptr(), stream) == 0
    assert lib.mlpsp_combine_rows_gradients(dd.data_ptr(), yd.data_ptr(), TYPES[dtype], D, wd.data_ptr(), *where, dy.view.data_ptr(),
                                            dw.view.data_ptr(), stream) == 0
    torch.cuda.synchronize()
    assert out.margins() and back.margins() and dy.margins() and dw.margins()
    named = slots[~bad].long()
    want = torch.full((R, D), MARK, dtype=dtype)      # rows that no slot names stay as they were
    want[named] = torch.where(lives[~bad][:, None], x[pixel[~bad]], torch.zeros((), dtype=dtype))
    assert torch.equal(out.view.cpu(), want)
    # tolerances as in test_record_routes_gpu.py: a rounding of 2^-24 per product and sum, half a step of the output's type
    half = torch.finfo(dtype).eps / 2
    grads = torch.full((R, D), MARK, dtype=torch.float64)
    grads[named] = w.double()[~bad][:, None] * dout.double()[pixel[~bad]] * lives[~bad][:, None]
    assert bool(((dy.view.cpu().double() - grads).abs() <= (half + 2.0 ** -24) * 1.01 * grads.abs() + 2.0 ** -25).all())
    rows = y.double()[slots.long().clamp(0, R - 1)] * lives[:, None]
    sums = torch.zeros(T, D, dtype=torch.float64).index_add_(0, pixel, w.double()[:, None] * rows)
    size = torch.zeros(T, D, dtype=torch.float64).index_add_(0, pixel, w.double()[:, None] * rows.abs())
    tol = 5 * 2.0 ** -24 * size
    assert bool(((back.view.cpu().double() - sums).abs() <= tol + half * (sums.abs() + tol) + 2.0 ** -25).all())
    terms = rows * dout.double()[pixel]
    assert bool(((dw.view.cpu().double() - terms.sum(1)).abs() <= (D + 5) * 2.0 ** -24 * terms.abs().sum(1)).all())


@pytest.mark.parametrize("D", [2, 8, 66])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_wrong_offsets_stay_inside(D, dtype):
    """Offsets that descend, start below zero and end behind the records, which no call has checked."""
    lib, T, R = L.load(), 700, 1500
    stream = torch.cuda.current_stream().cuda_stream
    g = torch.Generator().manual_seed(D)
    first = torch.randint(-2000, 4000, (T + 1,), generator=g)
    first[:4] = torch.tensor([-2 ** 62, 2 ** 62, -5, 2 ** 40])
    first, slots = first.cuda(), torch.randperm(R, generator=g).to(torch.int32).cuda()
    kept = torch.tensor([2 ** 50], device="cuda")      # beyond the records, too
    x, y, w = torch.ones(T, D, dtype=dtype, device="cuda"), torch.ones(R, D, dtype=dtype, device="cuda"), torch.ones(R, device="cuda")
    where = (T, 0, first.data_ptr(), slots.data_ptr(), R, kept.data_ptr())
    out, back, dy = Inside((R, D), dtype, 0), Inside((T, D), dtype, 0), Inside((R, D), dtype, 0)
    dw = Inside((R,), torch.float32, 0)
    assert lib.mlpsp_dispatch_rows(x.data_ptr(), TYPES[dtype], D, *where, out.view.data_ptr(), stream) == 0
    assert lib.mlpsp_combine_rows(y.data_ptr(), TYPES[dtype], D, None, *where, back.view.data_ptr(), stream) == 0
    assert lib.mlpsp_combine_rows_gradients(x.data_ptr(), y.data_ptr(), TYPES[dtype], D, w.data_ptr(), *where, dy.view.data_ptr(), dw.view.data_ptr(),
                                            stream) == 0
    torch.cuda.synchronize()
    for t in (out, back, dy, dw):
        assert t.margins()
    ones = (out.view == 1) | (out.view == MARK)
    assert bool(ones.all()) and bool(((dy.view == 1) | (dy.view == MARK)).all()) and bool(((dw.view == D) | (dw.view == MARK)).all())


@pytest.mark.parametrize("dtype", list(TYPES))
def test_gradient_of_a_weight_on_a_long_row(dtype):
    """65,536 products: a warp's lanes add 2,048 each, one behind the other, and then five times two sums."""
    from mlp_splatting_b200 import primitive_csr as pc
    T, D = 9, 65_536
    g = torch.Generator().manual_seed(4)
    route = pc.route_records(torch.randint(0, 5, (T, 2), generator=g, dtype=torch.int32).cuda(), 5)
    x, dout = torch.randn(2 * T, D, generator=g).to(dtype), torch.randn(T, D, generator=g).to(dtype)
    _, dw = pc.combine_rows_gradients(dout.cuda(), x.cuda(), route, torch.ones(T, 2, device="cuda"))
    terms = x.double()[route.slots.cpu().long()] * dout.double().repeat_interleave(2, 0)
    assert bool(((dw.cpu().double().view(-1) - terms.sum(1)).abs() <= (2048 + 5) * 2.0 ** -24 * terms.abs().sum(1)).all())
