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


def misaligned(call, **sizes):
    """Every pointer of a call in turn one byte off (sizes: the bytes of its elements); all others as they are."""
    for name, size in sizes.items():
        for off in {1, size // 2}:
            assert call(**{name: FAKE + off}) == -1 and b"aligned" in L.load().mlpsp_last_error(), (name, off)


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_pointers_off_their_elements(dtype):
    lib, size = L.load(), 4 if dtype == 0 else 2

    def dispatch(x=FAKE, first=FAKE, slots=FAKE, kept=FAKE, out=FAKE):
        return lib.mlpsp_dispatch_rows(x, dtype, 4, 2, 0, first, slots, 4, kept, out, None)

    def combine(y=FAKE, weights=FAKE, first=FAKE, slots=FAKE, kept=FAKE, out=FAKE):
        return lib.mlpsp_combine_rows(y, dtype, 4, weights, 2, 0, first, slots, 4, kept, out, None)

    def gradients(dout=FAKE, y=FAKE, weights=FAKE, first=FAKE, slots=FAKE, kept=FAKE, dy=FAKE, dw=FAKE):
        return lib.mlpsp_combine_rows_gradients(dout, y, dtype, 4, weights, 2, 0, first, slots, 4, kept, dy, dw, None)

    misaligned(dispatch, x=size, first=8, slots=4, kept=8, out=size)
    misaligned(combine, y=size, weights=4, first=8, slots=4, kept=8, out=size)
    misaligned(gradients, dout=size, y=size, weights=4, first=8, slots=4, kept=8, dy=size, dw=4)

    def ortho(update=FAKE, out=FAKE):
        return lib.mlpsp_orthogonalize(update, dtype, 1, 32, 72, *NS, out, None, None)

    def one_step(w=FAKE, g=FAKE, m=FAKE):
        return lib.mlpsp_muon_step((L.MuonTensor * 1)((w, g, m, 1, 32, 72, 1.0, dtype, 0)), 1, None, 0.1, 0.9, 1, 0.0, *NS, None, None)

    misaligned(ortho, update=size, out=size)
    misaligned(one_step, w=4, g=size, m=4)


def test_routes_off_their_elements():
    def route(ids=FAKE, first=FAKE, offsets=FAKE, slots=FAKE, scratch=FAKE):
        return L.load().mlpsp_route_records(ids, 4, 600, first, 2, offsets, slots, scratch, 1 << 20, None, None)

    misaligned(route, ids=4, first=8, offsets=8, slots=4, scratch=4)


def test_which_stacks_wait():
    """The cluster kernel's: by size, or by size and number (of 148 SMs, where no device answers)."""
    waits = L.load().mlpsp_orthogonalize_stack_waits
    assert [waits(*s) for s in ((1, 32, 800), (4000, 32, 800), (4000, 32, 801), (1, 64, 384), (4000, 64, 384), (4000, 384, 65))] == [1, 0, 1, 1, 0, 1]
    assert [waits(*s) for s in ((0, 128, 128), (-1, 128, 128), (1, 0, 4), (1, 129, 129), (1, 4, 2049), (1, 32, 512), (1, 256, 64))] == [0] * 7
