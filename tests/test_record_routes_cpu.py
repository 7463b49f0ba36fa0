"""Argument errors of the row routes, found on the host."""
import ctypes

import pytest
import torch

from mlp_splatting_b200 import _lib as L
from mlp_splatting_b200 import primitive_csr as pc

FAKE = 0x1000      # never dereferenced: the calls stop at their argument checks


def test_c_entries_check_their_arguments():
    lib = L.load()
    assert lib.mlpsp_dispatch_rows(FAKE, 5, 4, 2, 2, None, FAKE, 4, FAKE, FAKE, None) == -1
    assert b"unknown element type 5" in lib.mlpsp_last_error()
    assert lib.mlpsp_dispatch_rows(FAKE, 0, 0, 2, 2, None, FAKE, 4, FAKE, FAKE, None) == -1
    assert lib.mlpsp_dispatch_rows(FAKE, 0, 65537, 2, 2, None, FAKE, 4, FAKE, FAKE, None) == -4
    assert lib.mlpsp_dispatch_rows(FAKE, 0, 4, 2, 2, None, FAKE, 5, FAKE, FAKE, None) == -1
    assert b"pixels x fan" in lib.mlpsp_last_error()
    assert lib.mlpsp_combine_rows(FAKE, 0, 4, None, 1 << 31, 0, FAKE, FAKE, 4, FAKE, FAKE, None) == -4
    assert lib.mlpsp_combine_rows(FAKE, 0, 4, None, 2, 2, None, None, 4, FAKE, FAKE, None) == -1
    assert b"null pointer" in lib.mlpsp_last_error()
    assert lib.mlpsp_combine_rows_gradients(FAKE, FAKE, 0, 4, None, 2, 2, None, FAKE, 4, FAKE, None, None, None) == -1
    assert lib.mlpsp_combine_rows_gradients(FAKE, None, 0, 4, None, 2, 2, None, FAKE, 4, FAKE, FAKE, FAKE, None) == -1
    def route(ids=FAKE, R=4, n=4, offsets=FAKE, slots=FAKE, nbytes=1 << 20, found=None):
        return lib.mlpsp_route_records(ids, R, n, None, 0, offsets, slots, FAKE, nbytes, found, None)

    assert route(R=1 << 31, nbytes=1 << 40) == -4 and route(n=2 ** 31 - 1) == -4 and route(R=-1) == -1
    assert route(slots=None) == -1 and route(ids=None) == -1 and route(offsets=None) == -1
    assert route(n=600, nbytes=8) == -2 and b"scratch needs" in lib.mlpsp_last_error()
    assert lib.mlpsp_route_records_scratch_bytes(65_536, 511) == 0 and lib.mlpsp_route_records_scratch_bytes(65_537, 511) > 0
    assert route(found=ctypes.byref(ctypes.c_int32())) == -1 and b"no pixel offsets" in lib.mlpsp_last_error()
    assert lib.mlpsp_route_records_scratch_bytes(-1, 3) == -1 and lib.mlpsp_route_records_scratch_bytes(1000, 70_000) > 12_000
    # nothing to do: no launch, no pointer is looked at
    assert lib.mlpsp_dispatch_rows(None, 0, 4, 0, 2, None, None, 0, FAKE, None, None) == 0


def test_there_is_no_cpu_path():
    with pytest.raises(RuntimeError, match="no CPU path"):
        pc.route_records(torch.zeros(3, 2, dtype=torch.int32), 4)
    route = pc.RecordRoute(torch.zeros(2, dtype=torch.int64), torch.zeros(4, dtype=torch.int32), 2, 2)
    with pytest.raises(ValueError, match="one CUDA device"):
        pc.dispatch_rows(torch.zeros(2, 3), route)
