"""Argument errors of the orthogonalised updates, found on the host."""
import pytest
import torch

from mlp_splatting_b200 import _lib as L
from mlp_splatting_b200 import muon

FAKE = 0x1000      # never dereferenced: the calls stop at their argument checks
NS = (5, *muon.COEFFICIENTS, 1e-7)


def test_c_entries_check_their_arguments():
    lib = L.load()

    def ortho(update=FAKE, dtype=0, n=1, rows=32, cols=72, ns=NS, out=FAKE):
        return lib.mlpsp_orthogonalize(update, dtype, n, rows, cols, *ns, out, None, None)

    assert ortho(dtype=3) == -1 and b"element type 3" in lib.mlpsp_last_error()
    assert ortho(rows=129, cols=129) == -4 and ortho(cols=2049) == -4 and ortho(rows=0) == -1 and ortho(n=-1) == -1
    assert ortho(ns=(0, *NS[1:])) == -1 and ortho(ns=(33, *NS[1:])) == -1
    assert ortho(ns=(*NS[:4], 0.0)) == -1 and ortho(ns=(*NS[:4], float("nan"))) == -1
    for bad in ((5.0, 1.0, 1.0), (float("nan"), 0.0, 0.0), (float("inf"), 0.0, 0.0), (1.0, 40.0, 0.0), (4.1, 0.0, 0.0)):
        assert ortho(ns=(5, *bad, 1e-7)) == -1 and b"singular values leave" in lib.mlpsp_last_error()
    assert ortho(update=None) == -1 and ortho(out=None) == -1 and b"null pointer" in lib.mlpsp_last_error()
    assert ortho(n=0, update=None, out=None) == 0      # nothing to do: no launch

    def step(w=FAKE, g=FAKE, m=FAKE, lr=0.1, mu=0.9, wd=0.0, scale=1.0, rows=32):
        good = L.MuonTensor(None, None, None, 0, 32, 72, 1.0, 0, 0)      # nothing in it
        tensors = (L.MuonTensor * 2)(good, L.MuonTensor(w, g, m, 1, rows, 72, scale, 0, 0))
        return lib.mlpsp_muon_step(tensors, 2, None, lr, mu, 1, wd, *NS, None, None)

    assert step(rows=0) == -1
    assert lib.mlpsp_muon_step(None, 1, None, 0.1, 0.9, 1, 0.0, *NS, None, None) == -1
    assert lib.mlpsp_muon_step(None, 0, None, 0.1, 0.9, 1, 0.0, *NS, None, None) == 0
    assert step(w=None) == -1 and step(g=None) == -1 and step(m=None) == -1
    assert step(mu=1.0) == -1 and step(mu=-0.1) == -1 and step(lr=-1.0) == -1 and step(lr=float("inf")) == -1
    assert step(wd=float("nan")) == -1 and step(scale=0.0) == -1
    assert [lib.mlpsp_orthogonalize_waits(*s) for s in ((32, 512), (512, 1), (256, 64), (65, 65), (4, 513), (33, 257))] == [0, 0, 0, 1, 1, 1]


def test_there_is_no_cpu_path():
    with pytest.raises(ValueError, match="one CUDA device"):
        muon.orthogonalize(torch.ones(4, 4))
    with pytest.raises(ValueError, match="one CUDA device"):
        muon.muon_step(torch.ones(4, 4), torch.ones(4, 4), torch.ones(4, 4), lr=0.1)
