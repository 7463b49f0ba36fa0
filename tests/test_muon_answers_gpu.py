"""Calls wait for the device only where a kernel with bounded waits runs: the number of matrices decides, not their size alone."""
import pytest
import torch

from mlp_splatting_b200 import _lib as L
from mlp_splatting_b200 import muon

pytestmark = pytest.mark.gpu
WITHOUT = [(700, 32, 800), (1300, 700, 5), (400, 64, 384), (0, 128, 300)]      # by number; nothing to do


@pytest.mark.parametrize("shape", WITHOUT)
def test_many_matrices_do_not_wait(shape):
    assert L.load().mlpsp_orthogonalize_stack_waits(*shape) == 0 and L.load().mlpsp_orthogonalize_waits(*shape[1:]) == 1
    u = torch.randn(*shape, generator=torch.Generator().manual_seed(1)).cuda()
    w, m = torch.zeros_like(u), torch.zeros_like(u)
    want = muon.orthogonalize(u)
    muon.muon_step(w, u, m, lr=0.1)
    torch.cuda.synchronize()
    stepped = w.clone()
    torch.cuda._sleep(2_000_000_000)      # a second or so; the calls return while it runs
    behind = torch.cuda.Event()
    got = muon.orthogonalize(u)
    w.zero_(), m.zero_()
    muon.muon_step(w, u, m, lr=0.1)
    behind.record()
    assert not behind.query()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(w, stepped)
    # and may be captured with the check they do not need
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = muon.orthogonalize(u)
        muon.muon_step(w, u, m, lr=0.1)
    w.zero_(), m.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(w, stepped)


def test_few_do():
    assert L.load().mlpsp_orthogonalize_stack_waits(2, 32, 800) == 1
    u = torch.randn(2, 32, 800, device="cuda")
    before = torch.cuda.Event()
    torch.cuda._sleep(200_000_000)
    before.record()
    muon.orthogonalize(u)
    assert before.query()
    with pytest.raises(RuntimeError, match="check=False inside a graph capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            muon.muon_step([torch.zeros(700, 32, 800, device="cuda"), u], [torch.zeros(700, 32, 800, device="cuda"), u.clone()],
                           [torch.zeros(700, 32, 800, device="cuda"), u.clone()], lr=0.1)
