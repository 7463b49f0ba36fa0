"""What combine_rows keeps for its backward pass, and the pass in a captured graph."""
import pytest
import torch

from mlp_splatting_b200 import primitive_csr as pc

pytestmark = pytest.mark.gpu


def make(T=50, fan=3, N=9, D=5):
    g = torch.Generator().manual_seed(1)
    route = pc.route_records(torch.randint(-1, N, (T, fan), generator=g, dtype=torch.int32).cuda(), N)
    return (route, *(torch.randn(s, generator=g).cuda() for s in ((T, D), (T * fan, D), (T, fan))))


def test_only_what_the_gradients_read_is_kept():
    """The gradient of y reads the weights, that of the weights reads y: writing over the other one later is no error, and it is not kept alive."""
    route, dout, y, w = make()
    want_y, want_w = pc.combine_rows_gradients(dout, y, route, w)
    ones_y, _ = pc.combine_rows_gradients(dout, y, route)

    def kept(out):
        saved = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: (saved.append(t.data_ptr()), t)[1], lambda t: t):
            out()
        return saved

    yg, wg = y.clone().requires_grad_(), w.clone().requires_grad_()
    assert yg.data_ptr() not in kept(lambda: pc.combine_rows(yg, route, w)) and wg.data_ptr() not in kept(lambda: pc.combine_rows(y, route, wg))
    for weights, want in ((w.clone(), want_y), (None, ones_y)):
        rows = y.clone().requires_grad_()
        out = pc.combine_rows(rows, route, weights)
        with torch.no_grad():
            rows.mul_(2.0)
        assert torch.equal(torch.autograd.grad(out, rows, dout)[0], want)
    rows, weights = y.clone(), w.clone().requires_grad_()
    out = pc.combine_rows(rows, route, weights)
    with torch.no_grad():
        weights.zero_()
    assert torch.equal(torch.autograd.grad(out, weights, dout)[0], want_w)
    # what is read may not change
    for a, b, change in ((y.clone().requires_grad_(), w.clone(), 1), (y.clone(), w.clone().requires_grad_(), 0),
                         (y.clone().requires_grad_(), w.clone().requires_grad_(), 0), (y.clone().requires_grad_(), w.clone().requires_grad_(), 1)):
        out = pc.combine_rows(a, route, b)
        with torch.no_grad():
            (a, b)[change].mul_(2.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out, [t for t in (a, b) if t.requires_grad], dout)


def test_backward_in_a_graph():
    """Forward and backward pass captured together, replayed on new inputs."""
    route, dout, y, w = make()
    yg, wg = y.clone().requires_grad_(), w.clone().requires_grad_()
    xg = torch.randn(50, 5, device="cuda", requires_grad=True)

    def step():
        rows = pc.dispatch_rows(xg, route) * yg
        return torch.autograd.grad(pc.combine_rows(rows, route, wg), (xg, yg, wg), dout)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (3, 4):
        g = torch.Generator("cuda").manual_seed(seed)
        with torch.no_grad():
            for t in (xg, yg, wg, dout):
                t.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_the_capture_that_counts_is_that_of_the_ids_device(monkeypatch):
    """With ids on another device than the current one it is that device's stream that may be capturing."""
    entered, asked, real = [], [], torch.cuda.is_current_stream_capturing

    class On(pc._on):
        __slots__ = ()

        def __enter__(self):
            entered.append(self.d)
            return super().__enter__()

        def __exit__(self, *exc):
            entered.pop()
            return super().__exit__(*exc)

    monkeypatch.setattr(pc, "_on", On)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: (asked.append(list(entered)), real())[1])
    ids = torch.zeros(6, dtype=torch.int32, device="cuda")
    pc.route_records(ids, 2, torch.tensor([0, 2, 6], device="cuda"))
    assert asked == [[ids.device]]
