"""Device-side waits that give up in the Newton-Schulz kernel (a product that is left unanswered on request, so that its wait runs out
after a second): the call says so, and nothing that was not computed looks like a result."""
import pytest
import torch

from mlp_splatting_b200 import _lib as L
from mlp_splatting_b200 import muon

pytestmark = pytest.mark.gpu


@pytest.fixture
def withhold():
    lib = L.load()

    def set_to(product):
        assert lib.mlpsp_test_withhold_answer(product) == 0

    yield set_to
    set_to(0)


def update(*shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(sum(shape))).to(dtype).cuda()


# a cluster of three, a matrix in one CTA, eight matrices to a tile in a cluster of eight; the first step's products, a middle one, the last step's
@pytest.mark.parametrize("shape,dtype,product", [((3, 128, 300), torch.float32, 1), ((3, 128, 300), torch.bfloat16, 6), ((3, 128, 300), torch.float32, 13),
                                                 ((2, 100, 70), torch.float32, 3), ((2, 70, 100), torch.float16, 15), ((11, 16, 1100), torch.float32, 8)])
def test_a_wait_that_gives_up_leaves_nan(withhold, shape, dtype, product):
    u = update(*shape, dtype=dtype)
    want = muon.orthogonalize(u)
    withhold(product)
    out = muon.orthogonalize(u, out=torch.full_like(u, 7.0), check=False)
    torch.cuda.synchronize()
    withhold(0)
    hit = max(1, 128 // min(shape[1:])) if shape[0] > 3 else 1      # matrices of the first tile
    assert bool(out[:hit].isnan().all()) and torch.equal(out[hit:], want[hit:])
    assert torch.equal(muon.orthogonalize(u), want)                 # the next call is as before


@pytest.mark.parametrize("product", [14, 15])
def test_only_the_slice_that_waited(withhold, product):
    """Behind the last exchange a CTA's products are its own slice's alone: 300 columns, 112 to a CTA."""
    u = update(1, 128, 300)
    want = muon.orthogonalize(u)
    withhold(product)
    out = muon.orthogonalize(u, check=False)
    torch.cuda.synchronize()
    assert bool(out[..., :112].isnan().all()) and torch.equal(out[..., 112:], want[..., 112:])


def test_it_is_reported(withhold):
    u, w, m = update(2, 128, 300), update(2, 128, 300), torch.zeros(2, 128, 300, device="cuda")
    small, before = [update(4, 32, 72) for _ in range(2)] + [torch.zeros(4, 32, 72, device="cuda")], w.clone()
    expected = [t.clone() for t in (*small, w, m)]
    muon.muon_step([expected[0], expected[3]], [expected[1], u], [expected[2], expected[4]], lr=0.1)
    withhold(5)
    with pytest.raises(RuntimeError, match="orthogonalize: a device-side wait gave up"):
        muon.orthogonalize(u)
    version = w._version
    with pytest.raises(RuntimeError, match="muon_step: a device-side wait gave up"):
        muon.muon_step([small[0], w], [small[1], u], [small[2], m], lr=0.1)
    assert w._version > version
    for got, want in zip([small[0], small[2], m], [expected[0], expected[2], expected[4]]):
        assert torch.equal(got, want)      # other tensors, and all momenta
    assert bool(w[0].isnan().all()) and torch.equal(w[1], expected[3][1]) and not torch.equal(w[1], before[1])
