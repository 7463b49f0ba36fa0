"""What the host does when the library's call fails, on a library that is a stand-in."""
import pytest
import torch

from mlp_splatting_b200 import _lib as L
from mlp_splatting_b200 import muon


class Failing:
    """The library, but that its two entries fail with `code`."""

    def __init__(self, code):
        self.code, self.real = code, L.load()

    def __getattr__(self, name):
        if name in ("mlpsp_orthogonalize", "mlpsp_muon_step"):
            return lambda *args: self.code
        return getattr(self.real, name)


# launches before the failing one have written: the tensors count as changed; a refused call has written nothing
@pytest.mark.parametrize("code,written", [(-3, True), (-1, False), (-4, False)])
def test_a_launch_that_fails_raises_the_versions(monkeypatch, code, written):
    lib = Failing(code)
    monkeypatch.setattr(L, "load", lambda: lib)
    monkeypatch.setattr(muon, "_check_tensors", lambda tensors: torch.device("cpu"))
    monkeypatch.setattr(muon, "_stream_ptr", lambda device: None)
    w, g, m, out = (torch.ones(4, 32, 72) for _ in range(4))
    before = [t._version for t in (w, g, m, out)]
    with pytest.raises(RuntimeError, match=f"mlpsp_muon_step failed \\({code}\\)"):
        muon.muon_step(w, g, m, lr=0.1)
    with pytest.raises(RuntimeError, match=f"mlpsp_orthogonalize failed \\({code}\\)"):
        muon.orthogonalize(g, out=out)
    assert [t._version > b for t, b in zip((w, g, m, out), before)] == [written, False, written, written]
