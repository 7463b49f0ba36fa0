"""The first calls of a process, made by two threads at once: each needs kernels whose shared memory has to be allowed before."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
import threading
import torch
from mlp_splatting_b200 import muon
from mlp_splatting_b200 import primitive_csr as pc

torch.cuda.synchronize()
g = torch.Generator().manual_seed(1)
updates = [torch.randn(s, generator=g).cuda() for s in ((2, 128, 700), (700, 32, 800), (400, 64, 384), (1200, 16, 1024))]
ids = torch.randint(0, 200_000, (200_000, 1), generator=g, dtype=torch.int32).cuda()
w, grads = torch.randn(3, 128, 300, generator=g).cuda(), torch.randn(3, 128, 300, generator=g).cuda()
torch.cuda.synchronize()
barrier, results, failures = threading.Barrier(2), [None, None], []


def work():
    weights, momenta = w.clone(), torch.zeros_like(w)
    muon.muon_step(weights, grads, momenta, lr=0.1)
    route = pc.route_records(ids, 200_000)
    return [weights, route.offsets, route.slots, *(muon.orthogonalize(u) for u in updates)]


def first(k):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            barrier.wait()
            results[k] = work()
            torch.cuda.current_stream().synchronize()
    except Exception as e:
        failures.append(repr(e))


threads = [threading.Thread(target=first, args=(k,)) for k in range(2)]
for t in threads:
    t.start()
for t in threads:
    t.join()
assert not failures, failures
for a, b, c in zip(*results, work()):
    assert torch.equal(a, b) and torch.equal(a, c)
print("as one")
"""


@pytest.mark.parametrize("attempt", range(3))
def test_first_calls_of_two_threads(attempt):
    run = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "as one" in run.stdout, run.stdout + run.stderr
