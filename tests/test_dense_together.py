"""Norm, label scores and orthogonalisation side by side: from two host threads on streams of their own, against the
same calls one after another, bit for bit."""
import copy
import pickle
import sys
import threading

import pytest
import torch

from cbm4gnn_amd.labels import label_log_probs
from cbm4gnn_amd.norm import GraphBatch, group_norm
from cbm4gnn_amd.optim import orthogonalise


def say(*a):
    print("[gpu-case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda", 0)


def inputs(gpu, seed):
    g = torch.Generator().manual_seed(seed)
    rows, ch, classes = 3000 + 17 * seed, 64, 1500
    return {"x": torch.randn((rows, ch), generator=g).to(gpu).requires_grad_(),
            "z": torch.randn((50, classes), generator=g).to(gpu).requires_grad_(),
            "y": torch.randint(0, classes, (50,), generator=g).to(gpu),
            "g": torch.randn((100, 70 + seed), generator=g).to(gpu),
            "dy": torch.randn((rows, ch), generator=g).to(gpu)}


def run(t, graphs):
    n = group_norm(t["x"], 8, graphs=graphs, activation="silu")
    dx, = torch.autograd.grad(n, t["x"], t["dy"])
    r = label_log_probs(t["z"], t["y"], entropy=True, top=3)
    dz, = torch.autograd.grad(r.logp.sum() + r.entropy.sum(), t["z"])
    return [n.detach(), dx, *(v.detach() for v in r), dz, orthogonalise(t["g"])]


@pytest.mark.gpu
def test_two_threads_at_once(gpu):
    work = [inputs(gpu, 0), inputs(gpu, 1)]
    batches = [GraphBatch([0, 10, 10, 2000, len(t["x"])], device=gpu) for t in work]
    want = [run(t, b) for t, b in zip(work, batches)]
    torch.cuda.synchronize()
    say("threads begin")
    got, errors = [[], []], []

    def turns(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i].append(run(work[i], batches[i]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:                              # noqa: BLE001  (told to the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=turns, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    torch.cuda.synchronize()
    for i in (0, 1):
        assert len(got[i]) == 20
        for turn in got[i]:
            for p, q in zip(turn, want[i]):
                assert torch.equal(p, q)


@pytest.mark.gpu
def test_a_used_graph_batch_is_copied_and_pickled(gpu):
    b = GraphBatch([0, 3, 3, 9])
    x = torch.randn((9, 16), device=gpu)
    y = group_norm(x, 4, graphs=b)
    for other in (copy.deepcopy(b), pickle.loads(pickle.dumps(b))):
        assert torch.equal(group_norm(x, 4, graphs=other), y)
