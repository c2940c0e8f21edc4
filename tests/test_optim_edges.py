"""Orthogonalisation and the optimiser step where their definition leaves something open: zeros without an eps, lists whose
tensors meet."""
import sys

import pytest
import torch

from cbm4gnn_amd.optim import muon_step, orthogonalise


def say(*a):
    print("[gpu-case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda", 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1), (30, 50), (65, 40), (300, 1000)])
def test_zeros_give_zeros_without_an_eps(gpu, shape, dtype):
    """Also beside a matrix that is not zero, which they leave as it is (a call chooses its tiles by the shapes of all its
    matrices, so the same bits come from a call of the same shapes)."""
    say("zeros", shape, dtype)
    g = torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(dtype).to(gpu)
    both = torch.stack([torch.zeros_like(g), g])
    got = orthogonalise(both, eps=0.0)
    assert torch.equal(got[0], both[0]) and torch.equal(got[1], orthogonalise(torch.stack([g, g]), eps=0.0)[1]) and torch.isfinite(got).all()


@pytest.mark.gpu
def test_a_step_without_gradient_or_momentum_only_decays(gpu):
    say("muon zeros")
    w = torch.randn((20, 33), generator=torch.Generator().manual_seed(2)).to(gpu)
    before, m = w.clone(), torch.zeros_like(w)
    muon_step([w], [torch.zeros_like(w)], [m], lr=0.5, weight_decay=0.5, eps=0.0)
    assert torch.equal(w, 0.75 * before) and torch.equal(m, torch.zeros_like(m))
