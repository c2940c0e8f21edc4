"""Rows whose label is ignored may hold anything (padding, nodes that were never computed): no gradient comes out of them
unless their entropy or likeliest classes are asked for theirs."""
import sys

import pytest
import torch

from cbm4gnn_amd.labels import label_log_probs

IGNORE = -100


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
@pytest.mark.parametrize("classes", [1, 3, 41, 700, 3001, 50000])
def test_ignored_rows_of_nan_and_inf(gpu, classes, dtype):
    say("left out", classes, dtype)
    rows, top = 12, min(2, classes)
    g = torch.Generator().manual_seed(classes)
    z = torch.randn((rows, classes), generator=g).to(dtype)
    y = torch.randint(0, classes, (rows,), generator=g)
    bad = torch.tensor([1, 4, 5, 8, 11])
    z[1, 0] = float("nan")
    z[4] = float("nan")
    z[5, -1] = float("inf")
    z[8] = float("inf")
    z[11] = -float("inf")
    y[bad] = IGNORE
    y[2] = IGNORE                                           # an ordinary one
    good = torch.tensor([r for r in range(rows) if r not in bad])
    leaf = z.to(gpu).requires_grad_()
    r = label_log_probs(leaf, y.to(gpu), entropy=True, top=top)
    alone_leaf = z[good].to(gpu).requires_grad_()
    alone = label_log_probs(alone_leaf, y[good].to(gpu), entropy=True, top=top)
    assert torch.equal(r.logp[bad], torch.zeros(5, device=gpu))
    gl = torch.randn(rows, generator=g).to(gpu)
    gh, gt = torch.randn(rows, generator=g).to(gpu), torch.randn((rows, top), generator=g).to(gpu)
    gh[bad] = gt[bad] = 0.0
    for use_h in (False, True):
        for use_t in (False, True):
            pick = lambda q, rows=slice(None): ([q.logp] + [q.entropy] * use_h + [q.top_logp] * use_t,      # noqa: E731
                                                [gl[rows]] + [gh[rows]] * use_h + [gt[rows]] * use_t)
            got, = torch.autograd.grad(*(lambda o, d: (o, leaf, d))(*pick(r)), retain_graph=True)
            want, = torch.autograd.grad(*(lambda o, d: (o, alone_leaf, d))(*pick(alone, good)), retain_graph=True)
            assert torch.equal(got[bad], torch.zeros((5, classes), dtype=dtype, device=gpu)), (use_h, use_t)
            assert torch.equal(got[good], want) and torch.isfinite(want).all()
    gh[1], gt[5, 0] = 0.5, 0.5                              # what is asked for does come out: NaN, as the scores are
    got, = torch.autograd.grad((r.entropy, r.logp), leaf, (gh, gl), retain_graph=True)
    assert torch.isnan(got[1]).all() and not torch.isnan(got[[4, 5, 8, 11]]).any()
    got, = torch.autograd.grad((r.top_logp, r.logp), leaf, (gt, gl))
    assert torch.isnan(got[5]).any() and not torch.isnan(got[[1, 4, 8, 11]]).any()
