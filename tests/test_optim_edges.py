"""Orthogonalisation and the optimiser step where their definition leaves something open: zeros without an eps, lists whose
tensors meet."""
import sys

import pytest
import torch

from cbm4gnn_amd import _lib
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


def test_a_gradient_that_the_step_writes_is_refused():
    """Of whichever item: the items share launches, so one would read what another is writing."""
    ws, ms = [torch.zeros((4, 6)) for _ in range(3)], [torch.zeros((4, 6)) for _ in range(3)]
    for bad in (*ws, *ms, ws[2].view(6, 4).view(4, 6)):
        for at in range(3):
            gs = [torch.zeros((4, 6)) for _ in range(3)]
            gs[at] = bad
            with pytest.raises(ValueError, match="must not be"):
                muon_step(ws, gs, ms, lr=0.1)


CBM_ERR_NULL, CBM_ERR_SHAPE = 1, 3
BASE = 1 << 40


def muon_status(items):
    """Of (gradient, weight, momentum) = (address, ld) each, and a shape: without a workspace, so nothing can be launched."""
    held = (_lib.CbmOrthoItem * len(items))()
    for it, ((g, lg), (w, lw), (m, lm), (rows, cols)) in zip(held, items):
        it.src, it.weight, it.momentum, it.rows, it.cols = g, w, m, rows, cols
        it.ld_src, it.ld_weight, it.ld_momentum = lg, lw, lm
    return _lib.hip_lib().cbm_muon_step(held, len(items), 0.1, 0.9, 0.0, 1, 5, 1.0, 1.0, 1.0, 1e-7, None, None)


def ortho_status(items, dtype):
    held = (_lib.CbmOrthoItem * len(items))()
    for it, ((g, lg), (d, ld), (rows, cols)) in zip(held, items):
        it.src, it.dst, it.rows, it.cols, it.ld_src, it.ld_dst = g, d, rows, cols, lg, ld
    return _lib.hip_lib().cbm_orthogonalise(held, len(items), 5, 1.0, 1.0, 1.0, 1e-7, dtype, None, None)


def test_lists_whose_matrices_meet_are_refused():
    """Matrices that overlap in part, through the C ABI, on made-up addresses."""
    far = iter(range(BASE, 1 << 50, 1 << 30))
    new = lambda cols: (next(far), cols)                    # noqa: E731
    rows, cols = 5, 7
    size = 4 * rows * cols
    fine = [(new(7), new(7), new(7), (rows, cols)) for _ in range(30)]
    assert muon_status(fine) == CBM_ERR_NULL                # nothing amiss but the workspace
    w, m = fine[11][1][0], fine[29][2][0]
    for at in (w, w + 4, w - 4, w + size - 4, w - size + 4, m, m + 8):
        for item in ((new(7), (at, 7), new(7), (rows, cols)), (new(7), new(7), (at, 7), (rows, cols)), ((at, 7), new(7), new(7), (rows, cols))):
            for place in (0, 30):
                assert muon_status(fine[:place] + [item] + fine[place:]) == CBM_ERR_SHAPE
    for at in (w + size, w - size, m + size):
        assert muon_status(fine + [((at, 7), new(7), new(7), (rows, cols))]) == CBM_ERR_NULL
    g = fine[3][0]
    assert muon_status(fine + [(g, new(7), new(7), (rows, cols))]) == CBM_ERR_NULL                    # a gradient given twice
    ld = 40                                                 # columns of one buffer: 7, 20 and 13 wide
    parts = [((BASE + 4 * c, ld), new(width), new(width), (n, width)) for c, width, n in ((0, 7, 5), (7, 20, 9), (27, 13, 1))]
    turned = [(g, w, m, shape) for w, g, m, shape in parts]
    assert muon_status(turned) == CBM_ERR_NULL
    assert muon_status(turned + [(new(3), (BASE + 4 * 38, ld), new(3), (5, 3))]) == CBM_ERR_SHAPE       # into the next row
    assert muon_status([(new(7), new(7), new(7), (rows, cols)), ((BASE, 7), (BASE, 7), (BASE, 7), (0, 7))]) == CBM_ERR_NULL
    for dtype, e in ((0, 4), (1, 2), (2, 2)):
        many = [(new(7), new(7), (rows, cols)) for _ in range(30)]
        assert ortho_status(many, dtype) == CBM_ERR_NULL
        src, dst = many[4][0][0], many[28][1][0]
        for at in (src, src + e, dst, dst - e):
            assert ortho_status(many + [(new(7), (at, 7), (rows, cols))], dtype) == CBM_ERR_SHAPE
        assert ortho_status(many + [((dst, 7), new(7), (rows, cols))], dtype) == CBM_ERR_SHAPE
        assert ortho_status(many + [((src, 7), (src + e * rows * cols, 7), (rows, cols))], dtype) == CBM_ERR_NULL
