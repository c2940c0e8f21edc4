"""The Newton-Schulz products in each of their tiles (32, 64, 128, alone and mixed), wide and tall, every type, as a result
and as a weight update: bit for bit where the arithmetic is exact, and against 64 bits.

Exact arithmetic: with |G|_F = 2^k, eps = 0, b = 4^k beta and c = 16^k gamma, a step of whole numbers is one of whole numbers:
X = g / 2^k,  A = N / 4^k  with N = g g^T,  and  g' = a g + (beta N + gamma N N) g.  The kernels keep operands in two planes of
11 bits and leave out the product of the two low ones, and add in fp32: nothing is rounded where one operand of each product is
at most 2^11, the other at most 2^22, and all sums of magnitudes stay below 2^24; and nothing is infinite where the values of
X, A and B stay below fp16's largest, 65 504 (which the operator asks for).  ``whole_steps`` holds its inputs to that."""
import ctypes as C
import sys

import pytest
import torch

from cbm4gnn_amd import _lib
from cbm4gnn_amd.optim import NS_COEFFICIENTS, muon_step, orthogonalise

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def say(*a):
    print("[gpu-case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda", 0)


def tiles(shapes):
    items = (_lib.CbmOrthoItem * len(shapes))()
    for it, (r, c) in zip(items, shapes):
        it.rows, it.cols = r, c
    square, wide = C.c_int32(), C.c_int32()
    assert _lib.hip_lib().cbm_ortho_tiles(items, len(shapes), C.byref(square), C.byref(wide)) == 0
    return square.value, wide.value


# (tiles of the symmetric products, of the others): matrices that get them
CASES = {
    (32, 32): [(1, 130, 250), (3, 65, 40), (1, 602, 128)],
    (32, 64): [(1, 700, 1100), (1, 1100, 701)],
    (64, 64): [(1, 1000, 1100), (1, 1101, 1003)],
    (64, 128): [(8, 512, 1024), (8, 1023, 510)],
    (128, 128): [(1, 2048, 2048), (1, 1930, 2047), (1, 2047, 1931), (13, 500, 600)],
}
LISTED = [(pair, case) for pair, cases in CASES.items() for case in cases]


def test_each_pair_of_tiles_has_its_cases():
    for pair, (batch, rows, cols) in LISTED:
        assert tiles([(rows, cols)] * batch) == pair, (batch, rows, cols)
    assert tiles([]) == tiles([(0, 5), (3, 0)]) == (0, 0)
    assert tiles([(0, 5), (700, 1100)]) == tiles([(700, 1100)]) == (32, 64)
    assert tiles([(512, 1024)] * 40) == tiles([(512, 1024)] * 24)          # a turn holds 24
    lib = _lib.hip_lib()
    assert lib.cbm_ortho_tiles(None, 1, C.byref(C.c_int32()), C.byref(C.c_int32())) == 1
    assert lib.cbm_ortho_tiles(None, 0, None, None) == 1


def workspace(shapes):
    items = (_lib.CbmOrthoItem * len(shapes))()
    for it, (r, c) in zip(items, shapes):
        it.rows, it.cols = r, c
    return _lib.hip_lib().cbm_ortho_workspace_bytes(items, len(shapes))


@pytest.mark.parametrize("batch,rows,cols", [(8, 16, 2048), (1, 1, 1 << 20), (24, 33, 1024), (8, 64, 2048), (2048, 8, 1), (24, 1030, 130),
                                             (3, 4096, 300), (8, 512, 1024), (1, 2048, 2048), (5, 700, 1100), (24, 2, 4000)])
def test_padding_stays_within_bounds(batch, rows, cols):
    """No tile that more than doubles the work of tiles of 32, or takes a quarter more than tiles of 64; the workspace goes by
    the same sides."""
    shapes = [(rows, cols)] * batch
    unit = max(tiles(shapes))

    def work(tile):
        s, l = (-(-side // tile) * tile for side in (min(rows, cols), max(rows, cols)))
        return s * s * l, 12 * s * l + 8 * s * s
    assert unit == 32 or work(unit)[0] <= 2 * work(32)[0] * (1.25 if unit == 128 else 1)
    assert unit < 128 or work(128)[0] <= 1.25 * work(64)[0]
    assert workspace(shapes) == min(batch, 24) * work(unit)[1] + workspace([(1, 1)]) - (12 + 8) * 32 * 32


def test_small_matrices_beside_a_large_one_do_not_choose_its_tiles():
    assert tiles([(2048, 2048)]) == tiles([(2048, 2048), (16, 2048), (41, 128), (1, 9)]) == (128, 128)


def whole_numbers(rows, cols, k, seed, size=1):
    """A matrix of zeros and +-size whose squares sum to 4^k, at random places."""
    n = 4 ** k // size ** 2
    assert n * size ** 2 == 4 ** k and n <= rows * cols
    gen = torch.Generator().manual_seed(seed)
    g = torch.zeros(rows * cols, dtype=torch.float64)
    at = torch.randperm(rows * cols, generator=gen)[:n]
    g[at] = size * (2.0 * torch.randint(0, 2, (n,), generator=gen) - 1.0).double()
    return g.view(rows, cols)


def blocks(rows, cols, seed):
    """(matrix, k): blocks [[1, 1], [0, 1]] and single ones with signs, 4^k nonzeros in all, on rows and columns in random order.
    Few enough overlaps for whole numbers to stay small over two steps."""
    k = max(k for k in range(1, 6) if 3 * 4 ** k // 4 <= min(rows, cols))
    q = 4 ** k // 4
    gen = torch.Generator().manual_seed(seed)
    r, c = torch.randperm(rows, generator=gen)[:3 * q], torch.randperm(cols, generator=gen)[:3 * q]
    g = torch.zeros((rows, cols), dtype=torch.float64)
    for i, j in ((slice(0, q), slice(0, q)), (slice(0, q), slice(q, 2 * q)), (slice(q, 2 * q), slice(q, 2 * q)), (slice(2 * q, 3 * q),) * 2):
        g[r[i], c[j]] = 1.0
    signs = 2.0 * torch.randint(0, 2, (cols,), generator=gen).double() - 1.0
    return g * signs, k


def whole_steps(g, steps, a, beta, gamma):
    """The steps in whole numbers (float64 holds them), with what makes the kernels' arithmetic exact."""
    tall = g.size(0) > g.size(1)
    x = g.t().contiguous() if tall else g
    for _ in range(steps):
        xt = x.t().contiguous()
        n = x @ xt
        b = beta * n + gamma * (n @ n)
        # operands: one of 11 bits, one of 22; sums of magnitudes, whatever their order: 24
        assert float(x.abs().max()) <= 2 ** 11 and float(n.abs().max()) <= 2 ** 11 and float(b.abs().max()) <= 65504
        total = abs(a) * x.abs() + b.abs() @ x.abs()
        assert float((x.abs() @ xt.abs()).max()) < 2 ** 24 and float((n.abs() @ n.abs()).max()) < 2 ** 24 and float(total.max()) < 2 ** 24
        x = a * x + b @ x
    return x.t() if tall else x


@pytest.mark.gpu
@pytest.mark.parametrize("pair,case", LISTED)
def test_whole_numbers_bit_for_bit(gpu, pair, case):
    """One step over few and many nonzeros, and two steps, which go through the product that writes X in both orders."""
    batch, rows, cols = case
    say("whole", pair, case)
    runs = []
    for k, (a, beta, gamma) in ((5, (3, 2, -1)), (7, (1, 1, 1))):
        if 4 ** k <= rows * cols / 4:
            runs.append((1, k, (a, beta, gamma), [whole_numbers(rows, cols, k, i) for i in range(batch)]))
    for seed in (100, 200, 300):
        gs, ks = zip(*(blocks(rows, cols, seed + i) for i in range(batch)))
        runs.append((2, ks[0], (1, 1, -1), gs))
    for steps, k, (a, beta, gamma), gs in runs:
        g = torch.stack(list(gs)).to(gpu)
        want = torch.stack([whole_steps(m, steps, a, beta, gamma) for m in g])
        for dtype in (F32, BF16, F16):
            got = orthogonalise(g.to(dtype), steps=steps, coefficients=(a, beta * 4.0 ** k, gamma * 16.0 ** k), eps=0.0)
            assert torch.equal(got, (want / 2.0 ** k).to(F32).to(dtype)), (steps, k, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,batch", [(2048, 2048, 1), (1024, 1024, 4), (2048, 512, 8), (256, 1024, 3), (64, 64, 1)])
def test_whole_numbers_in_every_place(gpu, rows, cols, batch):
    """Matrices of +-1 without a zero and no square of A: every element takes part in every sum."""
    say("dense", rows, cols, batch)
    gen = torch.Generator().manual_seed(rows)
    g = 2.0 * torch.randint(0, 2, (batch, rows, cols), generator=gen).double() - 1.0
    norm = (rows * cols) ** 0.5
    assert norm == int(norm) and (int(norm) & (int(norm) - 1)) == 0
    want = torch.stack([whole_steps(m.to(gpu), 1, 3, 1, 0) for m in g])
    for dtype in (F32, BF16, F16):
        got = orthogonalise(g.to(dtype).to(gpu), steps=1, coefficients=(3.0, norm * norm, 0.0), eps=0.0)
        assert torch.equal(got, (want / norm).to(F32).to(dtype)), dtype


def exact(g, steps=5, coefficients=NS_COEFFICIENTS, eps=1e-7):
    """(result, bound of the Frobenius norm of a kernel's error) in 64 bits.  A product's operands carry 2^-22 each and its
    omitted part 2^-22 more, its sum over K at most (K / 8) u of the magnitudes, so each product of a step errs by at most
    (2^-20 + (K / 8) u) |P|_F |Q|_F; what a step leaves grows by at most the polynomial's steepest slope, a, in each later one."""
    a, b, c = coefficients
    x = g.double()
    tall = x.size(0) > x.size(1)
    x = x.t().contiguous() if tall else x
    x = x / (x.norm() + eps)
    s, l = x.shape
    delta_l, delta_s = 2.0 ** -20 + l / 8 * U, 2.0 ** -20 + s / 8 * U
    err = 8 * U * float(x.norm())
    for _ in range(steps):
        gram = x @ x.t().contiguous()
        poly = b * gram + c * (gram @ gram)
        top = float(torch.linalg.eigvalsh(gram.cpu())[-1]) * (1 + 1e-9)    # the square of the largest singular value
        e_gram = delta_l * float(x.norm()) ** 2
        e_poly = abs(b) * e_gram + abs(c) * (delta_s * float(gram.norm()) ** 2 + 2 * top * e_gram)
        e_step = top ** 0.5 * e_poly + delta_s * float(poly.norm() * x.norm()) + abs(a) * 2.0 ** -21 * float(x.norm())
        x = a * x + poly @ x
        err = a * err + e_step
    return (x.t() if tall else x), err


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("pair,case", [((32, 64), (1, 700, 1100)), ((64, 64), (1, 1101, 1003)), ((64, 128), (8, 512, 1024)),
                                       ((64, 128), (8, 1023, 510)), ((128, 128), (13, 500, 600)), ((128, 128), (1, 1930, 2047)),
                                       ((128, 128), (1, 2047, 1931))])
def test_against_64_bits(gpu, pair, case, dtype):
    batch, rows, cols = case
    say("64 bits", pair, case, dtype)
    assert tiles([(rows, cols)] * batch) == pair
    g = (1e-2 * torch.randn((batch, rows, cols), generator=torch.Generator().manual_seed(rows))).to(dtype).to(gpu)
    got = orthogonalise(g)
    assert torch.isfinite(got).all() and torch.equal(orthogonalise(g), got)
    for i in range(0, batch, 3):
        want, err = exact(g[i])
        half = torch.finfo(dtype).eps / 2 if dtype != F32 else U
        off = float((got[i].double() - want).norm())
        assert off <= err + half * float(want.norm()), (case, i, off)
        if dtype == F32:                                    # and not only within the worst case
            assert off <= 1e-5 * float(want.norm()), (case, i, off / float(want.norm()))
            assert float((got[i].double() - want).abs().max()) <= 1e-4 * float(want.abs().max()), (case, i)


@pytest.mark.gpu
@pytest.mark.parametrize("wide_tall,pair", [(((1900, 2100), (2101, 1903)), (128, 128)), (((700, 801), (901, 703)), (64, 64)),
                                            (((300, 2051), (2051, 301)), (32, 64)), (((512, 1025),) * 4 + ((1025, 511),) * 4, (64, 128))])
def test_weight_updates_of_mixed_lists(gpu, wide_tall, pair):
    """Large wide and tall weights beside tiny ones in padded storage: whole numbers, so the update's own roundings remain.
    The tiniest only without the square of A, which of a matrix of one row and norm 2^5 is 2^20 in whole numbers."""
    say("muon tiles", wide_tall, pair)
    k, lr = 5, 0.125
    for gamma, tiny in ((-1, [(17, 33, 2), (40, 9, 2)]), (0, [(17, 33, 2), (3, 8, 16), (40, 9, 2), (1, 70, 16)])):
        sizes = [(r, c, 1) for r, c in wide_tall] + tiny
        shapes = [(r, c) for r, c, _ in sizes]
        assert tiles(shapes) == pair
        gs = [whole_numbers(r, c, k, i, size) for i, (r, c, size) in enumerate(sizes)]
        os = [whole_steps(g.to(gpu), 1, 3, 1, gamma) / 2.0 ** k for g in gs]
        gen = torch.Generator().manual_seed(3)
        before = [torch.randn(s, generator=gen).to(gpu) for s in shapes]
        ws = [torch.full((r + 1, c + 5), 7.0, device=gpu)[:r, :c].copy_(w) for (r, c), w in zip(shapes, before)]
        ms = [torch.zeros(s, device=gpu) for s in shapes]
        muon_step(ws, [g.float().to(gpu) for g in gs], ms, lr=lr, momentum=0.5, nesterov=False, weight_decay=0.25, steps=1,
                  coefficients=(3.0, 4.0 ** k, gamma * 16.0 ** k), eps=0.0)
        for (r, c), w, m, g, o, old in zip(shapes, ws, ms, gs, os, before):
            assert torch.equal(m.double().cpu(), g), (r, c)
            scale = lr * max(1.0, r / c) ** 0.5
            want = (1 - lr * 0.25) * old.double() - scale * o
            # four roundings of u: the quotient and its root (of a factor), two products, a difference
            tol = 4 * U * (old.double().abs() + (scale * o).abs()) + 2 * U * want.abs()
            assert bool(((w.double() - want).abs() <= tol).all()), (r, c)
            assert bool((w._base[:, c:] == 7.0).all()) and bool((w._base[r:] == 7.0).all()), (r, c)
