"""Every row counts, once: tests of the group norm in which a row that is left out or taken twice cannot hide in a tolerance.

Each graph and group gets ONE element of its own, at another row in each call, until every row has had its turn:

* statistics: x is V there and 0 elsewhere, so mean = V / M and var = V^2 / M - mean^2 (M values) come from that row alone;
* gradients: dy is 1 there and 0 elsewhere, so db counts the elements (exactly), dw is their xh, and dx everywhere else in
  the group is  -r (w + xh w xh_there) / M.

Without the row, y and dx of the others are 0 (and dw, db miss it); twice, they are twice as large.  Tolerances are 2^-12 of
the values: statistics and sums take at most 100 roundings of u = 2^-24 each in a row (8 rows of a batch, 8 batches of a piece's
64 rows, 10 halvings over the slots, 4 operations at a time), a relative 2^-17, and xh of random rows is off by as much times
|x| r < 8.  A result in fewer bits adds half a step of its type, of its smallest step where it is subnormal."""
import sys

import numpy as np
import pytest
import torch

from cbm4gnn_amd.norm import GraphBatch, group_norm

U = 2.0 ** -24
REL = 2.0 ** -12
V = 1024.0
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def say(*a):
    print("[gpu-case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda", 0)


def places(ptr, groups, width, turn):
    """(row, channel) of each graph's and group's own element, by turn; graphs without rows have none."""
    ptr = torch.as_tensor(ptr)
    lo, n = ptr[:-1], ptr[1:] - ptr[:-1]
    lo, n = lo[n > 0][:, None], n[n > 0][:, None]
    g = torch.arange(groups)[None]
    return (lo + (turn * groups + g) % n).reshape(-1), (g * width + (turn + g) % width + 0 * lo).reshape(-1)


def turns_of(ptr, groups, most):
    """Enough turns for every row of every graph, or some of them: the first, the last, those around multiples of 64, others."""
    need = -(-int(np.diff(ptr).max()) // groups)
    if need <= most:
        return list(range(need))
    edges = {t for r in range(0, need * groups, 64 * groups) for t in (r // groups - 1, r // groups)} | {0, 1, need - 2, need - 1}
    rng = np.random.default_rng(0)
    picked = sorted(t for t in edges if 0 <= t < need)
    return picked[:40] + picked[-2:] + rng.integers(0, need, 40).tolist()


def statistics_hold(y, x, ptr, groups, eps, dtype):
    """Whether y is the norm of x, which holds one V per graph and group."""
    half = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    n = torch.as_tensor(np.diff(ptr))
    m = (n * (x.size(1) // groups)).double().repeat_interleave(n)[:, None].to(x.device)
    mean = V / m
    want = (x.double() - mean) / torch.sqrt(V * V / m - mean * mean + eps)
    return bool(((y.double() - want).abs() <= (REL + 2 * half) * want.abs() + torch.finfo(dtype).tiny * torch.finfo(dtype).eps).all())


def normalised(x, ptr, groups, eps):
    """(xh, r) in 64 bits, r [rows, groups]."""
    parts, rs = [], []
    for lo, hi in zip(ptr[:-1], ptr[1:]):
        if hi > lo:
            v = x[lo:hi].double().reshape(hi - lo, groups, -1)
            var, mean = torch.var_mean(v, (0, 2), correction=0, keepdim=True)
            r = 1.0 / torch.sqrt(var + eps)
            parts.append(((v - mean) * r).reshape(hi - lo, -1))
            rs.append(r.expand(hi - lo, groups, 1)[:, :, 0])
    return torch.cat(parts), torch.cat(rs)


def gradients_hold(dx, dw, db, dy, xh, r, w, ptr, groups, dtype):
    """Whether these are the gradients for dy, which holds one 1 per graph and group."""
    half = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    rows, ch = xh.shape
    d = dy.double()
    want_dw = (d * xh).sum(0)
    if not torch.equal(db.double(), d.sum(0)) or not bool(((dw.double() - want_dw).abs() <= REL * (d * xh.abs() + d).sum(0)).all()):
        return False
    n = torch.as_tensor(np.diff(ptr)).to(dy.device)
    graph = torch.arange(len(n), device=dy.device).repeat_interleave(n)
    m = (n.double() * (ch // groups))[graph][:, None]
    e = (d * w).reshape(rows, groups, -1)
    s1 = torch.zeros((len(n), groups), dtype=torch.float64, device=dy.device).index_add_(0, graph, e.sum(2))[graph] / m
    s2 = torch.zeros((len(n), groups), dtype=torch.float64, device=dy.device).index_add_(0, graph, (e * xh.reshape(e.shape)).sum(2))[graph] / m
    wide = lambda t: t[:, :, None].expand(rows, groups, ch // groups).reshape(rows, ch)      # noqa: E731
    e = e.reshape(rows, ch)
    want = wide(r) * (e - wide(s1) - xh * wide(s2))
    size = wide(r) * (e.abs() + (xh.abs() + 1) * (wide(s1).abs() + wide(s2).abs()))
    return bool(((dx.double() - want).abs() <= REL * size + 2 * half * want.abs() + torch.finfo(dtype).tiny * torch.finfo(dtype).eps).all())


def cut(rows, graphs, seed):
    at = np.sort(np.random.default_rng(seed).integers(0, rows + 1, graphs - 1)) if graphs > 1 else []
    return [0, *(int(a) for a in at), rows]


# (offsets of the graphs, channels, groups): one launch and pieces, widths that vectors divide and that they do not
CASES = [
    ([0, 9000], 33, 33), ([0, 9000], 602, 602), ([0, 9000], 64, 8), ([0, 4097], 258, 129), ([0, 20011], 128, 128), ([0, 3000], 602, 14),
    ([0, 513], 41, 41), ([0, 300], 602, 14), ([0, 65], 517, 47), ([0, 200], 2560, 2560), ([0, 64], 5120, 5),
    (cut(12000, 5, 1), 48, 48), (cut(12000, 5, 1), 33, 11), (cut(3001, 70, 2), 602, 602), (cut(6000, 300, 3), 256, 256), (cut(500, 90, 4), 40, 8),
    ([0, 1, 1, 9001, 9002, 9064, 9128, 9193], 96, 96),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_every_row_counts_once(gpu, case, dtype):
    ptr, ch, groups = CASES[case]
    rows = ptr[-1]
    say("rows", ptr[:8], len(ptr) - 1, ch, groups, dtype)
    graphs = None if len(ptr) == 2 else GraphBatch(ptr, device=gpu)
    gen = torch.Generator(device=gpu).manual_seed(case)
    w = (1 + 0.1 * torch.randn(ch, generator=gen, device=gpu)).requires_grad_()
    b = torch.zeros(ch, device=gpu, requires_grad=True)
    x = torch.randn((rows, ch), generator=gen, device=gpu).to(dtype).requires_grad_()
    xh, r = normalised(x.detach(), ptr, groups, 1e-5)
    y = group_norm(x, groups, w, b, graphs=graphs)
    for turn in turns_of(ptr, groups, 300):
        at = tuple(t.to(gpu) for t in places(ptr, groups, ch // groups, turn))
        one = torch.zeros((rows, ch), device=gpu)
        one[at] = 1.0
        one = one.to(dtype)
        with torch.no_grad():
            assert statistics_hold(group_norm(V * one, groups, graphs=graphs), V * one, ptr, groups, 1e-5, dtype), turn
        dx, dw, db = torch.autograd.grad(y, (x, w, b), one, retain_graph=True)
        assert gradients_hold(dx, dw, db, one, xh, r, w.detach().double(), ptr, groups, dtype), turn


def definition(x, groups, ptr, eps, count, once=None):
    """The norm in 64 bits with row ``once`` counted ``count`` times in the statistics."""
    out = torch.zeros_like(x, dtype=torch.float64)
    for lo, hi in zip(ptr[:-1], ptr[1:]):
        v = x[lo:hi].double().reshape(hi - lo, groups, -1)
        k = torch.ones((hi - lo, 1, 1), dtype=torch.float64)
        if once is not None and lo <= once < hi:
            k[once - lo] = count
        m = (hi - lo) * v.size(2)
        mean = (k * v).sum((0, 2), keepdim=True) / m
        var = (k * (v - mean) ** 2).sum((0, 2), keepdim=True) / m
        out[lo:hi] = ((v - mean) / torch.sqrt(var + eps)).reshape(hi - lo, -1)
    return out


@pytest.mark.parametrize("count", [0, 1, 2])
@pytest.mark.parametrize("ptr,ch,groups", [([0, 9000], 33, 33), ([0, 4097], 24, 3), ([0, 500, 3000], 16, 16)])
def test_these_tests_see_a_row_lost_or_doubled(ptr, ch, groups, count):
    """The checks on the definition itself, in which one row counts 0, 1 or 2 times: they hold for 1 alone."""
    at = places(ptr, groups, ch // groups, 7)
    one = torch.zeros((ptr[-1], ch))
    one[at] = 1.0
    row = int(at[0][-1])
    y = definition(V * one, groups, ptr, 1e-5, count, row)
    assert statistics_hold(y, V * one, ptr, groups, 1e-5, BF16) == (count == 1)
    gen = torch.Generator().manual_seed(1)
    x, w = torch.randn((ptr[-1], ch), generator=gen), (1 + 0.1 * torch.randn(ch, generator=gen)).double()
    xh, r = normalised(x, ptr, groups, 1e-5)
    dy = one.double().clone()
    dy[row] *= count                                        # what the sums see
    rows, wide = ptr[-1], lambda t: t[:, :, None].expand(rows, groups, ch // groups).reshape(rows, ch)      # noqa: E731
    sums = torch.zeros((2, rows, groups), dtype=torch.float64)
    for lo, hi in zip(ptr[:-1], ptr[1:]):
        e = (dy[lo:hi] * w).reshape(hi - lo, groups, -1)
        for k, t in enumerate((e, e * xh[lo:hi].reshape(e.shape))):
            sums[k, lo:hi] = t.sum((0, 2)) / e[:, 0].numel()
    dx = wide(r) * (one.double() * w - wide(sums[0]) - xh * wide(sums[1]))
    dw, db = (dy * xh).sum(0), dy.sum(0)
    good_dw, good_db = (one.double() * xh).sum(0), one.double().sum(0)
    hold = lambda *g: gradients_hold(*g, one, xh, r, w, ptr, groups, BF16)      # noqa: E731
    assert hold(dx, good_dw, good_db) == (count == 1)
    assert hold(wide(r) * 0 + dx, dw, good_db) == (count == 1) and hold(dx, good_dw, db) == (count == 1)


def test_every_row_has_its_turn():
    for ptr, ch, groups in CASES:
        if len(turns_of(ptr, groups, 300)) == -(-int(np.diff(ptr).max()) // groups):
            seen = torch.cat([places(ptr, groups, ch // groups, t)[0] for t in turns_of(ptr, groups, 300)])
            assert torch.equal(seen.unique(), torch.arange(ptr[-1])), ptr[:4]
    full = [len(turns_of(p, g, 300)) == -(-int(np.diff(p).max()) // g) for p, _, g in CASES]
    assert sum(full) >= 12
