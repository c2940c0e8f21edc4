"""Group norm with an activation against its definition in 64 bits on the CPU: one graph, batches of graphs (empty
ones and single nodes among them), dense batches, widths no vector divides, both launch forms, both directions; its
refusals (no GPU needed).

Tolerances count roundings.  With u = 2^-24 (half a step of fp32), a statistic over a graph is joined from batches:
no sum is longer than the graph's rows, so n u (sum of magnitudes) bounds its error, and 2^-21 covers the dozen
roundings of one element (subtract, scale, shift, exp with its argument, quotient, products).  A result in fewer bits
adds half a step of its type, ``finfo.eps / 2`` relative."""
import ctypes as C
import sys

import numpy as np
import pytest
import torch

from cbm4gnn_amd import _lib
from cbm4gnn_amd.norm import GraphBatch, GroupNorm, group_norm

U = 2.0 ** -24
FEW = 2.0 ** -21
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def say(*a):
    print("[gpu-case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda", 0)


def reference(x, groups, w, b, ptr, eps, act, dy):
    """(y, dx, dw, db, scale of y's error, scale of dx's error) in float64; x, dy [rows, C]."""
    x = x.detach().double().cpu()
    ch = x.size(1)
    w = torch.ones(ch, dtype=torch.float64) if w is None else w.detach().double().cpu()
    b = torch.zeros(ch, dtype=torch.float64) if b is None else b.detach().double().cpu()
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    dw, db = torch.zeros(ch, dtype=torch.float64), torch.zeros(ch, dtype=torch.float64)
    ey, edx = torch.zeros_like(x), torch.zeros_like(x)
    edw, edb = torch.zeros_like(dw), torch.zeros_like(db)
    dy = None if dy is None else dy.detach().double().cpu()
    for lo, hi in zip(ptr[:-1], ptr[1:]):
        if lo == hi:
            continue
        n = hi - lo
        v = x[lo:hi].reshape(n, groups, -1)
        mean = v.mean((0, 2), keepdim=True)
        var = ((v - mean) ** 2).mean((0, 2), keepdim=True)
        r = 1.0 / torch.sqrt(var + eps)
        xh = ((v - mean) * r).reshape(n, ch)
        u = xh * w + b
        s = torch.sigmoid(u)
        y[lo:hi] = u * s if act == "silu" else u.clamp(min=0) if act == "relu" else u
        # error of xh: of the mean (n u max|x| r) and of r (n u relative, on xh)
        size = v.abs().amax((0, 2), keepdim=True)
        rr, sz = r.expand_as(v).reshape(n, ch), size.expand_as(v).reshape(n, ch)
        exh = (n * U + FEW) * (xh.abs() + 1) + 4 * U * sz * rr + n * U * sz * rr * U
        eu = exh * w.abs() + FEW * (u.abs() + b.abs())
        ey[lo:hi] = 1.1 * eu + FEW * (1 + u.abs()) * y[lo:hi].abs()      # |silu'| < 1.1
        if dy is None:
            continue
        g = dy[lo:hi]
        d = g * (s * (1 + u * (1 - s))) if act == "silu" else g * (u > 0) if act == "relu" else g
        ed = 0.5 * eu * g.abs() + FEW * (1 + u.abs()) * d.abs() if act == "silu" else FEW * d.abs()   # |silu''| <= 0.5
        dw += (d * xh).sum(0)
        db += d.sum(0)
        edw += n * U * (d * xh).abs().sum(0) + (ed * xh.abs() + d.abs() * exh).sum(0)
        edb += n * U * d.abs().sum(0) + ed.sum(0)
        e = (d * w).reshape(n, groups, -1)
        xg = xh.reshape(n, groups, -1)
        c1, c2 = e.mean((0, 2), keepdim=True), (e * xg).mean((0, 2), keepdim=True)
        dx[lo:hi] = (r * (e - c1 - xg * c2)).reshape(n, ch)
        ee = (ed * w.abs() + FEW * (d * w).abs()).reshape(n, groups, -1)
        ex = exh.reshape(n, groups, -1)
        ec1 = n * U * e.abs().mean((0, 2), keepdim=True) + ee.mean((0, 2), keepdim=True)
        ec2 = n * U * (e * xg).abs().mean((0, 2), keepdim=True) + (ee * xg.abs() + e.abs() * ex).mean((0, 2), keepdim=True)
        parts = (e.abs() + c1.abs() + (xg * c2).abs())
        edx[lo:hi] = (r * (ee + ec1 + ex * c2.abs() + xg.abs() * ec2 + (n * U + FEW) * parts)).reshape(n, ch)
    return y, dx, dw, db, ey, edx, edw, edb


def close(got, want, err, dtype, what):
    half = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    # a subnormal result of fp16 is off by half of its smallest step
    tol = err + half * (want.abs() + err) + torch.finfo(dtype).tiny
    off = (got.detach().double().cpu() - want).abs()
    assert torch.isfinite(got).all(), what
    assert bool((off <= tol).all()), f"{what}: off by {float((off / tol).max()):.3g} times the tolerance"


def inputs(rows, ch, dtype, seed, offset=1.0, affine=True):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, ch), generator=g) * (0.5 + torch.rand(ch, generator=g)) + offset * torch.randn(ch, generator=g)).to(dtype)
    w = 1 + 0.1 * torch.randn(ch, generator=g) if affine else None
    b = 0.1 * torch.randn(ch, generator=g) if affine else None
    dy = torch.randn((rows, ch), generator=g).to(dtype)
    return x, w, b, dy


def ragged(rows, graphs, seed):
    cut = np.sort(np.random.default_rng(seed).integers(0, rows + 1, graphs - 1)) if graphs > 1 else np.zeros(0, dtype=np.int64)
    return [0, *cut.tolist(), rows]


def check(gpu, x, groups, w, b, dy, ptr, act, eps=1e-5, graphs=None, shape=None):
    xd = x.to(gpu) if shape is None else x.reshape(shape).to(gpu)
    leaves = [t if t is None else t.to(gpu).requires_grad_() for t in (xd, w, b)]
    y = group_norm(leaves[0], groups, leaves[1], leaves[2], graphs=graphs, eps=eps, activation=act)
    torch.cuda.synchronize()
    wanted = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(y, wanted, dy.reshape(y.shape).to(gpu))
    torch.cuda.synchronize()
    with torch.no_grad():
        again = group_norm(leaves[0], groups, leaves[1], leaves[2], graphs=graphs, eps=eps, activation=act)
    assert torch.equal(again, y)                           # the same bits with and without what the backward keeps
    ry, rdx, rdw, rdb, ey, edx, edw, edb = reference(x, groups, w, b, ptr, eps, act, dy)
    flat = lambda t: t.reshape(x.shape)                     # noqa: E731
    close(flat(y), ry, ey, x.dtype, "y")
    close(flat(grads[0]), rdx, edx, x.dtype, "dx")
    if w is not None:
        close(grads[1], rdw, edw + 1e-30, F32, "dw")
        close(grads[2], rdb, edb + 1e-30, F32, "db")
    second = torch.autograd.grad(group_norm(leaves[0], groups, leaves[1], leaves[2], graphs=graphs, eps=eps, activation=act), wanted,
                                 dy.reshape(y.shape).to(gpu))
    for p, q in zip(grads, second):
        assert torch.equal(p, q)                           # no order of additions depends on chance


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,ch,groups", [
    (1, 8, 2), (2, 1, 1), (7, 3, 3), (50, 24, 8), (64, 64, 4), (513, 41, 41), (300, 602, 14), (33, 1280, 5), (200, 5120, 1),
    (9000, 33, 3), (20011, 64, 8), (3000, 602, 7),
])
def test_one_graph(gpu, rows, ch, groups, dtype, act):
    say("norm", rows, ch, groups, dtype, act)
    x, w, b, dy = inputs(rows, ch, dtype, rows + ch)
    check(gpu, x, groups, w, b, dy, [0, rows], act)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,graphs,ch,groups,dtype", [
    (10, 10, 16, 2, F32), (500, 60, 128, 8, BF16), (500, 200, 64, 32, F16), (3001, 70, 602, 14, F16), (12000, 3, 128, 8, F32),
    (9001, 90, 40, 5, F32), (40000, 2, 24, 3, BF16), (6000, 300, 256, 32, BF16),
])
def test_batch_of_graphs(gpu, rows, graphs, ch, groups, dtype):
    say("norm batch", rows, graphs, ch, groups, dtype)
    ptr = ragged(rows, graphs, rows)
    x, w, b, dy = inputs(rows, ch, dtype, rows + graphs)
    check(gpu, x, groups, w, b, dy, ptr, "silu", graphs=GraphBatch(ptr))


@pytest.mark.gpu
def test_one_long_graph_among_many_short_ones(gpu):
    ptr = [0, 0, 1, 1, 15001, 15002, 15004, 15004] + list(range(15010, 15410, 4)) + [15410, 15410]
    say("norm skewed batch", ptr[-1])
    x, w, b, dy = inputs(ptr[-1], 48, F32, 3)
    check(gpu, x, 4, w, b, dy, ptr, "silu", graphs=GraphBatch(torch.tensor(ptr)))


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((5, 7, 16), 4), ((3, 4, 5, 24), 6), ((1, 9000, 64), 8), ((200, 1, 32), 4), ((4, 6000, 16), 2)])
def test_dense_batches(gpu, shape, groups):
    say("norm dense", shape, groups)
    rows, ch, per = int(np.prod(shape[:-1])), shape[-1], int(np.prod(shape[1:-1]))
    x, w, b, dy = inputs(rows, ch, F32, rows)
    check(gpu, x, groups, w, b, dy, list(range(0, rows + 1, per)), "silu", shape=shape)


@pytest.mark.gpu
def test_relu_and_no_parameters(gpu):
    """Values kept away from the ReLU's corner, where the gradient jumps."""
    say("norm relu")
    rows, ch, groups = 400, 32, 4
    x, w, b, dy = inputs(rows, ch, F32, 5)
    u = reference(x, groups, w, b, [0, rows], 1e-5, "none", None)[0]
    x = torch.where(u.abs() < 1e-3, x + 0.05, x)
    u = reference(x, groups, w, b, [0, rows], 1e-5, "none", None)[0]
    dy = torch.where(u.abs() < 1e-4, 0.0, dy.double()).float()
    check(gpu, x, groups, w, b, dy, [0, rows], "relu")
    x, _, _, dy = inputs(rows, ch, F32, 6, affine=False)
    check(gpu, x, groups, None, None, dy, [0, rows], "none")
    zero = torch.zeros((4, 8), device=gpu, requires_grad=True)      # u = 0 everywhere: the derivative there is 0
    y = group_norm(zero, 2, activation="relu")
    assert torch.equal(y, torch.zeros_like(y))
    assert torch.equal(torch.autograd.grad(y.sum(), zero)[0], torch.zeros_like(zero))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [40, 30000])
def test_a_mean_far_from_zero_costs_no_digits(gpu, rows):
    """Mean 4096, deviation 1: the squares alone would lose all of fp32's digits.  x itself carries u 4096 of rounding,
    which the reference shares: it starts from the same fp32 values."""
    say("norm far mean", rows)
    g = torch.Generator().manual_seed(rows)
    x = 4096 + torch.randn((rows, 16), generator=g)
    dy = torch.randn((rows, 16), generator=g)
    check(gpu, x, 4, torch.ones(16), torch.zeros(16), dy, [0, rows], "silu")


@pytest.mark.gpu
def test_strided_rows_and_expanded_gradients(gpu):
    say("norm strides")
    x, w, b, dy = inputs(300, 40, F32, 9)
    wide = torch.full((300, 57), float("nan"), device=gpu)
    wide[:, 3:43] = x.to(gpu)
    view = wide[:, 3:43].requires_grad_()                  # rows 57 apart, beginning 12 bytes into a row
    y = group_norm(view, 5, w.to(gpu), b.to(gpu), activation="silu")
    plain = x.to(gpu).requires_grad_()
    y2 = group_norm(plain, 5, w.to(gpu), b.to(gpu), activation="silu")
    assert torch.equal(y, y2) and y.is_contiguous()
    for make in (lambda t: t.sum(), lambda t: (t.t() @ torch.ones(300, 1, device=gpu)).sum()):
        a = torch.autograd.grad(make(y), view, retain_graph=True)[0]
        c = torch.autograd.grad(make(y2), plain, retain_graph=True)[0]
        assert torch.equal(a, c)
    turned = dy.t().contiguous().t().to(gpu)               # column-major gradient
    assert torch.equal(torch.autograd.grad(y, view, turned)[0], torch.autograd.grad(y2, plain, dy.to(gpu))[0])


@pytest.mark.gpu
def test_nan_stays_in_its_graph_and_group(gpu):
    say("norm nan")
    for rows, ptr in ((60, [0, 20, 40, 60]), (30000, [0, 10000, 20000, 30000])):
        x, w, b, dy = inputs(rows, 16, F32, 1)
        x[ptr[1] + 3, 5] = float("nan")                    # graph 1, group 1 of 4
        xd = x.to(gpu).requires_grad_()
        y = group_norm(xd, 4, w.to(gpu), b.to(gpu), graphs=GraphBatch(ptr), activation="silu")
        dx, = torch.autograd.grad(y, xd, dy.to(gpu))
        for t in (y, dx):
            bad = torch.isnan(t).cpu()
            assert bad[ptr[1]:ptr[2], 4:8].all()
            bad[ptr[1]:ptr[2], 4:8] = False
            assert not bad.any()


@pytest.mark.gpu
def test_a_backward_outlives_its_batch(gpu):
    """The GraphBatch is gone, and its memory handed out again, before the gradient is asked for."""
    say("norm batch gone")
    x, w, b, dy = (t.to(gpu) for t in inputs(900, 16, F32, 1))
    leaf = x.clone().requires_grad_()
    held = GraphBatch([0, 300, 900])
    want, = torch.autograd.grad(group_norm(leaf, 4, w, b, graphs=held, activation="silu"), leaf, dy)
    y = group_norm(leaf, 4, w, b, graphs=GraphBatch([0, 300, 900]), activation="silu")
    torch.cuda.synchronize()
    others = [torch.full((k,), 7, dtype=torch.int32, device=gpu) for k in (3, 3, 60, 60, 128, 128)]
    got, = torch.autograd.grad(y, leaf, dy)
    assert torch.equal(got, want) and len(others) == 6


@pytest.mark.gpu
def test_gradient_against_differences(gpu):
    """d/dh of sum(dy y(x + h v)) at 0 by central differences of the kernel's own forward.  Truncation: h^2 / 6 times
    the third derivative; rounding: each y is off by a few u, so the quotient by u sqrt(n) few / h.  h = 2^-6 balances
    both below 2e-3 of the norms here; the analytic value is of the order of |dx| |v|."""
    say("norm differences")
    rows, ch = 80, 24
    x, w, b, dy = (t.to(gpu) for t in inputs(rows, ch, F32, 2))
    v = torch.randn((rows, ch), generator=torch.Generator().manual_seed(4)).to(gpu)
    h = 2.0 ** -6
    run = lambda t: (group_norm(t, 4, w, b, activation="silu").double() * dy.double()).sum()    # noqa: E731
    numeric = float((run(x + h * v) - run(x - h * v)) / (2 * h))
    leaf = x.clone().requires_grad_()
    dx, = torch.autograd.grad(group_norm(leaf, 4, w, b, activation="silu"), leaf, dy)
    assert abs(float((dx.double() * v.double()).sum()) - numeric) <= 2e-3 * float(dx.norm() * v.norm())


@pytest.mark.gpu
def test_only_some_gradients_and_empty_inputs(gpu):
    say("norm needs")
    for rows in (50, 30000):
        x, w, b, dy = (t.to(gpu) for t in inputs(rows, 16, F32, 8))
        full = [t.clone().requires_grad_() for t in (x, w, b)]
        want = torch.autograd.grad(group_norm(full[0], 4, full[1], full[2], activation="silu"), full, dy)
        for i in range(3):
            args = [x, w, b]
            args[i] = args[i].clone().requires_grad_()
            got, = torch.autograd.grad(group_norm(args[0], 4, args[1], args[2], activation="silu"), args[i], dy)
            assert torch.equal(got, want[i])
    empty = torch.zeros((0, 16), device=gpu, requires_grad=True)
    w = torch.ones(16, device=gpu, requires_grad=True)
    for graphs in (None, GraphBatch([0, 0, 0]), GraphBatch([0])):
        y = group_norm(empty, 4, w, graphs=graphs)
        gx, gw = torch.autograd.grad(y.sum(), (empty, w))
        assert y.shape == (0, 16) and gx.shape == (0, 16) and torch.equal(gw, torch.zeros_like(gw))
    assert group_norm(torch.zeros((0, 4, 16), device=gpu), 4).shape == (0, 4, 16)


@pytest.mark.gpu
def test_another_stream_and_cpu_tensors(gpu):
    say("norm stream")
    x, w, b, dy = inputs(5000, 32, F32, 8)
    want = group_norm(x.to(gpu), 4, w.to(gpu), b.to(gpu), activation="silu")
    side = torch.cuda.Stream()
    batch = GraphBatch([0, 5000], device=gpu)
    xd, wd, bd = x.to(gpu), w.to(gpu), b.to(gpu)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = group_norm(xd, 4, wd, bd, activation="silu", graphs=batch)
    side.synchronize()
    assert torch.equal(got, want)
    xc = x.clone().requires_grad_()
    y = group_norm(xc, 4, w, b, activation="silu")
    assert y.device.type == "cpu" and torch.equal(y, want.cpu())
    leaf = x.to(gpu).requires_grad_()
    torch.autograd.backward(y, dy)
    gx, = torch.autograd.grad(group_norm(leaf, 4, wd, bd, activation="silu"), leaf, dy.to(gpu))
    assert torch.equal(xc.grad, gx.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,graphs", [(300, 5), (30000, 3)])
def test_captured_graphs_replay(gpu, rows, graphs):
    """Forward and gradients in two captured graphs over other inputs, replayed in turns with eager work between."""
    say("norm capture", rows)
    batch = GraphBatch(ragged(rows, graphs, 1), device=gpu)
    held = []
    for seed in (1, 2):
        x, w, b, dy = (t.to(gpu) for t in inputs(rows, 48, F32, seed))
        leaves = [t.requires_grad_() for t in (x, w, b)]
        run = lambda l=leaves, d=dy: torch.autograd.grad(group_norm(l[0], 6, l[1], l[2], graphs=batch, activation="silu"), l, d)   # noqa: E731
        want = run()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        held.append((graph, out, want, leaves, run))
    for turn in range(4):
        for graph, out, want, leaves, run in held:
            for t in out:
                t.fill_(float("nan"))
            graph.replay()
            eager = run()
            torch.cuda.synchronize()
            for p, q, r in zip(out, want, eager):
                assert torch.equal(p, q) and torch.equal(r, q), turn


@pytest.mark.gpu
def test_many_short_graphs_behind_a_long_one(gpu):
    """More graphs times groups than a join of 1024 threads each may have in one launch.  Whole numbers in dy: their
    sums are exact in any order."""
    short, ch, long = 300_000, 8, 20_000
    rows = long + 3 * short
    say("many pairs", rows, short)
    g = torch.Generator().manual_seed(5)
    x = torch.randn((rows, ch), generator=g) + torch.randn(ch, generator=g)
    dy = torch.randint(-3, 4, (rows, ch), generator=g).float()
    w, b = 1 + 0.1 * torch.randn(ch, generator=g), 0.1 * torch.randn(ch, generator=g)
    ptr = np.concatenate([[0], long + 3 * np.arange(short + 1)])
    leaves = [t.to(gpu).requires_grad_() for t in (x, w, b)]
    y = group_norm(leaves[0], ch, leaves[1], leaves[2], graphs=GraphBatch(ptr))
    dx, _, db = torch.autograd.grad(y, leaves, dy.to(gpu))
    assert torch.equal(db.cpu(), dy.sum(0))
    picks = [0, 1, 2, short] + np.random.default_rng(0).integers(1, short, 100).tolist()
    at = torch.cat([torch.arange(ptr[p], ptr[p + 1]) for p in picks])
    sub = np.concatenate([[0], np.cumsum([ptr[p + 1] - ptr[p] for p in picks])]).tolist()
    ry, rdx, _, _, ey, edx, _, _ = reference(x[at], ch, w, b, sub, 1e-5, "none", dy[at])
    close(y.detach().cpu()[at], ry, ey, F32, "y")
    close(dx.cpu()[at], rdx, edx, F32, "dx")


@pytest.mark.gpu
@pytest.mark.parametrize("first,graphs", [(1100, 2000), (2_190_000, 1)])
def test_elements_beyond_2_to_the_31(gpu, first, graphs):
    """The last graph of a batch whose elements pass 2^31, short graphs in one launch and a long one in pieces."""
    ch, groups, last = 1024, 32, 1100
    rows = first * graphs + last
    say("far elements", rows, ch)
    assert (rows - last) * ch > 1 << 31
    g = torch.Generator(device=gpu).manual_seed(2)
    x = torch.randn((rows, ch), generator=g, device=gpu, dtype=BF16).requires_grad_()
    dy = torch.randn((rows, ch), generator=g, device=gpu, dtype=BF16)
    w, b = (1 + 0.1 * torch.randn(ch, generator=g, device=gpu)).requires_grad_(), torch.zeros(ch, device=gpu, requires_grad=True)
    batch = GraphBatch([*range(0, first * graphs + 1, first), rows])
    y = group_norm(x, groups, w, b, graphs=batch, activation="silu")
    dx, _, db = torch.autograd.grad(y, (x, w, b), dy)
    tail = lambda t: t.detach()[-last:].cpu()               # noqa: E731
    ry, rdx, _, _, ey, edx, _, _ = reference(tail(x), groups, w, b, [0, last], 1e-5, "silu", tail(dy))
    close(tail(y), ry, ey, BF16, "y")
    close(tail(dx), rdx, edx, BF16, "dx")
    assert torch.isfinite(db).all()


@pytest.mark.gpu
def test_a_second_derivative_is_refused(gpu):
    x = torch.randn((40, 8), device=gpu, requires_grad=True)
    dx, = torch.autograd.grad(group_norm(x, 2, activation="silu").sum(), x, create_graph=True)
    plain, = torch.autograd.grad(group_norm(x, 2, activation="silu").sum(), x)
    assert torch.equal(dx, plain)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_struct_layout():
    assert C.sizeof(_lib.CbmNormBatch) == 56 and _lib.CbmNormBatch.ptr.offset == 24
    assert C.sizeof(_lib.CbmOrthoItem) == 72 and _lib.CbmOrthoItem.ld_src.offset == 40


def test_a_missing_autograd_library_fails_loudly(monkeypatch, tmp_path):
    monkeypatch.setattr(_lib, "_autograd", None)
    monkeypatch.setattr(_lib, "AUTOGRAD_LIB", str(tmp_path / "nope.so"))
    with pytest.raises(_lib.CbmLibraryError):
        _lib.autograd_lib()


def test_too_many_graphs():
    with pytest.raises(ValueError, match="at most"):
        group_norm(torch.empty(((1 << 21) + 1, 1, 2)), 1)
    with pytest.raises(ValueError, match="at most"):
        group_norm(torch.empty((1 << 20, 1, 33)), 33)
    with pytest.raises(ValueError, match="at most"):
        group_norm(torch.empty((0, 2)), 1, graphs=GraphBatch(np.zeros((1 << 21) + 2, dtype=np.int64)))


def test_refusals():
    x = torch.zeros((6, 8))
    with pytest.raises(TypeError):
        group_norm([1.0], 1)
    with pytest.raises(RuntimeError, match="NOT torch::kFloat32"):
        group_norm(x.double(), 2)
    with pytest.raises(RuntimeError, match="NOT torch::kFloat32"):
        group_norm(x, 2, torch.ones(8, dtype=torch.bfloat16))
    for bad in (dict(groups=3), dict(groups=0), dict(groups=-1), dict(groups=2, eps=-1.0), dict(groups=2, eps=float("nan")),
                dict(groups=2, activation="gelu"), dict(groups=2, weight=torch.ones(7)), dict(groups=2, bias=torch.ones(8, 1)),
                dict(groups=2, weight=torch.ones(16)[::2])):
        with pytest.raises(ValueError):
            group_norm(x, **bad)
    for t in (torch.zeros(8), torch.zeros((8, 6)).t(), torch.zeros((1, 8)).expand(6, 8), torch.zeros((6, 2, 8)).transpose(0, 1),
              torch.zeros((2, 0))):
        with pytest.raises(ValueError):
            group_norm(t, 2)
    with pytest.raises(TypeError):
        group_norm(x, 2, graphs=[0, 6])
    with pytest.raises(ValueError, match="6 rows"):
        group_norm(x, 2, graphs=GraphBatch([0, 3, 5]))     # rows behind the last graph
    with pytest.raises(ValueError):
        group_norm(x[None], 2, graphs=GraphBatch([0, 6]))
    for ptr in ([], [1, 2], [0, 3, 2], [[0, 1]], [0.0, 1.0], [0, 1 << 31]):
        with pytest.raises(ValueError):
            GraphBatch(ptr)
    with pytest.raises(ValueError):
        GroupNorm(3, 8)
    with pytest.raises(ValueError):
        GroupNorm(2, 8, activation="tanh")


def test_pieces_cover_every_row_once():
    """The host's cut of ragged batches: every row in one piece of its graph, pieces in order, none over the limit."""
    rng = np.random.default_rng(0)
    for case in range(40):
        rows = int(rng.integers(0, 300000 if case % 4 == 0 else 500))
        ptr = np.array(ragged(rows, int(rng.integers(1, 50)), case))
        b = GraphBatch(ptr)
        at = 0
        for p, (graph, start, count, zero) in enumerate(b._pieces):
            assert start == at and 0 < count <= b._rows and zero == 0
            assert ptr[graph] <= start and start + count <= ptr[graph + 1]
            assert b._piece_ptr[graph] <= p < b._piece_ptr[graph + 1]
            at = start + count
        assert at == rows == b.n_nodes and b._piece_ptr[-1] == len(b._pieces)
        assert b.max_nodes == max(np.diff(ptr), default=0)
