"""Label scores (log probability, entropy, likeliest classes) against their definition in 64 bits on the CPU, their
gradients against the formula and against differences, and the refusals (no GPU needed).

Tolerances count roundings: u = 2^-24.  A sum of exponentials is joined from partial sums; no chain of additions is
longer than ``chain`` below (the values of one lane, then a tree), every exponential is off by 2 u plus u |argument|."""
import sys

import pytest
import torch

from cbm4gnn_amd.labels import LabelScores, label_log_probs

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
IGNORE = -100


def say(*a):
    print("[gpu-case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda", 0)


def chain(classes):
    return 16 + 16 if classes <= 1024 else classes / 1024 + 64


def make(rows, classes, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    z = (spread * torch.randn((rows, classes), generator=g)).to(dtype)
    y = torch.randint(0, classes, (rows,), generator=g)
    y = torch.where(torch.rand(rows, generator=g) < 0.2, torch.full_like(y, IGNORE), y)
    return z, y


def best(z, k):
    """Stable order: equal values by ascending class."""
    return torch.sort(z.double(), dim=1, descending=True, stable=True).indices[:, :k]


def compare(r, z, y, top, what):
    z64 = z.double()
    lp = torch.log_softmax(z64, 1)
    n = chain(z.size(1))
    m = z64.amax(1)
    log_s = torch.log(torch.exp(z64 - m[:, None]).sum(1))
    p = lp.exp()
    d = torch.where(p > 0, p * (z64 - m[:, None]).abs(), 0.0).sum(1)       # mean |argument| of the exponentials
    base = (n + 8 + d) * U                                  # relative error of the sum = absolute error of its logarithm
    known = y != IGNORE
    want = torch.where(known, lp.gather(1, y.clamp(min=0)[:, None])[:, 0], 0.0)
    tol = base + 4 * U * (want.abs() + log_s.abs() + 1)
    assert bool(((r.logp.double().cpu() - want).abs() <= tol).all()), what
    assert bool((r.logp.cpu()[~known] == 0).all())
    h = -torch.where(p > 0, p * lp, 0.0).sum(1)
    tol_h = (n + 8 + d) * U * (2 + d) + 4 * U * (log_s.abs() + d + 1)
    assert bool(((r.entropy.double().cpu() - h).abs() <= tol_h).all()), what
    if top:
        order = best(z, top)
        assert torch.equal(r.top_index.cpu(), order), what
        want = lp.gather(1, order)
        tol = base[:, None] + 4 * U * (want.abs() + log_s.abs()[:, None] + 1)
        assert bool(((r.top_logp.double().cpu() - want).abs() <= tol).all()), what


def grad_reference(z, y, top, gl, gh, gt):
    z64 = z.double()
    lp = torch.log_softmax(z64, 1)
    p = lp.exp()
    plp = torch.where(p > 0, p * lp, 0.0)
    h = -plp.sum(1, keepdim=True)
    known = (y != IGNORE).double()[:, None]
    gl, gh = gl.double()[:, None] * known, gh.double()[:, None]
    g = torch.zeros_like(z64).scatter_add_(1, y.clamp(min=0)[:, None], gl)
    everything = gl.clone()
    if top:
        g = g.scatter_add(1, best(z, top), gt.double())
        everything = everything + gt.double().sum(1, keepdim=True)
    g = g - p * everything - gh * torch.where(p > 0, p * (lp + h), 0.0)
    n = chain(z.size(1)) + top + 16
    few = (n + 4 * torch.where(p > 0, lp.abs(), torch.zeros_like(lp)) + 4 * h) * U
    err = few * p * (everything.abs() + (0 if not top else gt.double().abs().sum(1, keepdim=True)) +
                     gh.abs() * (torch.where(p > 0, lp.abs(), torch.zeros_like(lp)) + h + 1)) + 8 * U * g.abs()
    # A probability below 2^-126 is not a normal number of fp32 and counts as 0 there, so an element loses
    # p |all + gh (log p + H)| < 2^-126 (|all| + |gh| (|log p| + H)); log p is above -88 - few for a p that is not far below.
    under = torch.where(p > 0, p.clamp(max=2.0 ** -126) * (everything.abs() + gh.abs() * (lp.abs() + h)), torch.zeros_like(p))
    return g, err + under


def check(gpu, z, y, top, what, seed=0):
    say("labels", what)
    zd = z.to(gpu).requires_grad_()
    r = label_log_probs(zd, y.to(gpu), entropy=True, top=top)
    torch.cuda.synchronize()
    compare(r, z, y, top, what)
    g = torch.Generator().manual_seed(seed)
    gl, gh, gt = torch.randn(z.size(0), generator=g), torch.randn(z.size(0), generator=g), torch.randn((z.size(0), max(top, 1)), generator=g)
    parts, grads = [r.logp, r.entropy], [gl.to(gpu), gh.to(gpu)]
    if top:
        parts.append(r.top_logp)
        grads.append(gt.to(gpu))
    got, = torch.autograd.grad(parts, zd, grads, retain_graph=True)
    again, = torch.autograd.grad(parts, zd, grads)
    torch.cuda.synchronize()
    assert torch.equal(got, again)
    want, err = grad_reference(z, y, top, gl, gh, gt)
    half = torch.finfo(z.dtype).eps / 2 if z.dtype != F32 else 0.0
    tol = err + half * (want.abs() + err) + torch.finfo(z.dtype).tiny
    off = (got.double().cpu() - want).abs()
    assert bool((off <= tol).all()), f"{what}: gradient off by {float((off / tol).max()):.3g} times the tolerance"
    with torch.no_grad():
        plain = label_log_probs(zd, y.to(gpu), entropy=True, top=top)
    for p, q in zip(plain, r):
        assert (p is None) == (q is None) and (p is None or torch.equal(p, q))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,classes,top", [
    (1, 1, 1), (1, 2, 2), (5, 3, 0), (70, 4, 3), (300, 41, 5), (33, 64, 8), (65, 65, 10), (3, 127, 32), (20, 172, 7), (9, 300, 32),
    (7, 513, 4), (5, 1024, 9), (5, 1025, 9), (2, 1031, 32), (3, 8193, 10), (1, 100000, 10), (700, 3001, 8), (2, 65537, 32), (600, 1500, 0),
])
def test_scores_and_gradients(gpu, rows, classes, top, dtype):
    z, y = make(rows, classes, dtype, rows + classes)
    check(gpu, z, y, top, (rows, classes, top, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes", [(40, 41), (4, 700), (3, 5000), (520, 9000)])
def test_equal_logits_go_to_the_lowest_class(gpu, rows, classes):
    g = torch.Generator().manual_seed(classes)
    z = torch.randint(-3, 4, (rows, classes), generator=g).float()
    z[0] = 1.5                                             # all equal
    z[1, ::2] = 0.0
    z[1, 1::2] = -0.0                                      # equal as well
    y = torch.randint(0, classes, (rows,), generator=g)
    check(gpu, z, y, min(32, classes), ("ties", rows, classes))


@pytest.mark.gpu
def test_rows_that_crowd_the_likeliest_classes(gpu):
    """Ascending and descending rows, and large values packed into the columns of 31 of the 128 parts a wide row is
    looked at in (more candidates than the list of 2048 holds: 31 parts of 156 columns each)."""
    rows, classes = 513, 20000
    g = torch.Generator().manual_seed(1)
    z = torch.rand((rows, classes), generator=g)
    col = torch.arange(classes)
    part = (col // 4) % 1024 % 128
    z[0] += 5.0 * (part < 31)
    z[1] = col / classes
    z[2] = -col / classes
    z[3] = 0.25
    z[4] += 5.0 * (part >= 97)
    y = torch.randint(0, classes, (rows,), generator=g)
    check(gpu, z, y, 32, "crowded fp32")
    part = (col // 8) % 1024 % 128
    zb = torch.rand((rows, classes), generator=g)
    zb[0] += 5.0 * (part < 31)
    check(gpu, zb.to(BF16), y, 32, "crowded bf16")
    zc = torch.rand((rows, classes), generator=g)
    zc[0, 4096:9000] += 5.0                                # neighbouring columns
    zc[1, :3000:2] += 5.0
    zc[2] = 0.0
    zc[3, 10000:10040] += 5.0
    check(gpu, zc, y, 32, "crowded neighbours")
    check(gpu, zc.to(BF16), y, 32, "crowded neighbours bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("classes", [41, 900, 3000, 50000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_masked_classes(gpu, classes, dtype):
    """-inf and the type's lowest value in masked places, rows with one class left and with none."""
    say("labels masked", classes, dtype)
    rows, top = 6, 5
    z, y = make(rows, classes, dtype, classes)
    g = torch.Generator().manual_seed(3)
    mask = torch.rand((rows, classes), generator=g) < 0.5
    mask[:, :8] = False
    z[mask] = -float("inf")
    z[1, mask[1]] = torch.finfo(dtype).min
    z[2] = -float("inf")
    z[2, 7] = 0.5                                          # one class left
    z[3] = -float("inf")                                   # none
    y = torch.tensor([1, 2, 7, 0, IGNORE, 3])
    zd = z.to(gpu).requires_grad_()
    r = label_log_probs(zd, y.to(gpu), entropy=True, top=top)
    keep = [0, 1, 4, 5]
    compare(type(r)(*(t[keep] for t in r)), z[keep], y[keep], top, "masked")
    assert float(r.logp[2]) == 0.0 and float(r.entropy[2]) == 0.0 and r.top_index[2].tolist() == [7, 0, 1, 2, 3]
    assert r.top_logp[2].tolist() == [0.0] + [-float("inf")] * 4
    assert float(r.logp[3]) == -float("inf") and float(r.entropy[3]) == 0.0
    assert r.top_index[3].tolist() == [0, 1, 2, 3, 4] and r.top_logp[3].tolist() == [-float("inf")] * 5
    grad, = torch.autograd.grad((r.logp, r.entropy), zd, (torch.ones(rows, device=gpu), torch.ones(rows, device=gpu)))
    grad = grad.float().cpu()
    assert torch.isfinite(grad).all()
    assert bool((grad[mask & (torch.arange(rows) != 1)[:, None]] == 0).all())
    assert bool((grad[2] == 0).all()), "one class left: nothing moves"
    assert bool((grad[3] == 0).all()), "none left: no gradient"


@pytest.mark.gpu
@pytest.mark.parametrize("classes", [41, 3000, 50000])
def test_nan_inf_and_labels_out_of_range_stay_in_their_row(gpu, classes):
    say("labels nan", classes)
    z, _ = make(6, classes, F32, 1)
    z[1, 3] = float("nan")
    z[2, 5] = float("inf")
    z[5, 0] = float("nan")
    y = torch.tensor([0, 1, 5, classes, -1, IGNORE])
    zd = z.to(gpu).requires_grad_()
    r = label_log_probs(zd, y.to(gpu), entropy=True, top=3)
    logp, ent = r.logp.cpu(), r.entropy.cpu()
    assert torch.isnan(logp[1:5]).all() and torch.isfinite(logp[0]) and float(logp[5]) == 0.0
    assert torch.isnan(ent[[1, 2, 5]]).all() and torch.isfinite(ent[[0, 3, 4]]).all()
    assert int(r.top_index[1, 0]) == 3 and int(r.top_index[5, 0]) == 0 and int(r.top_index[2, 0]) == 5
    good = best(z[[0, 3, 4]], 3)
    assert torch.equal(r.top_index.cpu()[[0, 3, 4]], good)
    grad, = torch.autograd.grad(r.logp, zd, torch.ones(6, device=gpu))
    grad = grad.cpu()
    assert torch.isfinite(grad[0]).all() and torch.isnan(grad[3]).all() and torch.isnan(grad[4]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes", [(30, 41), (3, 3001)])
def test_logits_far_from_zero(gpu, rows, classes):
    """An offset of 4096 on every logit changes nothing but the digits the logits themselves carry."""
    z, y = make(rows, classes, F32, 4)
    check(gpu, z + 4096.0, y, 4, ("offset", rows, classes))
    check(gpu, z - 30000.0, y, 4, ("offset", rows, classes))
    check(gpu, 40.0 * z, y, 4, ("peaked", rows, classes))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("classes", [41, 3001])
def test_strides_shapes_and_label_types(gpu, classes, dtype):
    say("labels strides", classes, dtype)
    z, y = make(24, classes, dtype, 7)
    want = label_log_probs(z.to(gpu), y.to(gpu), entropy=True, top=4)
    wide = torch.full((24, classes + 9), float("nan"), device=gpu, dtype=dtype)
    wide[:, 3:3 + classes] = z.to(gpu)
    got = label_log_probs(wide[:, 3:3 + classes], y.to(gpu).int(), entropy=True, top=4)
    for p, q in zip(got, want):
        assert torch.equal(p, q)
    cube = label_log_probs(z.to(gpu).view(2, 3, 4, classes), y.to(gpu).view(2, 3, 4), entropy=True, top=4)
    for p, q in zip(cube, want):
        assert torch.equal(p, q.view(2, 3, 4, *q.shape[1:]))
    one = label_log_probs(z[5].to(gpu), y[5].to(gpu), entropy=True, top=4)
    for p, q in zip(one, want):
        assert torch.equal(p, q[5])
    leaf = wide[:, 3:3 + classes].detach().requires_grad_()
    r = label_log_probs(leaf, torch.stack([y, y], 1).to(gpu)[:, 0], entropy=True)
    a, = torch.autograd.grad(r.logp.sum() + 0.5 * r.entropy.sum(), leaf)       # expanded gradients
    leaf2 = z.to(gpu).requires_grad_()
    r2 = label_log_probs(leaf2, y.to(gpu), entropy=True)
    b, = torch.autograd.grad(r2.logp.sum() + 0.5 * r2.entropy.sum(), leaf2)
    assert torch.equal(a, b)
    only = label_log_probs(z.to(gpu), top=4)
    assert only.logp is None and only.entropy is None and torch.equal(only.top_index, want.top_index)
    assert label_log_probs(z.to(gpu), y.to(gpu)).top_logp is None


@pytest.mark.gpu
def test_nothing_to_do_and_cpu_tensors(gpu):
    say("labels empty")
    r = label_log_probs(torch.zeros((0, 7), device=gpu, requires_grad=True), torch.zeros(0, dtype=torch.int64, device=gpu), entropy=True, top=2)
    assert r.logp.shape == (0,) and r.top_index.shape == (0, 2)
    z, y = make(20, 41, F32, 5)
    zc = z.clone().requires_grad_()
    r = label_log_probs(zc, y, entropy=True, top=3)
    zd = z.to(gpu).requires_grad_()
    q = label_log_probs(zd, y.to(gpu), entropy=True, top=3)
    for a, b in zip(r, q):
        assert a.device.type == "cpu" and torch.equal(a, b.cpu())
    (r.logp.sum() + r.entropy.sum()).backward()
    (q.logp.sum() + q.entropy.sum()).backward()
    assert torch.equal(zc.grad, zd.grad.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes", [(30, 41), (2, 9000)])
def test_gradient_against_differences(gpu, rows, classes):
    """Central differences of the kernel's own forward along a random direction.  h = 2^-5: truncation h^2 / 6 times the
    third derivative (of order one here), rounding u |scores| sqrt(rows) / h: together below 2e-3 of the norms."""
    say("labels differences", rows, classes)
    z, y = make(rows, classes, F32, 6)
    z, y = z.to(gpu), y.to(gpu)
    g = torch.Generator().manual_seed(8)
    v = torch.randn((rows, classes), generator=g).to(gpu)
    gl, gh = torch.randn(rows, generator=g).to(gpu), torch.randn(rows, generator=g).to(gpu)
    gt = torch.randn((rows, 3), generator=g).to(gpu)
    index = label_log_probs(z, y, top=3).top_index

    def run(t):
        r = label_log_probs(t, y, entropy=True)
        picked = torch.stack([label_log_probs(t, index[:, i]).logp for i in range(3)], 1)     # the classes that were likeliest
        return (r.logp.double() * gl).sum() + (r.entropy.double() * gh).sum() + (picked.double() * gt).sum()

    h = 2.0 ** -5
    numeric = float((run(z + h * v) - run(z - h * v)) / (2 * h))
    leaf = z.clone().requires_grad_()
    r = label_log_probs(leaf, y, entropy=True, top=3)
    grad, = torch.autograd.grad((r.logp, r.entropy, r.top_logp), leaf, (gl, gh, gt))
    assert abs(float((grad.double() * v.double()).sum()) - numeric) <= 2e-3 * float(grad.norm() * v.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes", [(300, 41), (2, 20000), (600, 1500)])
def test_captured_graphs_replay(gpu, rows, classes):
    say("labels capture", rows, classes)
    held = []
    for seed in (1, 2):
        z, y = make(rows, classes, F32, seed)
        zd, yd = z.to(gpu).requires_grad_(), y.to(gpu)
        gl = torch.randn(rows, generator=torch.Generator().manual_seed(seed)).to(gpu)

        def run(zd=zd, yd=yd, gl=gl):
            r = label_log_probs(zd, yd, entropy=True, top=4)
            g, = torch.autograd.grad((r.logp, r.entropy), zd, (gl, gl))
            return [t.detach() for t in r] + [g]
        want = run()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        held.append((graph, out, want, run))
    for turn in range(4):
        for graph, out, want, run in held:
            for t in out:
                t.fill_(-1)
            graph.replay()
            eager = run()
            torch.cuda.synchronize()
            for p, q, r in zip(out, want, eager):
                assert torch.equal(p, q) and torch.equal(r, q), turn


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes,dtype", [((1 << 25) + 5, 3, F32), ((1 << 21) + 3, 1100, BF16)])
def test_more_rows_than_one_launch(gpu, rows, classes, dtype):
    say("rows", rows, classes, dtype)
    g = torch.Generator(device=gpu).manual_seed(1)
    z = torch.randn((rows, classes), generator=g, device=gpu, dtype=dtype).requires_grad_()
    y = torch.randint(0, classes, (rows,), generator=g, device=gpu)
    y[::7] = IGNORE
    g_logp = torch.randn(rows, generator=g, device=gpu)
    r = label_log_probs(z, y, entropy=True, top=2)
    grad, = torch.autograd.grad(r.logp, z, g_logp)
    edge = 1 << (25 if classes < 1024 else 21)
    at = torch.cat([torch.arange(0, 200), torch.arange(edge - 100, rows)]).to(gpu)
    # a row's scores and gradient depend on nothing but the row: the same bits as those of a call of its own
    part = z.detach()[at].requires_grad_()
    q = label_log_probs(part, y[at], entropy=True, top=2)
    alone, = torch.autograd.grad(q.logp, part, g_logp[at])
    for name in r._fields:
        assert torch.equal(getattr(r, name).detach()[at], getattr(q, name).detach()), name
    assert torch.equal(grad[at], alone)
    compare(LabelScores(*(t.detach().cpu() for t in q)), part.detach().cpu(), y[at].cpu(), 2, "edge rows")


@pytest.mark.gpu
def test_a_second_derivative_is_refused(gpu):
    z, y = torch.randn((40, 8), device=gpu, requires_grad=True), torch.arange(40, device=gpu) % 8
    grad, = torch.autograd.grad(label_log_probs(z, y).logp.sum(), z, create_graph=True)
    plain, = torch.autograd.grad(label_log_probs(z, y).logp.sum(), z)
    assert torch.equal(grad, plain)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_refusals():
    z, y = torch.zeros((4, 5)), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(TypeError):
        label_log_probs([[1.0]], y)
    with pytest.raises(TypeError):
        label_log_probs(z, [0, 1, 2, 3])
    for bad in (z.double(), z.long()):
        with pytest.raises(RuntimeError, match="NOT torch::kFloat32"):
            label_log_probs(bad, y)
    with pytest.raises(RuntimeError, match="labels tensor"):
        label_log_probs(z, y.float())
    for bad in (dict(labels=y[:3]), dict(labels=y[:, None]), dict(labels=y, top=6), dict(labels=y, top=-1), dict()):
        with pytest.raises(ValueError):
            label_log_probs(z, **bad)
    with pytest.raises(ValueError):
        label_log_probs(torch.zeros((4, 50)), y, top=33)
    for bad in (torch.zeros((4, 0)), torch.zeros((5, 4)).t(), torch.zeros((1, 5)).expand(4, 5), torch.zeros(())):
        with pytest.raises(ValueError):
            label_log_probs(bad, y)
