"""Newton-Schulz orthogonalisation and the optimiser step around it against 64 bits on the CPU, the refusals (no GPU
needed), and a training step of the whole model: aggregation, norm, loss, update.

Tolerance of an orthogonalisation, from the steps themselves: a product's operands carry 2^-22 each and its omitted
part 2^-22 more, its sum over K at most (K / 8) u of the magnitudes (matrix instructions add 16 products at a time in
fp32, in two chains), so each of the three products of step k errs by at most delta = 2^-20 + (K / 8) 2^-24 of
|P|_F |Q|_F.  What step k leaves behind grows by at most the steepest slope of the step's polynomial, |f'(0)| = a, in
each later step."""
import sys

import numpy as np
import pytest
import torch

from cbm4gnn_amd.optim import NS_COEFFICIENTS, Muon, muon_step, orthogonalise

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


def exact(g, steps=5, coefficients=NS_COEFFICIENTS, eps=1e-7):
    """(result, bound of the Frobenius norm of a kernel's error) in 64 bits; g [rows, cols]."""
    a, b, c = coefficients
    x = g.double()
    tall = x.size(0) > x.size(1)
    x = x.t() if tall else x
    x = x / (x.norm() + eps)
    s, l = x.shape
    delta_l, delta_s = 2.0 ** -20 + l / 8 * U, 2.0 ** -20 + s / 8 * U
    err = 8 * U * float(x.norm())
    for _ in range(steps):
        gram = x @ x.t()
        poly = b * gram + c * gram @ gram
        e_gram = delta_l * float(x.norm()) ** 2
        e_poly = abs(b) * e_gram + abs(c) * (delta_s * float(gram.norm()) ** 2 + 2 * float(torch.linalg.matrix_norm(gram, 2)) * e_gram)
        e_step = float(torch.linalg.matrix_norm(x, 2)) * e_poly + delta_s * float(poly.norm() * x.norm()) + abs(a) * 2.0 ** -21 * float(x.norm())
        x = a * x + poly @ x
        err = a * err + e_step
    return (x.t() if tall else x), err


def close(got, want, err, dtype, what):
    half = torch.finfo(dtype).eps / 2 if dtype != F32 else U
    off = float((got.detach().double().cpu() - want).norm())
    tol = err + half * float(want.norm()) + torch.finfo(dtype).tiny
    assert torch.isfinite(got).all(), what
    assert off <= tol, f"{what}: off by {off / tol:.3g} times the tolerance"
    return off / max(float(want.norm()), 1e-300)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (9, 1), (3, 5), (41, 128), (128, 41), (64, 64), (65, 63), (128, 602), (602, 128),
                                       (130, 129), (200, 1000), (513, 300)])
def test_against_64_bits(gpu, rows, cols, dtype):
    say("ortho", rows, cols, dtype)
    g = (torch.randn((rows, cols), generator=torch.Generator().manual_seed(rows + cols)) * 1e-2).to(dtype)
    got = orthogonalise(g.to(gpu))
    want, err = exact(g)
    assert got.dtype == dtype and got.is_contiguous()
    close(got, want, err, dtype, (rows, cols))
    assert torch.equal(orthogonalise(g.to(gpu)), got)


@pytest.mark.gpu
def test_large_and_batched(gpu):
    say("ortho large")
    g = torch.randn((700, 1100), generator=torch.Generator().manual_seed(1))
    want, err = exact(g)
    rel = close(orthogonalise(g.to(gpu)), want, err, F32, "700 x 1100")
    assert rel < 1e-5                                       # and not only within the worst case
    many = torch.randn((3, 10, 40, 70), generator=torch.Generator().manual_seed(2))     # 30 matrices: more than share one launch
    got = orthogonalise(many.to(gpu))
    assert got.shape == many.shape
    for i in range(3):
        for j in range(10):
            want, err = exact(many[i, j])
            close(got[i, j], want, err, F32, (i, j))
            assert torch.equal(got[i, j], orthogonalise(many[i, j].to(gpu)))      # alone or among others: the same bits


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 12])
def test_steps_and_coefficients(gpu, steps):
    """The cubic that converges (1.5, -0.5, 0) brings every singular value to 1."""
    say("ortho steps", steps)
    g = torch.randn((48, 100), generator=torch.Generator().manual_seed(3))
    for abc in ((1.5, -0.5, 0.0), (2.0, -1.5, 0.5), NS_COEFFICIENTS):
        want, err = exact(g, steps, abc, 1e-3)
        got = orthogonalise(g.to(gpu), steps=steps, coefficients=abc, eps=1e-3)
        close(got, want, err, F32, abc)
    if steps == 12:
        o = orthogonalise(g.to(gpu), steps=12, coefficients=(1.5, -0.5, 0.0)).double().cpu()
        assert float((o @ o.t() - torch.eye(48, dtype=torch.float64)).abs().max()) < 1e-5


@pytest.mark.gpu
def test_sizes_of_values_and_special_ones(gpu):
    say("ortho values")
    g = torch.randn((30, 50), generator=torch.Generator().manual_seed(4))
    for scale in (1e-6, 1.0, 1e6, 1e25):                    # squares of 1e25 leave fp32
        want, err = exact(g * scale)
        close(orthogonalise((g * scale).to(gpu)), want, err, F32, scale)
    spiky = torch.zeros((30, 50))
    spiky[3, 7] = 5.0
    want, err = exact(spiky + 1e-5 * g)
    close(orthogonalise((spiky + 1e-5 * g).to(gpu)), want, err, F32, "one large entry")
    assert torch.equal(orthogonalise(torch.zeros((30, 50), device=gpu)).cpu(), torch.zeros((30, 50)))
    bad = torch.stack([g, g])
    bad[0, 2, 2] = float("nan")
    got = orthogonalise(bad.to(gpu)).cpu()
    assert torch.isnan(got[0]).all() and torch.equal(got[1], orthogonalise(g.to(gpu)).cpu())
    for shape in ((0, 5), (5, 0), (0, 3, 4), (2, 0, 4)):
        assert orthogonalise(torch.zeros(shape, device=gpu)).shape == shape
    wide = torch.full((30, 77), float("nan"), device=gpu)
    wide[:, 5:55] = g.to(gpu)
    assert torch.equal(orthogonalise(wide[:, 5:55]), orthogonalise(g.to(gpu)))
    assert torch.equal(orthogonalise(g), orthogonalise(g.to(gpu)).cpu())


@pytest.mark.gpu
def test_norms_outside_fp32(gpu):
    """Powers of two come out of X = G / |G| exactly, so the bits are those of the unscaled matrix."""
    say("ortho scales")
    g = torch.randint(-7, 8, (64, 80), generator=torch.Generator().manual_seed(9)).float()
    want = orthogonalise(g.to(gpu), eps=0.0)
    for power in (120, 124, -100, -145):                    # |G| = 2^8.2: beyond fp32 at 120; subnormal elements at -145
        scaled = torch.ldexp(g.double(), torch.tensor(power)).float()
        assert torch.isfinite(scaled).all() and torch.equal(scaled.double(), g.double() * 2.0 ** power)
        assert torch.equal(orthogonalise(scaled.to(gpu), eps=0.0), want), power


def muon_reference(w, g, m, lr, mu, decay, nesterov):
    m = mu * m.double() + g.double()
    o, err = exact(g.double() + mu * m if nesterov else m)
    scale = lr * max(1.0, w.size(0) / w.size(1)) ** 0.5
    return (1 - lr * decay) * w.double() - scale * o, m, scale * err


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_steps(gpu, nesterov):
    """Two steps over weights of mixed shapes, more of them than share a launch, some in padded storage."""
    say("muon", nesterov)
    shapes = [(41, 128), (128, 602), (300, 65), (1, 9)] + [(17 + i, 33) for i in range(24)]
    gen = torch.Generator().manual_seed(5)
    ws = [torch.randn(s, generator=gen) for s in shapes]
    ms = [torch.zeros(s) for s in shapes]
    dw = [torch.full((s[0], s[1] + 3), 7.0, device=gpu)[:, :s[1]].copy_(w) for s, w in zip(shapes, ws)]
    dm = [m.to(gpu) for m in ms]
    for _ in range(2):
        gs = [1e-3 * torch.randn(s, generator=gen) for s in shapes]
        muon_step(dw, [g.to(gpu) for g in gs], dm, lr=0.05, momentum=0.9, weight_decay=0.1, nesterov=nesterov)
        torch.cuda.synchronize()
        for i, (w, g, m) in enumerate(zip(ws, gs, ms)):
            rw, rm, err = muon_reference(w, g, m, 0.05, 0.9, 0.1, nesterov)
            assert float((dm[i].double().cpu() - rm).norm()) <= 4 * U * float(rm.norm() + m.double().norm()), i
            # the reference's momentum is not rounded; ours is, by 2 u, which the steps amplify like any error
            assert float((dw[i].double().cpu() - rw).norm()) <= err + 4 * U * float(w.double().norm() + rw.norm()), i
        ws, ms = [w.cpu().clone() for w in dw], [m.cpu().clone() for m in dm]
    assert all(bool((w._base[:, -3:] == 7.0).all()) for w in dw)


@pytest.mark.gpu
def test_muon_optimizer_is_the_step(gpu):
    say("muon optimizer")
    gen = torch.Generator().manual_seed(6)
    start = [torch.randn(s, generator=gen) for s in ((20, 30), (30, 8))]
    params = [torch.nn.Parameter(t.to(gpu)) for t in start] + [torch.nn.Parameter(torch.ones((3, 3), device=gpu))]
    opt = Muon([{"params": params[:1], "lr": 0.1}, {"params": params[1:]}], lr=0.01, weight_decay=0.2)
    ws, ms = [t.to(gpu) for t in start], [torch.zeros(t.shape, device=gpu) for t in start]
    for turn in range(3):
        gs = [torch.randn(t.shape, generator=gen).to(gpu) for t in start]
        params[0].grad, params[1].grad = gs[0].clone(), gs[1].t().contiguous().t()     # one of them column-major
        before = params[0]._version
        opt.step()
        assert params[0]._version > before
        for w, g, m, lr in zip(ws, gs, ms, (0.1, 0.01)):
            muon_step([w], [g], [m], lr=lr, weight_decay=0.2)
        for p, w in zip(params, ws):
            assert torch.equal(p.detach(), w), turn
    assert torch.equal(params[2].detach().cpu(), torch.ones((3, 3)))
    again = Muon([{"params": params[:1], "lr": 0.1}, {"params": params[1:]}])
    again.load_state_dict(opt.state_dict())
    assert torch.equal(again.state[params[0]]["momentum_buffer"], ms[0])
    host = [t.clone() for t in start], [torch.zeros(t.shape) for t in start]
    dev = [t.to(gpu) for t in start], [torch.zeros(t.shape, device=gpu) for t in start]
    gs = [torch.randn(t.shape, generator=gen) for t in start]
    muon_step(host[0], gs, host[1], lr=0.1)
    muon_step(dev[0], [g.to(gpu) for g in gs], dev[1], lr=0.1)
    for a, b in zip(host[0] + host[1], dev[0] + dev[1]):
        assert torch.equal(a, b.cpu())


@pytest.mark.gpu
def test_captured_graphs_replay(gpu):
    say("ortho capture")
    held = []
    for seed in (1, 2):
        g = torch.randn((100, 160), generator=torch.Generator().manual_seed(seed)).to(gpu)
        want = orthogonalise(g)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            orthogonalise(g)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = orthogonalise(g)
        held.append((graph, out, want, g))
    for _ in range(4):
        for graph, out, want, g in held:
            out.fill_(float("nan"))
            graph.replay()
            eager = orthogonalise(g)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(eager, want)


@pytest.mark.gpu
@pytest.mark.parametrize("fused", [True, False])
def test_a_training_step_of_the_model(gpu, fused):
    """Norm, loss and update as the GCN runs them, over a batch of three graphs, two steps, against the same model in
    64 bits on the CPU.  One rounding of fp32 per operation along a chain of about 20 operations with sums over at most
    90 nodes or 24 channels: 1e-4 of the weights' size covers it with the aggregation's own 1e-5."""
    from cbm4gnn_amd import graphs as gen_graphs
    from cbm4gnn_amd.gcn import CBMGCNLayer, TwoLayerGCN, build_operator, optimizers, train_step
    from cbm4gnn_amd.norm import GraphBatch, GroupNorm
    say("gcn train step", fused)
    sizes, parts, off = (40, 30, 20), [], 0
    for k, n in enumerate(sizes):
        parts.append(gen_graphs.add_self_loops(gen_graphs.erdos_renyi(n, 0.2, seed=k), n) + off)
        off += n
    ei = torch.from_numpy(np.concatenate(parts, axis=1).astype(np.int64))
    n, f_in, hidden, classes = off, 24, 16, 7
    op = build_operator(ei, alpha=1, normalized=True)
    batch = GraphBatch([0, 40, 70, 90], device=gpu)
    torch.manual_seed(0)
    model = TwoLayerGCN(CBMGCNLayer(f_in, hidden, op, fused=fused, norm=GroupNorm(4, hidden, activation="silu"), graphs=batch),
                        CBMGCNLayer(hidden, classes, op, fused=fused), relu_between=False).to(gpu)
    x = torch.randn((n, f_in))
    y = torch.randint(0, classes, (n,))
    y[::5] = -100
    deg = torch.zeros(n, dtype=torch.float64).index_add_(0, ei[0], torch.ones(ei.size(1), dtype=torch.float64))
    a = torch.zeros((n, n), dtype=torch.float64)
    a[ei[1], ei[0]] = (deg[ei[0]] * deg[ei[1]]) ** -0.5
    ref = {k: v.detach().double().cpu() for k, v in model.named_parameters()}
    w_names = ["first_layer.lin.weight", "last_layer.lin.weight"]
    mom = {k: torch.zeros_like(ref[k]) for k in w_names}
    adam = {k: [torch.zeros_like(v), torch.zeros_like(v)] for k, v in ref.items() if k not in w_names}

    def ref_logits(p):
        h = a @ (x.double() @ p["first_layer.lin.weight"].t())
        out = []
        for lo, hi in ((0, 40), (40, 70), (70, 90)):
            v = h[lo:hi].reshape(hi - lo, 4, -1)
            var, mean = torch.var_mean(v, (0, 2), correction=0, keepdim=True)
            u = ((v - mean) / torch.sqrt(var + 1e-5)).reshape(hi - lo, -1) * p["first_layer.norm.weight"] + p["first_layer.norm.bias"]
            out.append(u * torch.sigmoid(u))
        return a @ (torch.cat(out) @ p["last_layer.lin.weight"].t())

    opts = optimizers(model, lr=0.02, weight_decay=0.1, vector_lr=1e-2)
    for step in range(1, 3):
        loss = train_step(model, x.to(gpu), y.to(gpu), opts)
        p = {k: v.clone().requires_grad_() for k, v in ref.items()}
        want = torch.nn.functional.cross_entropy(ref_logits(p), y, ignore_index=-100)
        grads = dict(zip(p, torch.autograd.grad(want, list(p.values()))))
        assert abs(float(loss) - float(want)) <= 1e-5 * float(want.detach())
        for k, v in model.named_parameters():
            err = float((v.grad.double().cpu() - grads[k]).abs().max())
            assert err <= 1e-4 * float(grads[k].abs().max()), (k, err)
        for k in w_names:
            mom[k] = 0.95 * mom[k] + grads[k]
            o = exact(grads[k] + 0.95 * mom[k])[0]
            ref[k] = (1 - 0.02 * 0.1) * ref[k] - 0.02 * max(1.0, ref[k].size(0) / ref[k].size(1)) ** 0.5 * o
        for k, (m1, m2) in adam.items():
            m1.mul_(0.9).add_(0.1 * grads[k])
            m2.mul_(0.999).add_(0.001 * grads[k] ** 2)
            ref[k] = ref[k] - 1e-2 * (m1 / (1 - 0.9 ** step)) / ((m2 / (1 - 0.999 ** step)).sqrt() + 1e-8)
        for k, v in model.named_parameters():
            assert float((v.detach().double().cpu() - ref[k]).abs().max()) <= 1e-4 * float(ref[k].abs().max()) + 1e-6, (step, k)
            ref[k] = v.detach().double().cpu()              # the next step starts from the same weights
        for k in w_names:
            mom[k] = opts[0].state[dict(model.named_parameters())[k]]["momentum_buffer"].double().cpu()
    r = model.answer(x.to(gpu), top=3)
    logits = model(x.to(gpu)).detach().cpu()
    assert torch.equal(r.top_index.cpu(), torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :3])
    assert r.logp is None and r.entropy.shape == (n,)
    assert float(model.loss(x.to(gpu), torch.full((n,), -100, device=gpu)).detach()) == 0.0


def test_refusals():
    g = torch.zeros((4, 6))
    with pytest.raises(TypeError):
        orthogonalise([[1.0]])
    with pytest.raises(RuntimeError, match="NOT torch::kFloat32"):
        orthogonalise(g.double())
    for bad in (dict(steps=0), dict(coefficients=(1.0, 2.0)), dict(eps=-1.0), dict(eps=float("nan"))):
        with pytest.raises(ValueError):
            orthogonalise(g, **bad)
    for bad in (torch.zeros(5), torch.zeros((6, 4)).t(), torch.zeros((1, 6)).expand(4, 6), torch.zeros((2, 3, 4, 5)).transpose(0, 1)):
        with pytest.raises(ValueError):
            orthogonalise(bad)
    w, m = torch.zeros((4, 6)), torch.zeros((4, 6))
    with pytest.raises(ValueError):
        muon_step([w], [g], [], lr=0.1)
    with pytest.raises(ValueError):
        muon_step([w], [torch.zeros((6, 4))], [m], lr=0.1)
    with pytest.raises(ValueError):
        muon_step([torch.zeros(4)], [torch.zeros(4)], [torch.zeros(4)], lr=0.1)
    with pytest.raises(ValueError, match="twice"):
        muon_step([w, w], [g, g], [m, torch.zeros((4, 6))], lr=0.1)
    with pytest.raises(ValueError, match="twice"):
        muon_step([w], [g], [w], lr=0.1)
    with pytest.raises(ValueError, match="must not be"):
        muon_step([w], [w], [m], lr=0.1)
    with pytest.raises(RuntimeError, match="NOT torch::kFloat32"):
        muon_step([w.bfloat16()], [g], [m], lr=0.1)
    with pytest.raises(TypeError):
        muon_step([w], [None], [m], lr=0.1)
    muon_step([], [], [], lr=0.1)
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(RuntimeError):
        Muon([torch.nn.Parameter(w.bfloat16())])
    for bad in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(steps=0)):
        with pytest.raises(ValueError):
            Muon([torch.nn.Parameter(w)], **bad)
    from cbm4gnn_amd.gcn import CBMGCNLayer
    from cbm4gnn_amd.norm import GraphBatch, GroupNorm

    class Op:
        num_rows = 6
    with pytest.raises(ValueError, match="channels"):
        CBMGCNLayer(4, 6, Op(), norm=GroupNorm(2, 8))
    with pytest.raises(ValueError, match="norm"):
        CBMGCNLayer(4, 6, Op(), graphs=GraphBatch([0, 6]))
    with pytest.raises(ValueError, match="nodes"):
        CBMGCNLayer(4, 6, Op(), norm=GroupNorm(2, 6), graphs=GraphBatch([0, 5]))
