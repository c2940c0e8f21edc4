"""The largest sizes that the dense operators take, and one more."""
import sys

import pytest
import torch

from cbm4gnn_amd.labels import label_log_probs
from cbm4gnn_amd.norm import group_norm
from cbm4gnn_amd.optim import NS_COEFFICIENTS, orthogonalise

U = 2.0 ** -24
REL = 2.0 ** -14
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def say(*a):
    print("[gpu-case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda", 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape,groups", [((3, 65536), 1), ((3, 65536), 65536), ((300, 65536), 32), ((300, 65535), 5), ((2000, 65536), 65536),
                                          ((64, 2, 4096), 4096), ((70, 3, 65536), 16), ((64, 5, 8192), 8192)])
def test_widest_norms(gpu, shape, groups, dtype):
    """Against the definition in 64 bits.  Sums over at most 2^24 values in chains of at most 100 additions, then a tree: with
    |x| r < 8, 2^-14 of |xh| + 1 covers them and the element's own roundings; the gradient's sums likewise."""
    say("widest norm", shape, groups, dtype)
    gen = torch.Generator(device=gpu).manual_seed(groups)
    x = torch.randn(shape, generator=gen, device=gpu).to(dtype).requires_grad_()
    dy = torch.randn(shape, generator=gen, device=gpu).to(dtype)
    w = (1 + 0.1 * torch.randn(shape[-1], generator=gen, device=gpu)).requires_grad_()
    y = group_norm(x, groups, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    samples = 1 if len(shape) == 2 else shape[0]
    split = (samples, -1, groups, shape[-1] // groups)
    v, d = x.detach().double().reshape(split), dy.double().reshape(split)
    var, mean = torch.var_mean(v, (1, 3), correction=0, keepdim=True)
    r = 1.0 / torch.sqrt(var + 1e-5)
    xh, wd = (v - mean) * r, w.detach().double().reshape(groups, -1)
    e = d * wd
    c1, c2 = e.mean((1, 3), keepdim=True), (e * xh).mean((1, 3), keepdim=True)
    half = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    assert bool(((y.detach().double().reshape(split) - xh * wd).abs() <= (REL + 2 * half) * (xh.abs() + 1) * wd.abs()).all())
    want = r * (e - c1 - xh * c2)
    size = r * (e.abs() + (e.abs().mean((1, 3), keepdim=True) + (e * xh).abs().mean((1, 3), keepdim=True)) * (xh.abs() + 1) + 1e-3)
    assert bool(((dx.double().reshape(split) - want).abs() <= REL * size + 2 * half * want.abs() + 2.0 ** -25).all())
    terms = d * xh
    assert bool(((dw.double() - terms.sum((0, 1)).reshape(-1)).abs() <= REL * (terms.abs() + d.abs()).sum((0, 1)).reshape(-1)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,classes", [(1, 1 << 21), (2, (1 << 21) - 1), (3, (1 << 20) + 5)])
def test_most_classes(gpu, rows, classes, dtype):
    """Chains of at most 64 values of a thread, 10 halvings and 6 joins."""
    say("most classes", rows, classes, dtype)
    gen = torch.Generator(device=gpu).manual_seed(rows)
    z = torch.randn((rows, classes), generator=gen, device=gpu).to(dtype).requires_grad_()
    y = torch.randint(0, classes, (rows,), generator=gen, device=gpu)
    r = label_log_probs(z, y, entropy=True, top=32)
    grad, = torch.autograd.grad((r.logp, r.entropy), z, (torch.ones(rows, device=gpu), torch.full((rows,), 0.5, device=gpu)))
    z64 = z.detach().double()
    lp = torch.log_softmax(z64, 1)
    p = lp.exp()
    h = -(p * lp).sum(1)
    order = torch.sort(z64, dim=1, descending=True, stable=True).indices[:, :32]
    assert torch.equal(r.top_index, order)
    tol = 256 * U                                           # 100 roundings, exponentials of arguments up to 11, log S about 15
    assert bool(((r.logp.double() - lp.gather(1, y[:, None])[:, 0]).abs() <= tol).all())
    assert bool(((r.top_logp.double() - lp.gather(1, order)).abs() <= tol).all())
    assert bool(((r.entropy.double() - h).abs() <= tol * (2 + h)).all())
    want = torch.zeros_like(p).scatter_(1, y[:, None], 1.0) - p - 0.5 * p * (lp + h[:, None])
    half = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    size = p * (1 + 0.5 * (lp.abs() + h[:, None]))
    assert bool(((grad.double() - want).abs() <= tol * (size + want.abs()) + 2 * half * want.abs() + tiny).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(1, 1 << 20), (1 << 20, 1), (2, (1 << 20) - 1), ((1 << 19) + 3, 33)])
def test_longest_matrices(gpu, rows, cols):
    """Of few rows: the steps in 64 bits on the small side.  A sum over K = 2^20 is off by at most (K / 16 + K / 8 / 8) u of its
    magnitudes in the worst case (chains of eight wavefronts); random signs leave its root: 2^-14 covers 5 steps of it."""
    say("longest", rows, cols)
    g = torch.randn((rows, cols), generator=torch.Generator().manual_seed(rows)).to(gpu)
    got = orthogonalise(g)
    a, b, c = NS_COEFFICIENTS
    x = g.double() / (g.double().norm() + 1e-7)
    tall = rows > cols
    x = x.t().contiguous() if tall else x
    for _ in range(5):
        gram = x @ x.t().contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    want = x.t() if tall else x
    off = float((got.double() - want).norm() / want.norm())
    print("off", off)
    assert off <= REL


def test_one_more_is_refused():
    with pytest.raises(ValueError, match="at most"):
        group_norm(torch.empty((1, 65537)), 1)
    with pytest.raises(ValueError, match="at most"):
        label_log_probs(torch.empty((1, (1 << 21) + 1)), top=1)
    with pytest.raises(ValueError, match="at most"):
        orthogonalise(torch.empty((1, (1 << 20) + 1)))
    with pytest.raises(ValueError, match="at most"):
        orthogonalise(torch.empty(((1 << 20) + 1, 1)))
