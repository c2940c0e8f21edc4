"""The group norm of long graphs, in pieces, against 64 bits within tolerances that follow the kernel's chains of additions and
not the number of rows: what a piece of 64 rows would be missed in stays far below.

With u = 2^-24.  A channel's statistics of a piece take at most 100 roundings one after another (8 rows of a batch, 8 batches
of 64 rows, 10 halvings over the slots, 4 operations each), and are joined in 64 bits; so do the channel sums of the gradients
(64 rows, 10 halvings), whose sums for dw and db over the pieces take 16 more (parts / 128 in a row, 7 halvings).  So, K = 100:
  mean    off by K u max|x|;   var by K u (1 + 4 max|x| r) relative, the mean's error meeting the distance of two means;
  xh      off by K u max|x| r + |xh| K u (1 + 4 max|x| r) / 2, and a dozen roundings of the element (2^-21);
  dw, db  by (K + 16) u of their magnitudes, and what xh's error makes of each term."""
import sys

import pytest
import torch

from cbm4gnn_amd.norm import GraphBatch, group_norm
from test_norm import inputs

U, FEW, K = 2.0 ** -24, 2.0 ** -21, 100
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def say(*a):
    print("[gpu-case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda", 0)


def reference(x, groups, w, b, ptr, act, dy, lost=slice(0, 0), eps=1e-5):
    """[(value, error that the chains allow)] of y, dx, dw, db in 64 bits; rows ``lost`` left out of every sum."""
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    ch = x.size(1)
    counts = torch.ones(x.size(0), dtype=torch.float64)
    counts[lost] = 0.0
    y, dx, ey, edx = (torch.zeros_like(x) for _ in range(4))
    dw, db, edw, edb = (torch.zeros(ch, dtype=torch.float64) for _ in range(4))
    for lo, hi in zip(ptr[:-1], ptr[1:]):
        n, shape = hi - lo, (hi - lo, groups, ch // groups)
        v, k = x[lo:hi].reshape(shape), counts[lo:hi][:, None, None]
        over = lambda t: (k * t.reshape(shape)).sum((0, 2), keepdim=True) / (n * shape[2])      # noqa: E731
        flat = lambda t: t.expand(shape).reshape(n, ch)     # noqa: E731
        mean = over(v)
        r = 1.0 / torch.sqrt(over((v - mean) ** 2) + eps)
        size = flat(v.abs().amax((0, 2), keepdim=True) * r)
        xh, r = ((v - mean) * r).reshape(n, ch), flat(r)
        exh = K * U * size + xh.abs() * K * U * (1 + 4 * size) / 2 + FEW * (xh.abs() + 1)
        u = xh * w + b
        eu = exh * w.abs() + FEW * (u.abs() + b.abs())
        s = torch.sigmoid(u)
        y[lo:hi] = u * s if act == "silu" else u
        ey[lo:hi] = 1.1 * eu + FEW * (1 + u.abs()) * y[lo:hi].abs()
        g = dy[lo:hi]
        d = g * (s * (1 + u * (1 - s))) if act == "silu" else g
        ed = 0.5 * eu * g.abs() + FEW * (1 + u.abs()) * d.abs() if act == "silu" else FEW * d.abs()
        k1 = counts[lo:hi][:, None]
        dw += (k1 * d * xh).sum(0)
        db += (k1 * d).sum(0)
        edw += (K + 16) * U * (d * xh).abs().sum(0) + (ed * xh.abs() + d.abs() * exh).sum(0)
        edb += (K + 16) * U * d.abs().sum(0) + ed.sum(0)
        e, ee = d * w, ed * w.abs() + FEW * (d * w).abs()
        c1, c2 = flat(over(e)), flat(over(e * xh))
        mean_of = lambda t: flat(t.reshape(shape).mean((0, 2), keepdim=True))      # noqa: E731
        ec1 = K * U * mean_of(e.abs()) + mean_of(ee)
        ec2 = K * U * mean_of((e * xh).abs()) + mean_of(ee * xh.abs() + e.abs() * exh)
        dx[lo:hi] = r * (e - c1 - xh * c2)
        parts = e.abs() + c1.abs() + (xh * c2).abs()
        edx[lo:hi] = r * (ee + ec1 + exh * c2.abs() + xh.abs() * ec2 + FEW * parts) + K * U * (1 + 4 * size) / 2 * dx[lo:hi].abs()
    return [(y, ey), (dx, edx), (dw, edw), (db, edb)]


def excess(got, want, err, dtype):
    """How many times its tolerance the worst element is off."""
    info = torch.finfo(dtype)
    half = info.eps / 2 if dtype != F32 else 0.0
    tol = err + half * (want.abs() + err) + info.tiny * info.eps
    return float(((got.detach().double().cpu() - want).abs() / tol).max())


# offsets, channels, groups; all in pieces of 64 rows
CASES = [([0, 9000], 33, 3), ([0, 20011], 64, 8), ([0, 3000], 602, 7), ([0, 4000, 9000, 12007], 128, 8), ([0, 30000], 24, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("ptr,ch,groups", CASES)
def test_within_the_chains(gpu, ptr, ch, groups, dtype, act):
    say("chains", ptr, ch, groups, dtype, act)
    x, w, b, dy = inputs(ptr[-1], ch, dtype, ch)
    leaves = [t.to(gpu).requires_grad_() for t in (x, w, b)]
    y = group_norm(leaves[0], groups, leaves[1], leaves[2], graphs=GraphBatch(ptr) if len(ptr) > 2 else None, activation=act)
    grads = torch.autograd.grad(y, leaves, dy.to(gpu))
    for name, got, (want, err), t in zip(("y", "dx", "dw", "db"), (y, *grads), reference(x, groups, w, b, ptr, act, dy), (dtype, dtype, F32, F32)):
        assert torch.isfinite(got).all() and excess(got, want, err, t) <= 1.0, (name, excess(got, want, err, t))


@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("ptr,ch,groups", CASES)
def test_a_lost_piece_fails(ptr, ch, groups, act):
    """The first, the last and a middle piece left out of the definition's own sums."""
    x, w, b, dy = inputs(ptr[-1], ch, F32, ch)
    whole = reference(x, groups, w, b, ptr, act, dy)
    for lost in (slice(0, 64), slice(64 * (ptr[1] // 128), 64 * (ptr[1] // 128) + 64), slice(ptr[-1] - (ptr[-1] - ptr[-2]) % 64, ptr[-1])):
        wrong = reference(x, groups, w, b, ptr, act, dy, lost)
        for name, (got, _), (want, err) in zip(("y", "dx", "dw", "db"), wrong, whole):
            assert excess(got, want, err, F32) > 3.0, (name, lost, excess(got, want, err, F32))
