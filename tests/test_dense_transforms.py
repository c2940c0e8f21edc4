"""What follows torch's operators cannot follow the dense operators' kernels, which write through raw pointers: where it
would go on with a wrong result, the calls raise.  The checks run on CPU tensors too, before anything is launched."""
import sys

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from cbm4gnn_amd import _lib
from cbm4gnn_amd.labels import label_log_probs
from cbm4gnn_amd.norm import GroupNorm, group_norm
from cbm4gnn_amd.optim import muon_step, orthogonalise


def say(*a):
    print("[gpu-case]", *a, flush=True)
    sys.stdout.flush()


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda", 0)


def native(x, labels, weight=None, bias=None):
    """The two operators' native calls as a list, each of them without the public call's own checks."""
    lib = _lib.autograd_lib()
    batch = lib.NormBatch(1, x.size(0), x.size(0), 64, 0, [])
    return [lambda: lib.group_norm(x, weight, bias, batch, 2, 1e-5, 2), lambda: lib.label_scores(x, labels, True, 2, -100)]


FORWARD = "no forward-mode derivative"
TRACED = "cannot be traced"


def tracers():
    """Ways to trace f(x)."""
    return [lambda f, x: torch.jit.trace(f, x, check_trace=False), lambda f, x: make_fx(f)(x), lambda f, x: make_fx(f, tracing_mode="fake")(x)]


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused(requires_grad):
    """Of every differentiable input, whether or not it requires a gradient of its own."""
    x, w, labels = torch.randn((6, 8)), torch.ones(8), torch.arange(6)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.clone().requires_grad_(requires_grad), torch.ones_like(x))
        dual_w = forward_ad.make_dual(w.clone().requires_grad_(requires_grad), torch.ones_like(w))
        for call in native(dual, labels) + native(x, labels, dual_w)[:1] + native(x, labels, None, dual_w)[:1]:
            for context in (torch.enable_grad, torch.no_grad):
                with context(), pytest.raises(RuntimeError, match=FORWARD):
                    call()
        with pytest.raises(RuntimeError, match=FORWARD):
            orthogonalise(dual)
        for at in range(3):
            args = [[dual] if i == at else [torch.zeros_like(x)] for i in range(3)]
            with pytest.raises(RuntimeError, match=FORWARD):
                muon_step(*args, lr=0.1)


@pytest.mark.gpu
def test_forward_mode_is_refused_on_the_gpu_and_ends_with_its_level(gpu):
    say("forward mode")
    x, labels = torch.randn((6, 8), device=gpu), torch.arange(6, device=gpu)
    norm = GroupNorm(2, 8).to(gpu)
    want = [norm(x), label_log_probs(x, labels).logp, orthogonalise(x)]
    calls = [norm, lambda t: label_log_probs(t, labels).logp, orthogonalise]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        host = forward_ad.make_dual(x.cpu(), torch.ones_like(x).cpu())
        for call, plain in zip(calls, want):
            with pytest.raises(RuntimeError, match=FORWARD):
                call(dual)
            assert torch.equal(call(x), plain)              # a tensor without a tangent is as welcome as ever
            with forward_ad._set_fwd_grad_enabled(False):   # as inside a torch.autograd.Function
                assert torch.equal(call(dual), plain)
        for call in (lambda t: group_norm(t, 2), lambda t: label_log_probs(t, labels.cpu())):
            with pytest.raises(RuntimeError, match=FORWARD):
                call(host)
    for call, plain in zip(calls, want):
        assert torch.equal(call(x), plain)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("requires_grad", [False, True])
def test_tracing_is_refused(requires_grad):
    """A trace would hold the allocation of the result and nothing that fills it."""
    x, labels = torch.randn((6, 8)).requires_grad_(requires_grad), torch.arange(6)

    def muon(t):
        muon_step([t], [t + 1], [t + 2], lr=0.1)
        return t
    for trace in tracers():
        for k in range(2):
            for context in (torch.enable_grad, torch.no_grad):
                with context(), pytest.raises(RuntimeError, match=TRACED):
                    trace(lambda t: native(t, labels)[k](), x)
        with pytest.raises(RuntimeError, match=TRACED):
            trace(lambda t: orthogonalise(t), x)
        with pytest.raises(RuntimeError, match=TRACED + "|data pointer"):      # (a fake tensor has no memory to check for overlaps)
            trace(muon, x)


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore")
def test_tracing_is_refused_on_the_gpu_and_ends_with_its_trace(gpu):
    say("tracing")
    x, labels = torch.randn((6, 8), device=gpu), torch.arange(6, device=gpu)
    calls = [GroupNorm(2, 8).to(gpu), lambda t: label_log_probs(t, labels, entropy=True)[:2], lambda t: orthogonalise(t)]
    for trace in tracers()[:2]:
        for call in calls:
            want = call(x)
            with pytest.raises(RuntimeError, match=TRACED):
                trace(call, x)
            for p, q in zip(want, call(x)):
                assert torch.equal(p, q)
        for call in (lambda t: group_norm(t, 2), lambda t: label_log_probs(t, labels.cpu()).logp):
            with pytest.raises(RuntimeError, match=TRACED):
                trace(call, x.cpu())


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore")
def test_function_transforms_raise(gpu):
    """vmap, grad and jvp of torch.func hand wrapped tensors on, which have no memory of their own."""
    say("torch.func")
    x, labels = torch.randn((3, 6, 8), device=gpu), torch.arange(6, device=gpu)
    calls = [lambda t: group_norm(t, 2), lambda t: label_log_probs(t, labels).logp, lambda t: label_log_probs(t, entropy=True).entropy, orthogonalise]
    for call in calls:
        for transform in (lambda: torch.func.vmap(call)(x), lambda: torch.func.grad(lambda t: call(t).sum())(x[0]),
                          lambda: torch.func.jvp(call, (x[0],), (x[1],)), lambda: torch.func.functionalize(call)(x[0])):
            with pytest.raises((RuntimeError, ValueError)):     # ValueError: the C ABI's, of a pointer that is NULL
                transform()
    leaf = x[0].clone().requires_grad_()
    for call in calls[:3]:
        y = call(leaf)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, leaf, torch.ones((4, *y.shape), device=gpu), is_grads_batched=True)
    compiled = torch.compile(lambda t: group_norm(t * 2, 2) + 1, backend="eager")
    assert torch.equal(compiled(x[0]), group_norm(x[0] * 2, 2) + 1)
