"""The update of a GCN's weight matrices by orthogonalised momentum.

``orthogonalise`` maps a matrix towards the nearest one with orthonormal rows or columns by Newton-Schulz products;
``muon_step`` is the optimiser step around it for a list of weights, all of them in the same launches; ``Muon`` is
that step as a ``torch.optim.Optimizer``::

    opt = Muon([p for p in model.parameters() if p.dim() == 2], lr=0.02)

    momentum = mu momentum + grad;   u = grad + mu momentum (nesterov) or momentum
    x = u / (|u| + eps);   steps times:  x = a x + (b A + c A A) x,  A = x x^T  (on the shorter side)
    weight = (1 - lr decay) weight - lr sqrt(max(1, rows / cols)) x

Sums run in float32 and products to 2^-22 of their operands, whatever the matrices' type.  The reference trains
nothing (it has no backward through the multiply).
"""
from __future__ import annotations

import torch

from . import _lib
from ._dense import DTYPES, _require_gpu, _stream, check_dtype, ld, on_device, ptr

__all__ = ["orthogonalise", "muon_step", "Muon", "NS_COEFFICIENTS"]

# Published coefficients of the Muon optimiser: steepest at zero, at the price of singular values that end up
# between about 0.7 and 1.2 instead of at 1.
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_MAX_SIDE = 1 << 20


def _check_steps(steps, coefficients, eps):
    steps, eps = int(steps), float(eps)
    if steps < 1:
        raise ValueError(f"steps must be at least 1, got {steps}")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    if len(coefficients) != 3:
        raise ValueError("coefficients must be three numbers (a, b, c)")
    return steps, [float(v) for v in coefficients], eps


def _check_matrix(t, name):
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(t.shape)}")
    if t.size(1) > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must be row-major with unit column stride")
    if t.size(0) > 1 and t.stride(0) < t.size(1):
        raise ValueError(f"{name} has overlapping rows (stride {t.stride(0)} < width {t.size(1)})")
    if max(t.shape) > _MAX_SIDE:
        raise ValueError(f"{name}: sides of at most {_MAX_SIDE}")


def _workspace(lib, items, n, device):
    size = lib.cbm_ortho_workspace_bytes(items, n)
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


@torch.no_grad()
def orthogonalise(g, steps=5, coefficients=NS_COEFFICIENTS, eps=1e-7):
    """``steps`` Newton-Schulz steps on ``g`` / (|g| + eps): [rows, cols], or [..., rows, cols] for a batch of
    matrices.  float32, bfloat16 or float16; returns a contiguous tensor of its shape and type, outside
    autograd.  Matrices need unit stride along columns.  Zeros give zeros.  Products keep operands as fp16 pairs:
    coefficients under which values grow beyond 65 504 give infinities."""
    check_dtype(g, "g")
    steps, abc, eps = _check_steps(steps, coefficients, eps)
    if g.dim() < 2:
        raise ValueError(f"g must be [..., rows, cols], got shape {tuple(g.shape)}")
    if g.dim() == 2:
        mats = [g]
    else:
        try:
            mats = list(g.view(-1, *g.shape[-2:]).unbind(0)) if g.numel() else []
        except RuntimeError:
            raise ValueError("g: the dimensions before the last two must collapse into one") from None
    if mats:
        _check_matrix(mats[0], "g")
    _lib.autograd_lib().not_followed([g], "orthogonalise")    # torch.no_grad leaves the forward mode on
    _require_gpu()
    if not g.is_cuda:
        return orthogonalise(g.to("cuda"), steps, coefficients, eps).to(g.device)
    out = torch.empty(g.shape, dtype=g.dtype, device=g.device)
    if not g.numel():
        return out
    rows, cols = g.shape[-2:]
    lib = _lib.hip_lib()
    items = (_lib.CbmOrthoItem * len(mats))()
    size, to = out.element_size() * rows * cols, out.data_ptr()
    for i, m in enumerate(mats):
        it = items[i]
        it.src, it.dst, it.rows, it.cols, it.ld_src, it.ld_dst = m.data_ptr(), to + i * size, rows, cols, ld(m), cols
    ws = _workspace(lib, items, len(mats), g.device)
    with on_device(g.device):
        rc = lib.cbm_orthogonalise(items, len(mats), steps, *abc, eps, DTYPES[g.dtype], ptr(ws), _stream(g.device))
    _lib.check(rc, "cbm_orthogonalise")
    return out


@torch.no_grad()
def muon_step(weights, grads, buffers, *, lr, momentum=0.95, weight_decay=0.0, nesterov=True, steps=5,
              coefficients=NS_COEFFICIENTS, eps=1e-7):
    """One step over lists of float32 matrices on one GPU: ``buffers`` (momentum, zeros in the beginning) and
    ``weights`` are updated in place, in launches that all of them share: neither may overlap any other tensor of the
    step (a gradient may be given twice)."""
    steps, abc, eps = _check_steps(steps, coefficients, eps)
    weights, grads, buffers = list(weights), list(grads), list(buffers)
    if not len(weights) == len(grads) == len(buffers):
        raise ValueError(f"{len(weights)} weights, {len(grads)} gradients and {len(buffers)} momentum buffers")
    if not weights:
        return
    seen = set()
    for w, g, b in zip(weights, grads, buffers):
        for t, name in ((w, "weight"), (g, "gradient"), (b, "momentum buffer")):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a torch.Tensor")
            if t.dtype != torch.float32:
                raise RuntimeError(f"{name} tensor (NOT torch::kFloat32)")
            _check_matrix(t, name)
            if t.shape != w.shape:
                raise ValueError(f"{name} has shape {tuple(t.shape)}, the weight {tuple(w.shape)}")
            if t.device != weights[0].device:
                raise ValueError("all tensors of a step must be on one device")
        for t in (w, b):
            if t.numel() and t.data_ptr() in seen:
                raise ValueError("the same weight or momentum buffer is given twice")
            seen.add(t.data_ptr())
    if any(g.numel() and g.data_ptr() in seen for g in grads):
        raise ValueError("a gradient must not be a weight or momentum buffer of the step")
    _lib.autograd_lib().not_followed(weights + grads + buffers, "muon_step")
    _require_gpu()
    dev = weights[0].device
    if dev.type != "cuda":
        staged = [[t.to("cuda") for t in ts] for ts in (weights, grads, buffers)]
        muon_step(*staged, lr=lr, momentum=momentum, weight_decay=weight_decay, nesterov=nesterov, steps=steps,
                  coefficients=coefficients, eps=eps)
        for host, gpu in ((weights, staged[0]), (buffers, staged[2])):
            for t, s in zip(host, gpu):
                t.copy_(s)
        return
    lib = _lib.hip_lib()
    items = (_lib.CbmOrthoItem * len(weights))()
    for it, w, g, b in zip(items, weights, grads, buffers):
        it.src, it.weight, it.momentum = g.data_ptr(), w.data_ptr(), b.data_ptr()
        it.rows, it.cols = w.shape
        it.ld_src, it.ld_weight, it.ld_momentum = ld(g), ld(w), ld(b)
    ws = _workspace(lib, items, len(weights), dev)
    with on_device(dev):
        rc = lib.cbm_muon_step(items, len(weights), float(lr), float(momentum), float(weight_decay), int(bool(nesterov)), steps, *abc,
                               eps, ptr(ws), _stream(dev))
    _lib.check(rc, "cbm_muon_step")
    # the kernels wrote through raw pointers: let autograd see that what it may have saved has changed
    for t in weights + buffers:
        torch.autograd.graph.increment_version(t)


class Muon(torch.optim.Optimizer):
    """``muon_step`` over parameters that are float32 matrices (biases and norm weights belong to another
    optimiser).  Parameters without a gradient are left alone."""

    def __init__(self, params, lr=0.02, momentum=0.95, weight_decay=0.0, nesterov=True, steps=5, coefficients=NS_COEFFICIENTS,
                 eps=1e-7):
        if not lr >= 0.0 or not 0.0 <= momentum < 1.0 or not weight_decay >= 0.0:
            raise ValueError("lr and weight_decay must not be negative, momentum in [0, 1)")
        steps, coefficients, eps = _check_steps(steps, coefficients, eps)
        super().__init__(params, dict(lr=lr, momentum=momentum, weight_decay=weight_decay, nesterov=nesterov, steps=steps,
                                      coefficients=tuple(coefficients), eps=eps))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dtype != torch.float32:
                    raise RuntimeError("parameter (NOT torch::kFloat32)")
                _check_matrix(p, "parameter")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_device = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("Muon does not take sparse gradients")
                state = self.state[p]
                if "momentum_buffer" not in state:
                    state["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                g = p.grad
                if (g.size(1) > 1 and g.stride(1) != 1) or (g.size(0) > 1 and g.stride(0) < g.size(1)):
                    g = g.contiguous()
                by_device.setdefault(p.device, []).append((p, g, state["momentum_buffer"]))
            for triples in by_device.values():
                muon_step(*zip(*triples), lr=group["lr"], momentum=group["momentum"], weight_decay=group["weight_decay"],
                          nesterov=group["nesterov"], steps=group["steps"], coefficients=group["coefficients"], eps=group["eps"])
        return loss
