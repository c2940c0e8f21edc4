"""Group norm with an activation over node features, for the place between a GCN's layers.

The reference's model has nothing but a ReLU there (``benchmark/parallel/benchmark_gcn_cpu.py:84-88``).  Features
are [nodes, channels]; a group of channels is normalised over the nodes of ITS graph: one graph (the default), a
batch of graphs laid end to end (``GraphBatch``), or a dense batch [samples, ..., channels], where every index of
the first dimension is a graph of its own::

    y = group_norm(x, 8, weight, bias, graphs=GraphBatch(ptr), activation="silu")

Elements are float32, bfloat16 or float16; weight, bias and all statistics are float32.  The calls enqueue on
torch's current stream and return.  Calls on CPU tensors are staged through the GPU, as the multiply's are.
"""
from __future__ import annotations

import functools

import numpy as np
import torch
from torch import nn

from . import _lib
from ._dense import _require_gpu, _stream, check_dtype, check_int32, rows_view

__all__ = ["GraphBatch", "group_norm", "GroupNorm"]

# Rows of a piece of a graph that is too long for one workgroup: 512 pieces over all rows (2 workgroups per CU), at
# least 64 rows each.  232,965 x 128: joining 512 pieces takes 7 us, 1024 11 us, 2048 20 us, while the passes over the
# rows gain 2 us at most.
_PIECES, _MIN_PIECE_ROWS = 512, 64


def _piece_rows(rows):
    return max(_MIN_PIECE_ROWS, -(-rows // _PIECES))


@functools.lru_cache(maxsize=64)
def _equal_batch(samples, length):
    """The rows of ``samples`` graphs of ``length`` nodes each."""
    rows = samples * length
    return _lib.autograd_lib().NormBatch(samples, length, rows, _piece_rows(rows), 0, [])


class GraphBatch:
    """Where the graphs of a batch begin and end: ``ptr`` = [0, nodes of the first graph, ..., all nodes],
    ascending (a graph may be empty).  Checked on the host once; the device arrays are made once per device
    (``device=``: now, which a program that captures its calls into a HIP graph needs)."""

    def __init__(self, ptr, device=None):
        host = torch.as_tensor(ptr)
        if host.dim() != 1 or host.numel() < 1 or host.dtype.is_floating_point or host.dtype == torch.bool:
            raise ValueError("ptr must be a non-empty list of whole numbers")
        host = host.detach().cpu().numpy().astype(np.int64)
        lengths = np.diff(host)
        if host[0] != 0 or (lengths < 0).any():
            raise ValueError("ptr must begin with 0 and never fall")
        check_int32(int(host[-1]), "nodes of the batch")
        check_int32(len(lengths), "graphs of the batch")
        self.n_graphs, self.n_nodes = len(lengths), int(host[-1])
        self.max_nodes = int(lengths.max()) if len(lengths) else 0
        self._ptr = host.astype(np.int32)
        rows = self._rows = _piece_rows(self.n_nodes)
        per_graph = -(-lengths // rows)
        first = np.concatenate([[0], np.cumsum(per_graph)])
        graph = np.repeat(np.arange(self.n_graphs), per_graph)
        start = host[:-1][graph] + (np.arange(first[-1]) - first[:-1][graph]) * rows
        count = np.minimum(rows, host[1:][graph] - start)
        self._pieces = np.stack([graph, start, count, np.zeros_like(graph)], axis=1).astype(np.int32)
        self._piece_ptr = first.astype(np.int32)
        # longest first: a long graph begun last would run on alone
        self._order = np.argsort(-lengths, kind="stable").astype(np.int32)
        self._on = {}
        if device is not None:
            _require_gpu()
            self._struct(torch.device(device))

    def __getstate__(self):
        return {**self.__dict__, "_on": {}}                 # a copy makes its own device arrays

    def _struct(self, device):
        if device.index is None:
            device = torch.device(device.type, torch.cuda.current_device())
        held = self._on.get(device)
        if held is None:
            arrays = [torch.from_numpy(a).to(device) for a in (self._ptr, self._pieces, self._piece_ptr, self._order)]
            # whoever holds the struct (a backward to come) holds the arrays
            st = _lib.autograd_lib().NormBatch(self.n_graphs, self.max_nodes, self.n_nodes, self._rows, len(self._pieces), arrays)
            held = self._on[device] = (st, _stream(device).value)
        st, home = held
        if _stream(device).value != home:                   # not to be reused for others before this stream is done with them
            for a in st.arrays:
                a.record_stream(torch.cuda.current_stream(device))
        return st


def _check_channel(t, name, ch, device):
    if t is None:
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != torch.float32:
        raise RuntimeError(f"{name} tensor (NOT torch::kFloat32)")
    if t.dim() != 1 or t.size(0) != ch or (ch > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be [{ch}] with unit stride, got shape {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} and x are on different devices")


def group_norm(x, groups, weight=None, bias=None, *, graphs=None, eps=1e-5, activation="none"):
    """``activation((x - mean) / sqrt(var + eps) * weight + bias)`` with mean and (biased) variance per graph and
    group of ``channels / groups`` channels; differentiable in ``x``, ``weight`` and ``bias``.

    x: [nodes, channels] (one graph, or the graphs of ``graphs`` end to end), or [samples, ..., channels]
    (without ``graphs``: a graph per sample); unit stride along channels, rows any stride apart.
    activation: "none", "relu" (its derivative at zero is zero) or "silu".  Returns a contiguous tensor of x's
    shape and type.  A graph without nodes gives and takes nothing."""
    check_dtype(x, "x")
    if activation not in _lib.CBM_ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_lib.CBM_ACTIVATIONS)}, got {activation!r}")
    if x.dim() < 2:
        raise ValueError(f"x must be [nodes, channels] or [samples, ..., channels], got shape {tuple(x.shape)}")
    ch, groups, eps = x.size(-1), int(groups), float(eps)
    if groups < 1 or ch < 1 or ch % groups:
        raise ValueError(f"{ch} channels do not divide into {groups} groups")
    if ch > 1 << 16:
        raise ValueError(f"{ch} channels: at most {1 << 16}")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    if graphs is not None:
        if not isinstance(graphs, GraphBatch):
            raise TypeError("graphs must be a GraphBatch")
        if x.dim() != 2:
            raise ValueError("with graphs, x must be [nodes, channels]")
        if x.size(0) != graphs.n_nodes:
            raise ValueError(f"x has {x.size(0)} rows, the batch has {graphs.n_nodes} nodes")
    _check_channel(weight, "weight", ch, x.device)
    _check_channel(bias, "bias", ch, x.device)
    rows_view(x, "x")
    samples = graphs.n_graphs if graphs is not None else 1 if x.dim() == 2 else x.size(0)
    if samples > _lib.CBM_NORM_MAX_GRAPHS or samples * groups > _lib.CBM_NORM_MAX_PAIRS:
        raise ValueError(f"{samples} graphs of {groups} groups: at most {_lib.CBM_NORM_MAX_GRAPHS} graphs, and "
                         f"{_lib.CBM_NORM_MAX_PAIRS} graphs times groups")
    if graphs is None:
        check_int32(x.numel() // ch, "rows of x")
    _require_gpu()
    if not x.is_cuda:
        staged = [None if t is None else t.to("cuda") for t in (x, weight, bias)]
        return group_norm(staged[0], groups, *staged[1:], graphs=graphs, eps=eps, activation=activation).to(x.device)
    batch = graphs._struct(x.device) if graphs is not None else _equal_batch(samples, x.numel() // ch // samples if samples else 0)
    act = _lib.CBM_ACTIVATIONS[activation]
    return _lib.autograd_lib().group_norm(x, weight, bias, batch, groups, eps, act)


class GroupNorm(nn.Module):
    """``group_norm`` with a weight (ones) and a bias (zeros); ``affine=False`` leaves both out."""

    def __init__(self, groups: int, channels: int, eps: float = 1e-5, activation: str = "none", affine: bool = True):
        super().__init__()
        if groups < 1 or channels < 1 or channels % groups:
            raise ValueError(f"{channels} channels do not divide into {groups} groups")
        if activation not in _lib.CBM_ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(_lib.CBM_ACTIVATIONS)}, got {activation!r}")
        self.groups, self.channels, self.eps, self.activation = int(groups), int(channels), float(eps), activation
        self.weight = nn.Parameter(torch.ones(channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(channels)) if affine else None

    def forward(self, x, graphs=None):
        return group_norm(x, self.groups, self.weight, self.bias, graphs=graphs, eps=self.eps, activation=self.activation)

    def extra_repr(self):
        return f"{self.groups}, {self.channels}, eps={self.eps}, activation={self.activation!r}, affine={self.weight is not None}"
