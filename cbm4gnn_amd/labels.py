"""Scores of a node classifier's logits: the log probability of each node's label, the entropy of its distribution
and its likeliest classes, in one pass over the logits, and their gradient.

The reference's benchmark stops at the logits (``benchmark/parallel/benchmark_gcn_cpu.py:70-103``)::

    r = label_log_probs(logits, labels, entropy=True, top=5)
    loss = -r.logp.sum() / (labels != -100).sum()

Logits are float32, bfloat16 or float16, scores float32; a probability below 2^-126 counts as 0.  The calls enqueue on torch's current stream and return.
Calls on CPU tensors are staged through the GPU, as the multiply's are.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from ._dense import _require_gpu, check_dtype, check_int32, rows_view

__all__ = ["LabelScores", "label_log_probs"]


class LabelScores(NamedTuple):
    """What ``label_log_probs`` returns; parts that were not asked for are None.  ``logp`` and ``entropy`` have the
    shape of the logits without the classes, ``top_logp`` and ``top_index`` (int64) one dimension of ``top`` more."""
    logp: Optional[torch.Tensor]
    entropy: Optional[torch.Tensor]
    top_logp: Optional[torch.Tensor]
    top_index: Optional[torch.Tensor]


def label_log_probs(logits, labels=None, *, entropy=False, top=0, ignore_index=-100) -> LabelScores:
    """Scores of ``softmax(logits)`` along the last dimension, differentiable in the logits.

    labels (int64 or int32, the logits' shape without the classes): ``logp`` is the log probability of each; 0,
    without a gradient, where the label is ``ignore_index``; NaN (its gradient too) where it is any other number
    outside the classes.  None: no ``logp``.  entropy: -sum p log p.  top (at most 32 and the number of
    classes): the likeliest classes and their log probabilities, descending, equal logits by ascending class; a
    NaN counts as the largest.

    A row of -inf alone has log probabilities -inf, entropy 0 and no gradient; a NaN or +inf makes the scores of
    its row NaN, and their gradients.  A row whose label is ignored may hold either: it scores 0, and its gradient is 0
    where that of its entropy and of its likeliest classes is.  Logits need unit stride along the classes, rows may be
    any stride apart."""
    check_dtype(logits, "logits")
    z = rows_view(logits, "logits")
    rows, classes = z.shape
    top, ignore_index = int(top), int(ignore_index)
    if classes < 1:
        raise ValueError("logits have no classes")
    if not 0 <= top <= min(_lib.CBM_LABELS_MAX_TOP, classes):
        raise ValueError(f"top must be between 0 and {min(_lib.CBM_LABELS_MAX_TOP, classes)}, got {top}")
    check_int32(rows, "rows of logits")
    if classes > _lib.CBM_LABELS_MAX_CLASSES:
        raise ValueError(f"{classes} classes: at most {_lib.CBM_LABELS_MAX_CLASSES}")
    lead = logits.shape[:-1]
    if labels is not None:
        if not isinstance(labels, torch.Tensor):
            raise TypeError("labels must be a torch.Tensor")
        if labels.dtype not in (torch.int64, torch.int32):
            raise RuntimeError("labels tensor (NOT torch::kInt64 or kInt32)")
        if labels.shape != lead:
            raise ValueError(f"labels have shape {tuple(labels.shape)}, the logits' rows {tuple(lead)}")
        if labels.device != logits.device:
            raise ValueError("labels and logits are on different devices")
    if labels is None and not entropy and not top:
        raise ValueError("nothing asked for: give labels, entropy=True or top > 0")
    _require_gpu()
    if not logits.is_cuda:
        r = label_log_probs(logits.to("cuda"), None if labels is None else labels.to("cuda"), entropy=entropy, top=top,
                            ignore_index=ignore_index)
        return LabelScores(*(None if t is None else t.to(logits.device) for t in r))
    if labels is not None:
        if labels.dtype != torch.int64 or labels.dim() != 1 or not labels.is_contiguous():
            labels = labels.reshape(rows).to(torch.int64).contiguous()
    parts = _lib.autograd_lib().label_scores(z, labels, bool(entropy), top, ignore_index)
    if logits.dim() != 2:
        parts = tuple(None if t is None else t.reshape((*lead, *t.shape[1:])) for t in parts)
    return LabelScores(*parts)
