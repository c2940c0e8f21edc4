"""What the dense operators (``norm``, ``labels``, ``optim``) share: element types, layout checks, launches."""
from __future__ import annotations

import torch

from .cbm import _require_gpu, _stream  # noqa: F401  (the streams and the no-GPU error are the multiply's)

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def check_dtype(t, name):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in DTYPES:
        raise RuntimeError(f"{name} tensor (NOT torch::kFloat32, kBFloat16 or kHalf)")


def check_int32(value, what):
    if value > 0x7FFFFFFF:
        raise ValueError(f"{what}: {value} is more than the kernels index with 32 bits")


def rows_view(t, name):
    """``t`` as a matrix [rows, width] with unit column stride, without a copy; ValueError where its
    strides do not allow one."""
    if t.dim() < 1:
        raise ValueError(f"{name} must have at least one dimension")
    width = t.size(-1)
    if width > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have unit stride along its last dimension")
    if t.dim() == 2:
        m = t
    elif t.dim() == 1:
        m = t[None]
    else:
        try:
            m = t.view(-1, width)
        except RuntimeError:
            raise ValueError(f"{name}: the dimensions before the last must collapse into rows of one stride") from None
    if m.size(0) > 1 and m.stride(0) < width:
        raise ValueError(f"{name} has overlapping rows (stride {m.stride(0)} < width {width})")
    return m


def ld(t):
    return t.stride(0) if t.size(0) > 1 else max(t.size(1), 1)


def ptr(t):
    return t.data_ptr() if t is not None else None


def on_device(device):
    """Context that makes ``device`` current; free where it already is."""
    return _Here if device.index is None or device.index == torch.cuda.current_device() else torch.cuda.device(device)


class _Nothing:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_Here = _Nothing()
