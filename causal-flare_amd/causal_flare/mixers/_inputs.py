"""Argument checks and layouts shared by the token mixers."""
from __future__ import annotations

import contextlib
import ctypes

import torch

from .. import _lib


def _check_device(name, **tensors):
    """Every tensor on one GPU, that of the first."""
    device = None
    for what, t in tensors.items():
        if t is None:
            continue
        if t.device.type != "cuda":
            raise RuntimeError(f"{name} requires GPU tensors (got {what} on {t.device}).")
        if device is None:
            device = t.device
        elif t.device != device:
            raise ValueError(f"{name} expects every tensor on {device}. Got {what} on {t.device}")
    return device


def _check_float(name, **tensors):
    for what, t in tensors.items():
        if t is not None and not t.dtype.is_floating_point:
            raise ValueError(f"{name} expects floating-point tensors. Got {what} of {t.dtype}")


def _check_shape(name, what, t, shape):
    if t is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} expects {what} {list(shape)}. Got {tuple(t.shape)}")


def _check_integers(name, what, t, shape):
    if t is None:
        return
    _check_shape(name, what, t, shape)
    if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype is torch.bool:
        raise ValueError(f"{name} expects integers in {what}. Got {t.dtype}")


def _int32(t):
    if t is None or (t.dtype is torch.int32 and t.is_contiguous()):
        return t
    return t.to(torch.int32).contiguous()


def _f32(t):
    if t is None or (t.dtype is torch.float32 and t.is_contiguous()):
        return t
    return t.detach().to(torch.float32).contiguous()


def _row_mask(name, mask, B, device):
    """A decode's mask of rows, [B] or [B, 1]: int32 [B] (0: the row sits out)."""
    if mask is None:
        return None
    if mask.dim() == 2 and mask.shape[1] == 1:
        mask = mask[:, 0]
    if mask.dim() != 1 or mask.shape[0] != B:
        raise ValueError(f"{name} attention_mask must be [B] or [B, 1]. Got {tuple(mask.shape)}")
    return (mask != 0).to(device=device, dtype=torch.int32).contiguous()


def _rows(t, dtype):
    """`t` [B, n, ..] in `dtype` with its last dimension adjacent in memory, and tokens less than 2^22
    elements apart; other strides stay."""
    if t is None:
        return None
    if t.dtype is not dtype:
        t = t.detach().to(dtype)
    if (t.shape[-1] <= 1 or t.stride(-1) == 1) and t.stride(1) < 1 << 22:
        return t
    return t.detach().clone(memory_format=torch.contiguous_format)


def _aligned_rows(t, dtype):
    """`_rows` with every row on a 16-byte boundary."""
    t = _rows(t, dtype)
    size = t.element_size()
    if t.data_ptr() % 16 or any(s * size % 16 for s in t.stride()[:-1]) or t.stride(-1) != 1:
        t = t.detach().clone(memory_format=torch.contiguous_format)
    return t


def _strides(*values):
    return (ctypes.c_int64 * len(values))(*values)


def _on(device):
    """The kernels' device as the current one."""
    if torch.cuda.current_device() == device.index:
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _training(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# Single tokens: the call's host work counts, and these look at what the common call needs to
# hold, with no messages; where it does not, the caller takes the general path with its checks.
_CODES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _plain_f32(t, device, *shape):
    return t is None or (t.dtype is torch.float32 and t.shape == shape and t.device == device and t.is_contiguous())


def _raw_stream(index):
    return torch._C._cuda_getCurrentRawStream(index)


def _ptr(t):
    return None if t is None else t.data_ptr()
