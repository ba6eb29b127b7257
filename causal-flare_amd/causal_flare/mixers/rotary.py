"""Rotary positions of queries and keys, for softmax attention beside or in place of its bias on distance.

Pair i of a head's first R dimensions, (a, b), is turned by the angle position * frequencies[i]:

    (a, b) -> (a cos - b sin, a sin + b cos)

The pairs are dimensions i and i + R / 2, or 2i and 2i + 1 (`interleaved`); dimensions from R on stay
as they are.  Angles are exact to some 1e-9 of a radian, however far the position; sines, cosines and products are
taken in float32 and rounded once.
"""
from __future__ import annotations

import math

import torch
import torch.autograd as autograd
import torch.autograd.forward_ad as forward_ad
from torch.autograd.function import once_differentiable

from .. import _lib
from .._common import _compute_dtype
from ._inputs import (
    _CODES,
    _check_device,
    _check_float,
    _check_integers,
    _int32,
    _on,
    _ptr,
    _raw_stream,
    _rows,
    _strides,
    _training,
)


def rotary_frequencies(
    dim: int,
    base: float = 10000.0,
    factor: float = 1.0,
    original_length: float | None = None,
    low_turns: float = 1.0,
    high_turns: float = 32.0,
) -> torch.Tensor:
    """Radians a token of each pair, float64 [dim / 2] on the host: base^(-2 i / dim), for contexts `factor`
    times as long.

    Without original_length all frequencies are divided by factor.  With it, those that make at least
    high_turns turns over so many tokens stay as they are, those of low_turns and fewer are divided by factor,
    and those between are mixed, linearly in the turns.
    """
    if dim < 2 or dim % 2:
        raise ValueError(f"rotary_frequencies expects an even number of dimensions. Got {dim}")
    if not (0 < base < math.inf and 0 < factor < math.inf):
        raise ValueError(f"rotary_frequencies expects positive base and factor. Got {base!r}, {factor!r}")
    f = float(base) ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if original_length is None:
        return f / factor
    if not (0 < original_length < math.inf and low_turns < high_turns):
        raise ValueError("rotary_frequencies expects a positive original_length and low_turns below high_turns. "
                         f"Got {original_length!r}, {low_turns!r}, {high_turns!r}")
    keep = ((original_length * f / (2 * math.pi) - low_turns) / (high_turns - low_turns)).clamp(0, 1)
    return f * (keep + (1 - keep) / factor)


def _launch(q, k, dtype, frequencies, positions, lengths, interleaved, inverse):
    """Rows that the kernel reads in place, [B, N, heads, D] or one token's [B, heads, D], of `dtype`, turned."""
    shape, step, G, to = q.shape, (0, 0), 0, None
    if len(shape) == 4:
        step = (q.stride(1), 0 if k is None else k.stride(1))
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    strides = (q.stride(0), step[0], q.stride(-2))
    if k is None:
        strides += (0, 0, 0)
    else:
        G, to = k.shape[-2], torch.empty_like(k, memory_format=torch.contiguous_format)
        strides += (k.stride(0), step[1], k.stride(-2))
    rc = _lib.lib().flare_rotary(
        q.data_ptr(), _ptr(k), _strides(*strides), _CODES[dtype], shape[0], shape[1] if len(shape) == 4 else 1, shape[-2], G,
        shape[-1], 2 * frequencies.shape[0], frequencies.data_ptr(), _ptr(positions), _ptr(lengths), int(interleaved),
        int(inverse), out.data_ptr(), _ptr(to), _raw_stream(q.device.index))
    if rc:
        _lib.check(rc, "flare_rotary")
    return out, to


def _turn(q, k, frequencies, positions, lengths, interleaved, inverse):
    """The pairs of q [B, N, H, D] and k [B, N, G, D] (or None) turned; each keeps its type."""
    dtype = q.dtype
    if (k is not None and dtype in _CODES and k.dtype is dtype and q.stride(-1) == 1 and k.stride(-1) == 1
            and q.device.index == torch.cuda.current_device()):
        return _launch(q, k, dtype, frequencies, positions, lengths, interleaved, inverse)
    dtype = _compute_dtype(q, k)
    with _on(q.device):
        y, z = _launch(_rows(q, dtype), _rows(k, dtype), dtype, frequencies, positions, lengths, interleaved, inverse)
    return y if q.dtype is dtype else y.to(q.dtype), z if k is None or k.dtype is dtype else z.to(k.dtype)


def _plain(Q, K, frequencies, positions, lengths):
    """Whether this is the common call: Q and K of one type on the current device, rows that the kernel reads in place,
    int32 positions or lengths, and no tangents, which `RotaryPositions` has none for and refuses."""
    if K is None or forward_ad._current_level >= 0:
        return False
    dtype, device, shape, keys = Q.dtype, Q.device, Q.shape, K.shape
    if (dtype not in _CODES or device.type != "cuda" or device.index != torch.cuda.current_device() or len(shape) not in (3, 4)
            or len(keys) != len(shape) or K.dtype is not dtype or K.device != device or Q.stride(-1) != 1
            or K.stride(-1) != 1 or not isinstance(frequencies, torch.Tensor)):
        return False
    D, G = shape[-1], keys[-2]
    if (keys != (shape[:-2] + (G, D)) or not Q.numel() or not G or frequencies.dtype is not torch.float64
            or frequencies.dim() != 1 or frequencies.device.type != "cpu" or not frequencies.is_contiguous()
            or frequencies.requires_grad):
        return False
    if not 2 <= 2 * frequencies.shape[0] <= D or D > 256 or (positions is not None and lengths is not None):
        return False
    if positions is not None:
        t, want = positions, (shape[0], shape[1] if len(shape) == 4 else 1)
    else:
        t, want = lengths, shape[:1]
    return t is None or (isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.shape == want and t.device == device
                         and t.is_contiguous())


class RotaryPositions(autograd.Function):
    """Turned queries and keys; their gradients are turned back."""

    @staticmethod
    def forward(ctx, Q, K, frequencies, positions, lengths, interleaved):
        ctx.save_for_backward(frequencies, positions, lengths)
        ctx.options = (interleaved, K is not None)
        q, k = _turn(Q, K, frequencies, positions, lengths, interleaved, False)
        return q if k is None else (q, k)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        frequencies, positions, lengths = ctx.saved_tensors
        interleaved, keys = ctx.options
        need_q, need_k = ctx.needs_input_grad[0], keys and ctx.needs_input_grad[1]
        dq, dk = None, None
        if need_q:
            dq, dk = _turn(grads[0], grads[1] if need_k else None, frequencies, positions, lengths, interleaved, True)
        elif need_k:
            dk, _ = _turn(grads[1], None, frequencies, positions, lengths, interleaved, True)
        return dq, dk, None, None, None, None


def rotary_positions(
    Q: torch.Tensor,
    K: torch.Tensor | None,
    frequencies: torch.Tensor,
    positions: torch.Tensor | None = None,
    lengths: torch.Tensor | None = None,
    interleaved: bool = False,
):
    """Q [B, N, H, D] and K [B, N, G, D] (or None) turned by their positions: (Q, K), or Q alone.

    Differentiable in Q and K, backwards (tangents are refused).  Single tokens may be given as [B, H, D] and
    [B, G, D].  frequencies: float64 [R / 2] on the host (`rotary_frequencies`), R up to D; the rest of a head
    stays as it is.  positions: integers [B, N] within 32 bits (of packed documents, say), any sign; or
    lengths: integers [B], the tokens that each sequence's cache holds already: token t is at position lengths[b] + t.
    Without either it is at t.  D up to 256.
    """
    name = "rotary_positions"
    if _plain(Q, K, frequencies, positions, lengths):
        if not _training(Q, K):
            return _launch(Q, K, Q.dtype, frequencies, positions, lengths, interleaved, False)
        if Q.dim() == 4:
            return RotaryPositions.apply(Q, K, frequencies, positions, lengths, interleaved)
    token = Q.dim() == 3
    if Q.dim() not in (3, 4) or (K is not None and K.dim() != Q.dim()):
        raise ValueError(f"{name} expects Q [B, N, H, D] and K [B, N, G, D], or without N. Got Q={tuple(Q.shape)}"
                         + ("" if K is None else f", K={tuple(K.shape)}"))
    if token:
        Q, K = Q[:, None], None if K is None else K[:, None]
    B, N, H, D = Q.shape
    if K is not None and (K.shape[:2] != Q.shape[:2] or K.shape[3] != D):
        raise ValueError(f"{name} expects K [B, N, G, D] with B={B}, N={N}, D={D}. Got {tuple(K.shape)}")
    if H < 1 or (K is not None and K.shape[2] < 1):
        raise ValueError(f"{name} expects heads. Got Q={tuple(Q.shape)}" + ("" if K is None else f", K={tuple(K.shape)}"))
    _check_float(name, Q=Q, K=K)
    if (not isinstance(frequencies, torch.Tensor) or frequencies.device.type != "cpu"
            or frequencies.dtype is not torch.float64 or frequencies.dim() != 1):
        raise ValueError(f"{name} expects frequencies as a float64 tensor [R / 2] on the host. Got {frequencies!r:.80}")
    if frequencies.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{name} has no gradient for frequencies; pass frequencies.detach()")
    R = 2 * frequencies.shape[0]
    if not 2 <= R <= D or D > 256:
        raise ValueError(f"{name} turns 2 to D dimensions of heads of up to 256. Got {R} of D={D}")
    _check_integers(name, "positions", positions, (B, N))
    _check_integers(name, "lengths", lengths, (B,))
    if positions is not None and lengths is not None:
        raise ValueError(f"{name} expects positions or lengths, not both")
    _check_device(name, Q=Q, K=K, positions=positions, lengths=lengths)
    if B * N == 0:
        out = Q.clone() if K is None else (Q.clone(), K.clone())
    else:
        out = RotaryPositions.apply(Q, K, frequencies.contiguous(), _int32(positions), _int32(lengths),
                                    bool(interleaved))
    if K is None:
        return out[:, 0] if token else out
    return (out[0][:, 0], out[1][:, 0]) if token else out
