"""Short causal convolution over the tokens, one filter a channel.

    pre_t = bias + sum_{k < W} weight[:, W - 1 - k] * x_{t-k}        y_t = pre_t or silu(pre_t)

Layouts: x [B, N, C], weight [C, W] (W of 2, 3 or 4; the last column meets the token itself),
bias [C], y [B, N, C].  x may be a slice of a wider tensor: its last dimension has to be
adjacent in memory, and anything else is copied.  x may be float32, bfloat16 or float16 (float64 is
computed in float32); weight and bias are used in float32 and sums are kept in float32.

A cache is ``{"window": [B, W - 1, C]}``, the last inputs in x's type, oldest first.
"""
from __future__ import annotations

import torch
import torch.autograd as autograd
from torch.autograd.function import once_differentiable

from .. import _lib
from .._common import _compute_dtype
from ._inputs import (
    _CODES,
    _check_device,
    _check_float,
    _check_integers,
    _check_shape,
    _f32,
    _int32,
    _on,
    _plain_f32,
    _ptr,
    _raw_stream,
    _row_mask,
    _rows,
)


def _check(name, x, weight, bias, activation):
    if x.dim() != 3:
        raise ValueError(f"{name} expects x [B, N, C]. Got {tuple(x.shape)}")
    B, N, C = x.shape
    if weight.dim() != 2 or weight.shape[0] != C:
        raise ValueError(f"{name} expects weight [C, W] with C={C}. Got {tuple(weight.shape)}")
    if weight.shape[1] not in (2, 3, 4):
        raise ValueError(f"{name} supports filters of 2, 3 or 4 tokens. Got W={weight.shape[1]}")
    _check_shape(name, "bias", bias, (C,))
    if activation not in (None, "silu"):
        raise ValueError(f"{name} expects activation None or 'silu'. Got {activation!r}")
    _check_float(name, x=x, weight=weight, bias=bias)


def _window(name, state, B, W, C, dtype, device):
    if not isinstance(state, dict) or "window" not in state:
        raise ValueError(f"{name} expects a state {{'window': [B, W - 1, C]}}. Got {state!r:.80}")
    _check_shape(name, "state['window']", state["window"], (B, W - 1, C))
    return state["window"].to(device=device, dtype=dtype).contiguous()


def _run(x, weight, bias, activation, document_ids=None, lengths=None, window=None, window_out=None):
    B, N, C = x.shape
    dtype = _compute_dtype(x)
    xr, w, b = _rows(x, dtype), _f32(weight), _f32(bias)
    ids, lens = _int32(document_ids), _int32(lengths)
    y = torch.empty((B, N, C), device=x.device, dtype=dtype)
    P = _ptr
    with _on(x.device):
        rc = _lib.lib().flare_conv_forward(
            P(xr), xr.stride(0), xr.stride(1), P(w), P(b), int(activation == "silu"), _lib.dtype_code(dtype), B, N, C,
            weight.shape[1], P(ids), P(lens), P(window), P(y), P(window_out), _raw_stream(x.device.index))
    _lib.check(rc, "flare_conv_forward")
    return y


class ShortConvolution(autograd.Function):
    """The convolution over whole sequences, with gradients for x, weight and bias."""

    @staticmethod
    def forward(ctx, x, weight, bias, activation, document_ids):
        ctx.save_for_backward(x, weight, bias, document_ids)
        ctx.activation = activation
        if x.numel() == 0:
            return torch.empty_like(x)
        return _run(x, weight, bias, activation, document_ids).to(x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, document_ids = ctx.saved_tensors
        if x.numel() == 0:
            return tuple(None if t is None else torch.zeros_like(t) for t in (x, weight, bias)) + (None, None)
        B, N, C = x.shape
        W = weight.shape[1]
        dtype = _compute_dtype(x)
        xr, w, b, ids = _rows(x, dtype), _f32(weight), _f32(bias), _int32(document_ids)
        g = dy.to(dtype).contiguous()
        dx = torch.empty((B, N, C), device=x.device, dtype=dtype)
        dw = torch.empty((C, W), device=x.device, dtype=torch.float32)
        db = None if bias is None else torch.empty((C,), device=x.device, dtype=torch.float32)
        lib = _lib.lib()
        nbytes = lib.flare_conv_backward_workspace_size(B, N, C, W)
        ws = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
        P = _ptr
        with _on(x.device):
            rc = lib.flare_conv_backward(
                P(xr), xr.stride(0), xr.stride(1), P(w), P(b), int(ctx.activation == "silu"), _lib.dtype_code(dtype),
                B, N, C, W, P(ids), P(g), P(dx), P(dw), P(db), P(ws), nbytes, _raw_stream(x.device.index))
        _lib.check(rc, "flare_conv_backward")
        return dx.to(x.dtype), dw.to(weight.dtype), None if bias is None else db.to(bias.dtype), None, None


def short_convolution(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    activation: str | None = None,
    document_ids: torch.Tensor | None = None,
):
    """Short causal convolution of whole sequences, differentiable in x, weight and bias.

    document_ids: integers [B, N].  A token sees back to where its run of equal ids begins, and
    no further; a token of a negative id is padding, with y = 0 and no gradient.
    """
    name = "short_convolution"
    _check(name, x, weight, bias, activation)
    _check_integers(name, "document_ids", document_ids, x.shape[:2])
    _check_device(name, x=x, weight=weight, bias=bias, document_ids=document_ids)
    return ShortConvolution.apply(x, weight, bias, activation, document_ids)


def short_convolution_prefill(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    activation: str | None = None,
    state: dict[str, torch.Tensor] | None = None,
    lengths: torch.Tensor | None = None,
):
    """Prompts that continue `state` (None: nothing before them): (y, new state).

    lengths: integers [B], each sequence's real tokens (all N by default; taken as 0 or N where
    they lie outside that).  Rows behind them give y = 0 and do not enter the new state.  The
    input state is left as it is.
    """
    name = "short_convolution_prefill"
    _check(name, x, weight, bias, activation)
    B, N, C = x.shape
    _check_integers(name, "lengths", lengths, (B,))
    _check_device(name, x=x, weight=weight, bias=bias, lengths=lengths)
    W, dtype = weight.shape[1], _compute_dtype(x)
    window = None if state is None else _window(name, state, B, W, C, dtype, x.device)
    if x.numel() == 0:
        new = torch.zeros((B, W - 1, C), device=x.device, dtype=dtype) if window is None else window.clone()
        return torch.empty_like(x, requires_grad=False), {"window": new.to(x.dtype)}
    new = torch.empty((B, W - 1, C), device=x.device, dtype=dtype)
    y = _run(x, weight, bias, activation, lengths=lengths, window=window, window_out=new)
    return y.to(x.dtype), {"window": new.to(x.dtype)}


def _step_fast(x, weight, bias, activation, state):
    """The common call, or None: x [B, C] or [B, 1, C] of the window's type, fp32 weights."""
    if x.dim() == 3 and x.shape[1] == 1:
        B, _, C = x.shape
    elif x.dim() == 2:
        B, C = x.shape
    else:
        return None
    device, code = x.device, _CODES.get(x.dtype)
    if code is None or not B * C or device.type != "cuda" or device.index != torch.cuda.current_device():
        return None
    W = weight.shape[-1]
    window = state.get("window") if isinstance(state, dict) else None
    if (activation not in (None, "silu") or W not in (2, 3, 4) or (C > 1 and x.stride(-1) != 1)
            or not _plain_f32(weight, device, C, W) or not _plain_f32(bias, device, C) or window is None
            or window.dtype is not x.dtype or window.shape != (B, W - 1, C) or window.device != device
            or not window.is_contiguous()):
        return None
    y = torch.empty((B, 1, C), device=device, dtype=x.dtype)
    _lib.check(_lib.lib().flare_conv_step(
        x.data_ptr(), x.stride(0), weight.data_ptr(), _ptr(bias), 1 if activation else 0, code, B, C, W, None,
        window.data_ptr(), y.data_ptr(), _raw_stream(device.index)), "flare_conv_step")
    return y, {"window": window}


def short_convolution_decode(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    activation: str | None = None,
    state: dict[str, torch.Tensor] | None = None,
    attention_mask: torch.Tensor | None = None,
):
    """One token a sequence, x [B, C] or [B, 1, C]: (y [B, 1, C], state).

    A contiguous window of x's type is updated in place and returned.  attention_mask [B] or
    [B, 1]: a row of 0 keeps its window and gets y = 0.
    """
    name = "short_convolution_decode"
    if attention_mask is None and state is not None:
        out = _step_fast(x, weight, bias, activation, state)
        if out is not None:
            return out
    if x.dim() == 2:
        x = x[:, None]
    _check(name, x, weight, bias, activation)
    if x.shape[1] != 1:
        raise ValueError(f"{name} expects x [B, C] or [B, 1, C]. Got {tuple(x.shape)}")
    B, _, C = x.shape
    device = _check_device(name, x=x, weight=weight, bias=bias)
    mask = _row_mask(name, attention_mask, B, device)
    W, dtype = weight.shape[1], _compute_dtype(x)
    if state is None:
        window = torch.zeros((B, W - 1, C), device=device, dtype=dtype)
    else:
        window = _window(name, state, B, W, C, dtype, device)
    xr, w, b = _rows(x, dtype), _f32(weight), _f32(bias)
    y = torch.empty((B, 1, C), device=device, dtype=dtype)
    if y.numel() == 0:
        return y.to(x.dtype), {"window": window}
    P = _ptr
    with _on(device):
        rc = _lib.lib().flare_conv_step(P(xr), xr.stride(0), P(w), P(b), int(activation == "silu"),
                                        _lib.dtype_code(dtype), B, C, W, P(mask), P(window), P(y),
                                        _raw_stream(device.index))
    _lib.check(rc, "flare_conv_step")
    return y.to(x.dtype), {"window": window}
