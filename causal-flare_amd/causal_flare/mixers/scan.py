"""Selective state space scan.

    delta_t = dt_t + dt_bias, or softplus of it
    h_t     = exp(delta_t A) h_{t-1} + delta_t x_t B_t          [C, S]
    y_t     = (sum_s C_t h_t + D x_t) silu(z_t)                 [C]

Layouts: x, dt, z [B, N, C]; A [C, S] (1 to 64 states a channel); B, C [B, N, S], or [B, N, G, S]
where channel c reads group c // (C / G); D, dt_bias [C].  x, dt, z, B and C may be slices of
wider tensors: the last dimension has to be adjacent in memory, and anything else is copied.
They may be float32, bfloat16 or float16 (one type: their promotion; float64 is computed in
float32); A, D and dt_bias are used
in float32, and so are states, decays and sums.

A cache is ``{"h": [B, C, S]}`` in float32.
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
    _strides,
    _training,
)

_MAX_STATES = 64


def _check(name, x, dt, A, B, C, D, z, dt_bias):
    """(batch, tokens, channels, states, groups) of checked inputs."""
    if x.dim() != 3:
        raise ValueError(f"{name} expects x [B, N, C]. Got {tuple(x.shape)}")
    nb, n, c = x.shape
    _check_shape(name, "dt", dt, x.shape)
    _check_shape(name, "z", z, x.shape)
    if A.dim() != 2 or A.shape[0] != c:
        raise ValueError(f"{name} expects A [C, S] with C={c}. Got {tuple(A.shape)}")
    s = A.shape[1]
    if not 1 <= s <= _MAX_STATES:
        raise ValueError(f"{name} supports 1 to {_MAX_STATES} states a channel. Got S={s}")
    if B.dim() not in (3, 4) or tuple(B.shape[:2]) != (nb, n) or B.shape[-1] != s:
        raise ValueError(f"{name} expects B [B, N, S] or [B, N, G, S] with B={nb}, N={n}, S={s}. Got {tuple(B.shape)}")
    g = B.shape[2] if B.dim() == 4 else 1
    _check_shape(name, "C", C, B.shape)
    if g < 1 or c % g:
        raise ValueError(f"{name} expects channels that divide into the groups of B and C. Got C={c}, G={g}")
    _check_shape(name, "D", D, (c,))
    _check_shape(name, "dt_bias", dt_bias, (c,))
    _check_float(name, x=x, dt=dt, A=A, B=B, C=C, D=D, z=z, dt_bias=dt_bias)
    return nb, n, c, s, g


class _Inputs:
    """The tensors as the kernels take them, and the strides that go with them."""

    def __init__(self, x, dt, A, B, C, D, z, dt_bias):
        self.dtype = _compute_dtype(x, dt, B, C, z)
        self.x, self.dt, self.z = (_rows(t, self.dtype) for t in (x, dt, z))
        self.B, self.C = (_rows(t if t.dim() == 4 else t[:, :, None], self.dtype) for t in (B, C))
        self.A, self.D, self.dt_bias = _f32(A), _f32(D), _f32(dt_bias)
        zs = (0, 0) if z is None else (self.z.stride(0), self.z.stride(1))
        self.strides = _strides(self.x.stride(0), self.x.stride(1), self.dt.stride(0), self.dt.stride(1), *zs,
                                *self.B.stride()[:3], *self.C.stride()[:3])

    def pointers(self):
        P = _ptr
        return P(self.x), P(self.dt), P(self.A), P(self.B), P(self.C), P(self.D), P(self.z), P(self.dt_bias)


def _padded(S):
    return 8 if S <= 8 else 16 if S <= 16 else 32 if S <= 32 else 64


def _run(x, dt, A, B, C, D, z, dt_bias, dt_softplus, sizes, training, document_ids=None, lengths=None, h0=None,
         h_fin=None):
    """(y, the states kept for the backward or None, the chunk length)."""
    nb, n, c, s, g = sizes
    t = _Inputs(x, dt, A, B, C, D, z, dt_bias)
    lib = _lib.lib()
    chunk = int(lib.flare_scan_chunk(nb, n, c, s, g, int(training)))
    kept = None
    if training:
        kept = torch.empty((nb, -(-n // int(lib.flare_scan_kept_tokens(s))), _padded(s), c), device=x.device,
                           dtype=torch.float32)
    nbytes = lib.flare_scan_forward_workspace_size(nb, n, c, s, g, chunk)
    ws = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
    y = torch.empty((nb, n, c), device=x.device, dtype=t.dtype)
    ids, lens = _int32(document_ids), _int32(lengths)
    P = _ptr
    with _on(x.device):
        rc = lib.flare_scan_forward(*t.pointers(), int(bool(dt_softplus)), _lib.dtype_code(t.dtype), nb, n, c, s, g,
                                    t.strides, P(ids), P(lens), P(h0), P(y), P(h_fin), chunk, P(kept), P(ws),
                                    nbytes, _raw_stream(x.device.index))
    _lib.check(rc, "flare_scan_forward")
    return y, kept, chunk


class StateSpaceScan(autograd.Function):
    """The scan over whole sequences, with gradients for every floating-point input."""

    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, dt_softplus, document_ids, sizes, training):
        ctx.sizes, ctx.softplus, ctx.chunk = sizes, dt_softplus, 0
        if x.numel() == 0:
            ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, document_ids, None)
            return torch.empty_like(x)
        y, kept, ctx.chunk = _run(x, dt, A, B, C, D, z, dt_bias, dt_softplus, sizes, training, document_ids)
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, document_ids, kept)
        return y.to(x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, dt, A, B, C, D, z, dt_bias, document_ids, kept = ctx.saved_tensors
        leaves = (x, dt, A, B, C, D, z, dt_bias)
        if x.numel() == 0:
            return tuple(None if t is None else torch.zeros_like(t) for t in leaves) + (None,) * 4
        nb, n, c, s, g = ctx.sizes
        t = _Inputs(*leaves)
        device, f32 = x.device, torch.float32
        gy = dy.to(t.dtype).contiguous()

        def empty(*shape, dtype=t.dtype):
            return torch.empty(shape, device=device, dtype=dtype)

        dx, ddt, dB, dC = empty(nb, n, c), empty(nb, n, c), empty(nb, n, g, s), empty(nb, n, g, s)
        dA = empty(c, s, dtype=f32)
        dz = None if z is None else empty(nb, n, c)
        dD = None if D is None else empty(c, dtype=f32)
        dbias = None if dt_bias is None else empty(c, dtype=f32)
        ids = _int32(document_ids)
        lib = _lib.lib()
        nbytes = lib.flare_scan_backward_workspace_size(nb, n, c, s, g, ctx.chunk)
        ws = torch.empty(nbytes, device=device, dtype=torch.uint8)
        P = _ptr
        with _on(device):
            rc = lib.flare_scan_backward(*t.pointers(), int(bool(ctx.softplus)), _lib.dtype_code(t.dtype), nb, n, c, s,
                                         g, t.strides, P(ids), P(gy), ctx.chunk, P(kept), P(dx), P(ddt), P(dA),
                                         P(dB), P(dC), P(dD), P(dz), P(dbias), P(ws), nbytes, _raw_stream(device.index))
        _lib.check(rc, "flare_scan_backward")
        grads = (dx, ddt, dA, dB.view(B.shape), dC.view(C.shape), dD, dz, dbias)
        return tuple(None if d is None else d.to(ref.dtype) for d, ref in zip(grads, leaves)) + (None,) * 4


def _state(name, state, nb, c, s, device):
    if not isinstance(state, dict) or "h" not in state:
        raise ValueError(f"{name} expects a state {{'h': [B, C, S]}}. Got {state!r:.80}")
    _check_shape(name, "state['h']", state["h"], (nb, c, s))
    return state["h"].to(device=device, dtype=torch.float32).contiguous()


def state_space_scan(
    x: torch.Tensor,
    dt: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: torch.Tensor | None = None,
    z: torch.Tensor | None = None,
    dt_bias: torch.Tensor | None = None,
    dt_softplus: bool = False,
    document_ids: torch.Tensor | None = None,
):
    """Selective scan of whole sequences from h = 0, differentiable in every floating-point input.

    document_ids: integers [B, N].  The state starts from 0 where an id differs from the one
    before; a token of a negative id is padding, with y = 0 and no gradient.
    """
    name = "state_space_scan"
    sizes = _check(name, x, dt, A, B, C, D, z, dt_bias)
    _check_integers(name, "document_ids", document_ids, x.shape[:2])
    _check_device(name, x=x, dt=dt, A=A, B=B, C=C, D=D, z=z, dt_bias=dt_bias, document_ids=document_ids)
    return StateSpaceScan.apply(x, dt, A, B, C, D, z, dt_bias, dt_softplus, document_ids, sizes,
                                _training(x, dt, A, B, C, D, z, dt_bias))


def state_space_scan_prefill(
    x: torch.Tensor,
    dt: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: torch.Tensor | None = None,
    z: torch.Tensor | None = None,
    dt_bias: torch.Tensor | None = None,
    dt_softplus: bool = False,
    state: dict[str, torch.Tensor] | None = None,
    lengths: torch.Tensor | None = None,
):
    """Prompts that continue `state` (None: h = 0): (y, new state).

    lengths: integers [B], each sequence's real tokens (all N by default; taken as 0 or N where
    they lie outside that).  Rows behind them give y = 0 and leave the state alone.  The input
    state is left as it is.
    """
    name = "state_space_scan_prefill"
    sizes = nb, n, c, s, g = _check(name, x, dt, A, B, C, D, z, dt_bias)
    _check_integers(name, "lengths", lengths, (nb,))
    device = _check_device(name, x=x, dt=dt, A=A, B=B, C=C, D=D, z=z, dt_bias=dt_bias, lengths=lengths)
    h0 = None if state is None else _state(name, state, nb, c, s, device)
    if x.numel() == 0:
        h = torch.zeros((nb, c, s), device=device) if h0 is None else h0.clone()
        return torch.empty_like(x, requires_grad=False), {"h": h}
    h = torch.empty((nb, c, s), device=device, dtype=torch.float32)
    y, _, _ = _run(x, dt, A, B, C, D, z, dt_bias, dt_softplus, sizes, False, lengths=lengths, h0=h0, h_fin=h)
    return y.to(x.dtype), {"h": h}


def _step_fast(x, dt, A, B, C, D, z, dt_bias, softplus, state):
    """The common call, or None: one type for x, dt, z, B and C, fp32 parameters and state."""
    token = x.dim() == 3
    if x.dim() not in (2, 3) or (token and x.shape[1] != 1) or A.dim() != 2:
        return None
    nb, c, s = x.shape[0], x.shape[-1], A.shape[1]
    dtype, device = x.dtype, x.device
    code = _CODES.get(dtype)
    if (code is None or not nb * c or not 1 <= s <= _MAX_STATES or device.type != "cuda"
            or device.index != torch.cuda.current_device()):
        return None
    grouped = B.dim() == x.dim() + 1
    g = B.shape[-2] if grouped else 1
    want = (nb, 1) if token else (nb,)
    want = want + (g, s) if grouped else want + (s,)
    if B.dim() != len(want) or B.shape != want or C.shape != want or g < 1 or c % g:
        return None
    for t, n in ((x, c), (dt, c), (z, c), (B, s), (C, s)):
        if t is not None and (t.dtype is not dtype or t.device != device or (n > 1 and t.stride(-1) != 1)):
            return None
    h = state.get("h") if isinstance(state, dict) else None
    if (dt.shape != x.shape or (z is not None and z.shape != x.shape) or not _plain_f32(A, device, c, s)
            or not _plain_f32(D, device, c) or not _plain_f32(dt_bias, device, c) or h is None
            or not _plain_f32(h, device, nb, c, s)):
        return None
    strides = _strides(x.stride(0), 0, dt.stride(0), 0, 0 if z is None else z.stride(0), 0, B.stride(0), 0,
                       B.stride(-2) if grouped else 0, C.stride(0), 0, C.stride(-2) if grouped else 0)
    y = torch.empty((nb, 1, c), device=device, dtype=dtype)
    _lib.check(_lib.lib().flare_scan_step(
        x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(), _ptr(D), _ptr(z), _ptr(dt_bias),
        1 if softplus else 0, code, nb, c, s, g, strides, None, h.data_ptr(), y.data_ptr(),
        _raw_stream(device.index)), "flare_scan_step")
    return y, {"h": h}


def state_space_scan_decode(
    x: torch.Tensor,
    dt: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: torch.Tensor | None = None,
    z: torch.Tensor | None = None,
    dt_bias: torch.Tensor | None = None,
    dt_softplus: bool = False,
    state: dict[str, torch.Tensor] | None = None,
    attention_mask: torch.Tensor | None = None,
):
    """One token a sequence: (y [B, 1, C], state).

    x, dt, z [B, 1, C] and B, C [B, 1, S] or [B, 1, G, S], or all of them without the dimension
    of the token (B and C then [B, S] or [B, G, S]).  A contiguous float32 state is updated in
    place and returned.  attention_mask [B] or [B, 1]: a row of 0 keeps its state and gets y = 0.
    """
    name = "state_space_scan_decode"
    if attention_mask is None and state is not None:
        out = _step_fast(x, dt, A, B, C, D, z, dt_bias, dt_softplus, state)
        if out is not None:
            return out
    if x.dim() == 2:
        x, dt, B, C = x[:, None], dt[:, None], B[:, None], C[:, None]
        z = None if z is None else z[:, None]
    nb, n, c, s, g = _check(name, x, dt, A, B, C, D, z, dt_bias)
    if n != 1:
        raise ValueError(f"{name} expects one token a sequence. Got x {tuple(x.shape)}")
    device = _check_device(name, x=x, dt=dt, A=A, B=B, C=C, D=D, z=z, dt_bias=dt_bias)
    mask = _row_mask(name, attention_mask, nb, device)
    if state is None:
        h = torch.zeros((nb, c, s), device=device, dtype=torch.float32)
    else:
        h = _state(name, state, nb, c, s, device)
    t = _Inputs(x, dt, A, B, C, D, z, dt_bias)
    y = torch.empty((nb, 1, c), device=device, dtype=t.dtype)
    if y.numel() == 0:
        return y.to(x.dtype), {"h": h}
    P = _ptr
    with _on(device):
        rc = _lib.lib().flare_scan_step(*t.pointers(), int(bool(dt_softplus)), _lib.dtype_code(t.dtype), nb, c, s, g,
                                        t.strides, P(mask), P(h), P(y), _raw_stream(device.index))
    _lib.check(rc, "flare_scan_step")
    return y.to(x.dtype), {"h": h}
