"""Exact softmax attention with capped scores, a bias on distance, documents and prefixes.

    x_ij = scale q_i . k_j, or softcap tanh(scale q_i . k_j / softcap)
    s_ij = x_ij - slope_h |i - j|           y_i = sum_j softmax_j(s_ij) v_j

Query i sees key j if j <= i or j < prefix (all keys without `causal`), and if the two have the
same document id, not negative.  A query that sees nothing gives y = 0.

Layouts: Q [B, N, H, D], K and V [B, N, G, D] with H a multiple of G (head h reads key head
h // (H / G)), D a multiple of 16 up to 128.  Q, K and V may be slices of wider tensors: rows of
D adjacent elements on 16-byte boundaries are read in place, anything else is copied.  They may
be float32, bfloat16 or float16 (one type: their promotion; float64 is computed in float32).  Scores,
maxima and sums are kept in float32; 16-bit inputs have their weights rounded to their type for the
products with V and dY, and the scores' gradients in two parts for those with K and Q.  A call that is
to be differentiated keeps Q, K, V, y, a float32 a row of a head and, of 16-bit inputs, what y was
rounded by (as large as y) until its backward.

A cache is ``{"k": [B, S, G, D], "v": [B, S, G, D]}``, room for S tokens a sequence; how many each
holds is the caller's to keep, in `lengths`.
"""
from __future__ import annotations

import torch
import torch.autograd as autograd
from torch.autograd.function import once_differentiable

from .. import _lib
from .._common import _compute_dtype, _resolve_attn_scale
from ._inputs import (
    _CODES,
    _aligned_rows,
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
    _strides,
    _training,
)


# Caps that the kernels take: what scale / cap and the cap itself can be with in float32.
_LEAST_CAP, _MOST_CAP = 2.0 ** -100, 2.0 ** 100


def _check_scores(name, H, scale, softcap, slopes):
    """The cap, 0 for none, of checked arguments."""
    _check_shape(name, "slopes", slopes, (H,))
    _check_float(name, slopes=slopes)
    if slopes is not None and slopes.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{name} has no gradient for slopes; pass slopes.detach()")
    if softcap is None:
        return 0.0
    if not _LEAST_CAP <= softcap <= _MOST_CAP:
        raise ValueError(f"{name} expects softcap None or positive, between 2^-100 and 2^100. Got {softcap!r}")
    return float(softcap)


def _check_heads(name, Q, K, V):
    if Q.dim() != 4 or K.dim() != 4 or V.dim() != 4:
        raise ValueError(f"{name} expects Q [B, N, H, D] and K, V [B, N, G, D]. "
                         f"Got Q={tuple(Q.shape)}, K={tuple(K.shape)}, V={tuple(V.shape)}")
    B, N, H, D = Q.shape
    G = K.shape[2]
    if tuple(K.shape) != (B, N, G, D) or K.shape != V.shape:
        raise ValueError(f"{name} expects K and V [B, N, G, D] with B={B}, N={N}, D={D}. "
                         f"Got K={tuple(K.shape)}, V={tuple(V.shape)}")
    if H < 1 or G < 1 or H % G:
        raise ValueError(f"{name} expects query heads that divide into the key heads. Got H={H}, G={G}")
    if D % 16 or not 16 <= D <= 128:
        raise ValueError(f"{name} supports head dimensions that are multiples of 16 up to 128. Got D={D}")
    _check_float(name, Q=Q, K=K, V=V)
    return B, N, H, G, D


def _check_cache(name, cache, lengths, Q, K, V, B, G, D):
    """The cache's tensors: they are written in place, so they have to be what the kernels take."""
    if not isinstance(cache, dict) or "k" not in cache or "v" not in cache:
        raise ValueError(f"{name} expects a cache {{'k', 'v'}} of [B, S, G, D]. Got {cache!r:.80}")
    k, v = cache["k"], cache["v"]
    for what, t in (("cache['k']", k), ("cache['v']", v), ("lengths", lengths)):
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{name} expects a tensor in {what}. Got {t!r:.80}")
    if k.dim() != 4 or k.shape[1] < 1 or (k.shape[0], k.shape[2], k.shape[3]) != (B, G, D) or k.shape != v.shape:
        raise ValueError(f"{name} expects cache['k'] and cache['v'] [B, S, G, D] with B={B}, G={G}, D={D}. "
                         f"Got {tuple(k.shape)}, {tuple(v.shape)}")
    for what, t in (("Q", Q), ("K", K), ("V", V), ("cache['v']", v)):
        if t.dtype != k.dtype:
            raise ValueError(f"{name} expects one type for Q, K, V and the cache. Got {what} of {t.dtype} and "
                             f"cache['k'] of {k.dtype}")
    _lib.dtype_code(k.dtype)
    if not (k.is_contiguous() and v.is_contiguous()) or k.data_ptr() % 16 or v.data_ptr() % 16:
        raise ValueError(f"{name} writes the cache in place and expects it contiguous, on 16-byte boundaries")
    _check_integers(name, "lengths", lengths, (B,))
    return k, v


class SoftmaxAttention(autograd.Function):
    """Attention over whole sequences, with gradients for Q, K and V."""

    @staticmethod
    def forward(ctx, Q, K, V, scale, causal, softcap, slopes, document_ids, prefix_lengths, training):
        B, N, H, D = Q.shape
        G = K.shape[2]
        ctx.options = (scale, causal, softcap)
        if Q.numel() == 0:
            ctx.save_for_backward(Q, K, V, None, None, None, None, None, None)
            return torch.empty_like(Q)
        dtype = _compute_dtype(Q, K, V)
        q, k, v = (_aligned_rows(t, dtype) for t in (Q, K, V))
        sl, ids, pre = _f32(slopes), _int32(document_ids), _int32(prefix_lengths)
        y = torch.empty((B, N, H, D), device=Q.device, dtype=dtype)
        lse = torch.empty((B, H, N), device=Q.device, dtype=torch.float32) if training else None
        rest = torch.empty_like(y) if training and dtype is not torch.float32 else None
        lib = _lib.lib()
        nbytes = lib.flare_attn_forward_workspace_size(B, N, N, H, D, _lib.dtype_code(dtype))
        ws = torch.empty(nbytes, device=Q.device, dtype=torch.uint8)
        P = _ptr
        with _on(Q.device):
            rc = lib.flare_attn_forward(
                P(q), P(k), P(v), _strides(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3]), _lib.dtype_code(dtype),
                B, N, N, H, G, D, scale, softcap, P(sl), int(causal), P(ids), P(pre), None, None, P(y), P(rest),
                P(lse), P(ws), nbytes, _raw_stream(Q.device.index))
        _lib.check(rc, "flare_attn_forward")
        if training:
            ctx.save_for_backward(Q, K, V, sl, ids, pre, y, rest, lse)
        return y.to(Q.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        Q, K, V, sl, ids, pre, y, rest, lse = ctx.saved_tensors
        if Q.numel() == 0:
            return tuple(torch.zeros_like(t) for t in (Q, K, V)) + (None,) * 7
        B, N, H, D = Q.shape
        G = K.shape[2]
        scale, causal, softcap = ctx.options
        dtype = y.dtype
        q, k, v = (_aligned_rows(t, dtype) for t in (Q, K, V))
        g = _aligned_rows(dy, dtype).contiguous()
        dq, dk, dv = (torch.empty(t.shape, device=t.device, dtype=dtype) for t in (Q, K, V))
        lib = _lib.lib()
        nbytes = lib.flare_attn_backward_workspace_size(B, N, H, G, D, _lib.dtype_code(dtype))
        ws = torch.empty(nbytes, device=Q.device, dtype=torch.uint8)
        P = _ptr
        with _on(Q.device):
            rc = lib.flare_attn_backward(
                P(q), P(k), P(v), _strides(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3]), _lib.dtype_code(dtype),
                B, N, H, G, D, scale, softcap, P(sl), int(causal), P(ids), P(pre), P(y), P(rest), P(lse), P(g), P(dq),
                P(dk), P(dv), P(ws), nbytes, _raw_stream(Q.device.index))
        _lib.check(rc, "flare_attn_backward")
        return (dq.to(Q.dtype), dk.to(K.dtype), dv.to(V.dtype)) + (None,) * 7


def softmax_attention(
    Q: torch.Tensor,
    K: torch.Tensor,
    V: torch.Tensor,
    scale: float | None = None,
    causal: bool = True,
    softcap: float | None = None,
    slopes: torch.Tensor | None = None,
    document_ids: torch.Tensor | None = None,
    prefix_lengths: torch.Tensor | None = None,
):
    """Softmax attention of whole sequences, differentiable in Q, K and V.

    scale: D**-0.5 by default.  softcap: between 2^-100 and 2^100.  slopes: [H], the bias on distance
    (constants, no gradient).  document_ids: integers [B, N]; queries see keys of their own id only,
    and a negative id is padding, with y = 0 and no gradient.  prefix_lengths: integers [B]; the
    first so many keys of a sequence are seen by all its queries (of the same document).
    """
    name = "softmax_attention"
    B, N, H, G, D = _check_heads(name, Q, K, V)
    cap = _check_scores(name, H, scale, softcap, slopes)
    _check_integers(name, "document_ids", document_ids, (B, N))
    _check_integers(name, "prefix_lengths", prefix_lengths, (B,))
    if prefix_lengths is not None and not causal:
        raise ValueError(f"{name}: prefix_lengths say nothing without causal")
    _check_device(name, Q=Q, K=K, V=V, slopes=slopes, document_ids=document_ids, prefix_lengths=prefix_lengths)
    return SoftmaxAttention.apply(Q, K, V, _resolve_attn_scale(scale, D), bool(causal), cap, slopes, document_ids,
                                  prefix_lengths, _training(Q, K, V))


def softmax_attention_prefill(
    Q: torch.Tensor,
    K: torch.Tensor,
    V: torch.Tensor,
    cache: dict[str, torch.Tensor],
    lengths: torch.Tensor,
    scale: float | None = None,
    softcap: float | None = None,
    slopes: torch.Tensor | None = None,
    prefix_lengths: torch.Tensor | None = None,
    new_lengths: torch.Tensor | None = None,
):
    """Prompts that continue the cache: (y [B, T, H, D], the same cache).

    lengths: integers [B], the tokens each sequence's cache holds already.  The new keys and
    values are written behind them, in place, and the new queries, at positions lengths[b] + t,
    see the cached and the new ones causally (and the first prefix_lengths[b] positions, as far
    as they are there, whole).  new_lengths: integers [B], how many of the T rows are real (all by
    default); rows behind them give y = 0 and are not written.  `lengths` is not changed.  A
    sequence of negative length sits out (y = 0); one whose new tokens do not fit the cache is not
    written at all, and its y is NaN.
    """
    name = "softmax_attention_prefill"
    B, T, H, G, D = _check_heads(name, Q, K, V)
    cap = _check_scores(name, H, scale, softcap, slopes)
    kc, vc = _check_cache(name, cache, lengths, Q, K, V, B, G, D)
    _check_integers(name, "prefix_lengths", prefix_lengths, (B,))
    _check_integers(name, "new_lengths", new_lengths, (B,))
    device = _check_device(name, Q=Q, K=K, V=V, cache_k=kc, cache_v=vc, lengths=lengths, slopes=slopes,
                           prefix_lengths=prefix_lengths, new_lengths=new_lengths)
    y = torch.empty((B, T, H, D), device=device, dtype=kc.dtype)
    if y.numel() == 0:
        return y, cache
    S, code = kc.shape[1], _lib.dtype_code(kc.dtype)
    q, k, v = (_aligned_rows(t, kc.dtype) for t in (Q, K, V))
    sl, pre, lens, new = _f32(slopes), _int32(prefix_lengths), _int32(lengths), _int32(new_lengths)
    lib, P = _lib.lib(), _ptr
    nbytes = lib.flare_attn_forward_workspace_size(B, T, S, H, D, code)
    ws = torch.empty(nbytes, device=device, dtype=torch.uint8)
    with _on(device):
        stream = _raw_stream(device.index)
        rc = lib.flare_attn_append(P(k), P(v), _strides(*k.stride()[:3], *v.stride()[:3]), code, B, T, S, G, D, P(lens),
                                   P(new), P(kc), P(vc), stream)
        _lib.check(rc, "flare_attn_append")
        rc = lib.flare_attn_forward(
            P(q), P(kc), P(vc), _strides(*q.stride()[:3], *kc.stride()[:3], *vc.stride()[:3]), code, B, T, S, H, G, D,
            _resolve_attn_scale(scale, D), cap, P(sl), 1, None, P(pre), P(lens), P(new), P(y), None, None, P(ws), nbytes,
            stream)
    _lib.check(rc, "flare_attn_forward")
    return y, cache


def _step_fast(Q, K, V, cache, lengths, scale, softcap, slopes):
    """The common call, or None: one type, rows and a cache that the kernel reads in place, int32 lengths."""
    token = Q.dim() == 4
    if Q.dim() not in (3, 4) or (token and Q.shape[1] != 1) or not isinstance(cache, dict):
        return None
    kc, vc = cache.get("k"), cache.get("v")
    B, H, D = Q.shape[0], Q.shape[-2], Q.shape[-1]
    dtype, device = Q.dtype, Q.device
    code = _CODES.get(dtype)
    if (not isinstance(kc, torch.Tensor) or not isinstance(vc, torch.Tensor) or not isinstance(lengths, torch.Tensor)
            or kc.dim() != 4 or K.dim() != Q.dim() or code is None or device.type != "cuda"
            or device.index != torch.cuda.current_device()):
        return None
    S, G = kc.shape[1], K.shape[-2]
    want = (B, 1, G, D) if token else (B, G, D)
    if (K.shape != want or V.shape != want or kc.shape != (B, S, G, D) or vc.shape != kc.shape or not B * S * G
            or H < 1 or H % G or D % 16 or not 16 <= D <= 128 or lengths.dtype is not torch.int32
            or lengths.shape != (B,) or lengths.device != device or not lengths.is_contiguous()
            or not _plain_f32(slopes, device, H) or (slopes is not None and slopes.requires_grad)
            or (softcap is not None and not _LEAST_CAP <= softcap <= _MOST_CAP)):
        return None
    pointers = [t.data_ptr() for t in (Q, K, V, kc, vc)]
    strides, spread = [], 0
    for t in (Q, K, V):
        strides += (t.stride(0), t.stride(-2))
        if t.stride(-1) != 1:
            return None
    for x in strides:
        spread |= x * Q.element_size()
    for x in pointers:
        spread |= x
    if spread % 16 or not (kc.is_contiguous() and vc.is_contiguous()):
        return None
    for t in (K, V, kc, vc):
        if t.dtype is not dtype or t.device != device:
            return None
    y = torch.empty((B, 1, H, D), device=device, dtype=dtype)
    lib = _lib.lib()
    nbytes = lib.flare_attn_step_workspace_size(B, S, H, G, D)
    ws = torch.empty(nbytes, device=device, dtype=torch.uint8) if nbytes else None
    _lib.check(lib.flare_attn_step(
        *pointers[:3], _strides(*strides), code, B, S, H, G, D, _resolve_attn_scale(scale, D), softcap or 0.0,
        _ptr(slopes), lengths.data_ptr(), *pointers[3:], y.data_ptr(), _ptr(ws), nbytes, _raw_stream(device.index)),
        "flare_attn_step")
    return y, cache


def softmax_attention_decode(
    Q: torch.Tensor,
    K: torch.Tensor,
    V: torch.Tensor,
    cache: dict[str, torch.Tensor],
    lengths: torch.Tensor,
    scale: float | None = None,
    softcap: float | None = None,
    slopes: torch.Tensor | None = None,
):
    """One token a sequence, Q [B, H, D] or [B, 1, H, D] and K, V likewise: (y [B, 1, H, D], the same cache).

    lengths: integers [B], the tokens each sequence's cache holds already.  The token's key and
    value are written behind them, in place, and its query sees all lengths[b] + 1.  `lengths` is
    not changed.  A sequence of negative length sits out (y = 0, nothing written); one whose cache
    is full is not written, and its y is NaN.
    """
    name = "softmax_attention_decode"
    out = _step_fast(Q, K, V, cache, lengths, scale, softcap, slopes)
    if out is not None:
        return out
    Q, K, V = (t[:, None] if t.dim() == 3 else t for t in (Q, K, V))
    B, T, H, G, D = _check_heads(name, Q, K, V)
    if T != 1:
        raise ValueError(f"{name} expects one token a sequence. Got Q={tuple(Q.shape)}")
    cap = _check_scores(name, H, scale, softcap, slopes)
    kc, vc = _check_cache(name, cache, lengths, Q, K, V, B, G, D)
    device = _check_device(name, Q=Q, K=K, V=V, cache_k=kc, cache_v=vc, lengths=lengths, slopes=slopes)
    y = torch.empty((B, 1, H, D), device=device, dtype=kc.dtype)
    if B == 0:
        return y, cache
    S = kc.shape[1]
    q, k, v = (_aligned_rows(t, kc.dtype) for t in (Q, K, V))
    sl, lens = _f32(slopes), _int32(lengths)
    lib, P = _lib.lib(), _ptr
    nbytes = lib.flare_attn_step_workspace_size(B, S, H, G, D)
    ws = torch.empty(nbytes, device=device, dtype=torch.uint8) if nbytes else None
    strides = _strides(q.stride(0), q.stride(2), k.stride(0), k.stride(2), v.stride(0), v.stride(2))
    with _on(device):
        rc = lib.flare_attn_step(P(q), P(k), P(v), strides, _lib.dtype_code(kc.dtype), B, S, H, G, D,
                                 _resolve_attn_scale(scale, D), cap, P(sl), P(lens), P(kc), P(vc), P(y), P(ws), nbytes,
                                 _raw_stream(device.index))
    _lib.check(rc, "flare_attn_step")
    return y, cache
