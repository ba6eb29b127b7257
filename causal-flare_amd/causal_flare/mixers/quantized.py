"""A cache of keys and values in 8 or 4 bits, for softmax attention.

``{"k", "v", "k_scale", "v_scale"}``: a token's key or value of one head is cut into blocks of 32
dimensions (the last may have 16), each with a power of 2 of its own,

    value = code 2^(scale - 127)

k, v: 8 bits, float8_e4m3fn [B, S, G, D], or 4, uint8 [B, S, G, D / 2] of two e2m1 codes (0, 1/2, 1, 3/2, 2,
3, 4, 6 and a sign; the lower index in the lower half).  k_scale, v_scale: uint8 [B, S, G, ceil(D / 32)].  The
scale is the least for which the block's largest value rounds to no more than the largest code (up to the
range of the type that is written from); values are rounded to the nearest code, ties to the even one.  A block
that holds an infinite value or a NaN is NaN, with a scale of 255.  The root of the mean square of what
normally distributed values are rounded by is 2.7% of theirs with 8 bits and 11% with 4.

`softmax_attention_prefill` and `softmax_attention_decode` take such a cache in place of one of the queries'
type.  They write new keys and values to it first and see them as it holds them, so that a prompt in pieces gives
what it gives whole.  Its codes have to be such as the calls write.  Queries of float16 see what it holds rounded to
float16: of a cache written from a wider type, values beyond 65504 are infinite to them.
"""
from __future__ import annotations

import torch

from .. import _lib
from ._inputs import (
    _CODES,
    _aligned_rows,
    _check_device,
    _check_float,
    _check_integers,
    _f32,
    _int32,
    _on,
    _plain_f32,
    _ptr,
    _raw_stream,
    _strides,
)

_BLOCK = 32
_FAR = 2 ** 31 - 1
_PARTS = ("k", "k_scale", "v", "v_scale")
_FORMS = {torch.uint8: 4, torch.float8_e4m3fn: 8}


def is_quantized(cache) -> bool:
    """Whether a cache is one of `quantized_cache`: with scales, and no keys of a type that queries have."""
    return isinstance(cache, dict) and "k_scale" in cache and getattr(cache.get("k"), "dtype", None) not in _CODES


def quantized_cache(B: int, S: int, G: int, D: int, bits: int = 8, device="cuda") -> dict[str, torch.Tensor]:
    """An empty cache of S tokens for each of B sequences, G key heads of D dimensions, in 8 or 4 bits."""
    name = "quantized_cache"
    if bits not in (4, 8):
        raise ValueError(f"{name} expects 8 or 4 bits. Got {bits!r}")
    if B < 0 or S < 1 or G < 1 or D % 16 or not 16 <= D <= 128:
        raise ValueError(f"{name} expects positive sizes, and head dimensions that are multiples of 16 up to 128. "
                         f"Got B={B}, S={S}, G={G}, D={D}")
    cache = {}
    for n in ("k", "v"):
        codes = torch.zeros((B, S, G, D * bits // 8), device=device, dtype=torch.uint8)
        cache[n] = codes.view(torch.float8_e4m3fn) if bits == 8 else codes
        cache[n + "_scale"] = torch.zeros((B, S, G, -(-D // _BLOCK)), device=device, dtype=torch.uint8)
    return cache


def check_quantized(name, cache):
    """(bits, B, S, G, D) of a cache whose tensors are what the kernels read and write in place."""
    if not isinstance(cache, dict) or any(not isinstance(cache.get(n), torch.Tensor) for n in _PARTS):
        raise ValueError(f"{name} expects a cache {{'k', 'v', 'k_scale', 'v_scale'}} of quantized_cache. Got {cache!r:.80}")
    k = cache["k"]
    if k.dtype not in (torch.uint8, torch.float8_e4m3fn):
        raise ValueError(f"{name} expects codes of float8_e4m3fn, or uint8 for 4 bits. Got {k.dtype}")
    bits = 4 if k.dtype is torch.uint8 else 8
    if k.dim() != 4:
        raise ValueError(f"{name} expects cache['k'] [B, S, G, D or D / 2]. Got {tuple(k.shape)}")
    B, S, G, D = k.shape[0], k.shape[1], k.shape[2], k.shape[3] * 8 // bits
    if D % 16 or not 16 <= D <= 128 or S < 1 or G < 1:
        raise ValueError(f"{name} supports head dimensions that are multiples of 16 up to 128. Got cache['k'] "
                         f"{tuple(k.shape)} of {bits} bits")
    scales = (B, S, G, -(-D // _BLOCK))
    for n, shape, dtype in (("v", k.shape, k.dtype), ("k_scale", scales, torch.uint8), ("v_scale", scales, torch.uint8)):
        if tuple(cache[n].shape) != tuple(shape) or cache[n].dtype is not dtype:
            raise ValueError(f"{name} expects cache[{n!r}] {list(shape)} of {dtype}. Got {tuple(cache[n].shape)} of "
                             f"{cache[n].dtype}")
    for n in _PARTS:
        if not cache[n].is_contiguous() or (n in ("k", "v") and cache[n].data_ptr() % 16):
            raise ValueError(f"{name} writes the cache in place and expects it contiguous, on 16-byte boundaries")
    return bits, B, S, G, D


def _plain_parts(cache, device):
    """(bits, shape of k, pointers of the four) of a cache that the kernels take on `device`, or None."""
    try:
        k, ks, v, vs = (cache[n] for n in _PARTS)
        shape, dtype = k.shape, k.dtype
        B, S, G, W = shape
        bits = _FORMS[dtype]
        D = W * 8 // bits
        scales = (B, S, G, (D + _BLOCK - 1) // _BLOCK)
        if (v.shape != shape or v.dtype is not dtype or ks.shape != scales or vs.shape != scales or D % 16 or not 16 <= D <= 128
                or ks.dtype is not torch.uint8 or vs.dtype is not torch.uint8 or not B * S * G):
            return None
        for t in (k, ks, v, vs):
            if t.device != device or not t.is_contiguous():
                return None
        pointers = (k.data_ptr(), ks.data_ptr(), v.data_ptr(), vs.data_ptr())
    except (KeyError, TypeError, ValueError, AttributeError):
        return None
    return None if (pointers[0] | pointers[2]) % 16 else (bits, B, S, G, D, pointers)


def _plain_int32(t, device, B):
    return t is None or (isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.shape == (B,) and t.device == device
                         and t.is_contiguous())


def attend_fast(Q, K, V, cache, lengths, scale, softcap, slopes, prefix_lengths, new_lengths):
    """y [B, T, H, D] of the common call, or None: one type, rows and a cache that the kernels read in place, on the
    current device, int32 lengths; Q, K, V of T tokens or, without that dimension, of one.  softcap: None or within the
    kernels' range."""
    dtype, device, shape = Q.dtype, Q.device, Q.shape
    code = _CODES.get(dtype)
    if (code is None or device.type != "cuda" or device.index != torch.cuda.current_device() or lengths is None
            or len(shape) not in (3, 4)):
        return None
    parts = _plain_parts(cache, device)
    if parts is None:
        return None
    bits, B, S, G, D, held = parts
    many = len(shape) == 4
    T, H = shape[1] if many else 1, shape[-2]
    want = (B, T, G, D) if many else (B, G, D)
    if (shape[0] != B or shape[-1] != D or T < 1 or H < 1 or H % G or K.shape != want or V.shape != want
            or not (_plain_int32(lengths, device, B) and _plain_int32(prefix_lengths, device, B)
                    and _plain_int32(new_lengths, device, B))):
        return None
    if slopes is not None and (not _plain_f32(slopes, device, H) or slopes.requires_grad):
        return None
    strides, spread = [], 0
    for t in (Q, K, V):
        if t.stride(-1) != 1 or t.dtype is not dtype or t.device != device:
            return None
        a, b, c = t.stride(0), t.stride(1) if many else 0, t.stride(-2)
        if b >= 1 << 22:
            return None
        strides += (a, b, c)
        spread |= a | b | c
    pointers = (Q.data_ptr(), K.data_ptr(), V.data_ptr())
    if (spread * Q.element_size() | pointers[0] | pointers[1] | pointers[2]) % 16:
        return None
    y = torch.empty((B, T, H, D), device=device, dtype=dtype)
    lib = _lib.lib()
    nbytes = lib.flare_qattn_workspace_size(B, T, S, H, G, D, code, bits)
    ws = torch.empty(nbytes, device=device, dtype=torch.uint8) if nbytes else None
    rc = lib.flare_qattn(
        *pointers, _strides(*strides), code, bits, B, T, S, H, G, D, scale, softcap or 0.0, _ptr(slopes), _ptr(prefix_lengths),
        lengths.data_ptr(), _ptr(new_lengths), *held, y.data_ptr(), _ptr(ws), nbytes, _raw_stream(device.index))
    if rc:
        _lib.check(rc, "flare_qattn")
    return y


def check_lengths(name, lengths, B):
    if not isinstance(lengths, torch.Tensor):
        raise ValueError(f"{name} expects a tensor in lengths. Got {lengths!r:.80}")
    _check_integers(name, "lengths", lengths, (B,))


def quantized_cache_write(
    cache: dict[str, torch.Tensor],
    K: torch.Tensor,
    V: torch.Tensor,
    lengths: torch.Tensor,
    new_lengths: torch.Tensor | None = None,
):
    """K and V [B, T, G, D] behind what the cache holds, in place; returns the cache.

    lengths: integers [B], the tokens each sequence's cache holds already, not changed.  new_lengths: integers
    [B], how many of the T rows are real (all by default); those behind them are not written.  A sequence of
    negative length sits out, and one whose new tokens do not fit the cache is not written at all.
    """
    name = "quantized_cache_write"
    bits, B, S, G, D = check_quantized(name, cache)
    if K.dim() != 4 or V.shape != K.shape or (K.shape[0], K.shape[2], K.shape[3]) != (B, G, D):
        raise ValueError(f"{name} expects K and V [B, T, G, D] with B={B}, G={G}, D={D}. Got {tuple(K.shape)}, "
                         f"{tuple(V.shape)}")
    _check_float(name, K=K, V=V)
    if V.dtype != K.dtype:
        raise ValueError(f"{name} expects one type for K and V. Got {K.dtype}, {V.dtype}")
    code = _lib.dtype_code(K.dtype)
    check_lengths(name, lengths, B)
    _check_integers(name, "new_lengths", new_lengths, (B,))
    device = _check_device(name, K=K, V=V, lengths=lengths, new_lengths=new_lengths, **{"cache_" + n: cache[n] for n in _PARTS})
    if K.numel() == 0:
        return cache
    k, v = _aligned_rows(K, K.dtype), _aligned_rows(V, K.dtype)
    lens, new = _int32(lengths), _int32(new_lengths)
    P = _ptr
    with _on(device):
        rc = _lib.lib().flare_qcache_write(
            P(k), P(v), _strides(*k.stride()[:3], *v.stride()[:3]), code, bits, B, K.shape[1], S, G, D, P(lens), P(new),
            *(cache[n].data_ptr() for n in _PARTS), _raw_stream(device.index))
    _lib.check(rc, "flare_qcache_write")
    return cache


def _read_fast(cache, first, count, dtype):
    """The common call, or None: a cache on the current device, int32 `first`."""
    code = _CODES.get(dtype)
    device = cache["k"].device if isinstance(cache, dict) and isinstance(cache.get("k"), torch.Tensor) else None
    if code is None or device is None or device.type != "cuda" or device.index != torch.cuda.current_device():
        return None
    parts = _plain_parts(cache, device)
    if parts is None:
        return None
    bits, B, S, G, D, held = parts
    count = S if count is None else count
    if type(count) is not int or count < 1:
        return None
    at = None
    if first is not None:
        if (not isinstance(first, torch.Tensor) or first.dtype is not torch.int32 or first.shape != (B,)
                or first.device != device or not first.is_contiguous()):
            return None
        at = first.data_ptr()
    k = torch.empty((B, count, G, D), device=device, dtype=dtype)
    v = torch.empty_like(k)
    rc = _lib.lib().flare_qcache_read(*held, code, bits, B, count, S, G, D, at, k.data_ptr(), v.data_ptr(),
                                      _raw_stream(device.index))
    if rc:
        _lib.check(rc, "flare_qcache_read")
    return k, v


def quantized_cache_read(
    cache: dict[str, torch.Tensor],
    first: torch.Tensor | None = None,
    count: int | None = None,
    dtype: torch.dtype = torch.bfloat16,
):
    """What the cache holds as tensors K, V [B, count, G, D] of `dtype`: rows first[b] .. first[b] + count - 1 of
    each sequence (all by default), 0 where these lie outside of the cache.

    first: integers [B].  dtype: bfloat16 or float32, in which every value is exact, or float16, in which it is
    if it was written from that type (and rounded to it otherwise, infinite beyond its range).
    """
    name = "quantized_cache_read"
    out = _read_fast(cache, first, count, dtype)
    if out is not None:
        return out
    bits, B, S, G, D = check_quantized(name, cache)
    code = _lib.dtype_code(dtype)
    _check_integers(name, "first", first, (B,))
    count = S if count is None else int(count)
    if count < 0:
        raise ValueError(f"{name} expects a count of rows, not negative. Got {count}")
    device = _check_device(name, first=first, **{"cache_" + n: cache[n] for n in _PARTS})
    k, v = (torch.empty((B, count, G, D), device=device, dtype=dtype) for _ in range(2))
    if k.numel() == 0:
        return k, v
    if first is not None and first.dtype is torch.int64:
        first = first.clamp(-_FAR, _FAR)             # rows beyond 32 bits are outside too
    at = _int32(first)
    P = _ptr
    with _on(device):
        rc = _lib.lib().flare_qcache_read(*(cache[n].data_ptr() for n in _PARTS), code, bits, B, count, S, G, D, P(at), P(k),
                                          P(v), _raw_stream(device.index))
    _lib.check(rc, "flare_qcache_read")
    return k, v


def attend_quantized(name, Q, K, V, cache, lengths, scale, cap, slopes, prefix_lengths, new_lengths):
    """Attention of new tokens, K and V of checked shapes, over a quantised cache that receives them: y."""
    B, T, H, D = Q.shape
    bits, cB, S, G, cD = check_quantized(name, cache)
    if (cB, G, cD) != (B, K.shape[2], D):
        raise ValueError(f"{name} expects a cache of B={B} sequences, G={K.shape[2]} heads of D={D}. Got B={cB}, G={G}, D={cD}")
    if K.dtype != Q.dtype or V.dtype != Q.dtype:
        raise ValueError(f"{name} expects one type for Q, K and V. Got {Q.dtype}, {K.dtype}, {V.dtype}")
    code = _lib.dtype_code(Q.dtype)
    check_lengths(name, lengths, B)
    device = _check_device(name, Q=Q, K=K, V=V, **{"cache_" + n: cache[n] for n in _PARTS}, lengths=lengths, slopes=slopes,
                           prefix_lengths=prefix_lengths, new_lengths=new_lengths)
    y = torch.empty((B, T, H, D), device=device, dtype=Q.dtype)
    if y.numel() == 0:
        return y
    q, k, v = (_aligned_rows(t, Q.dtype) for t in (Q, K, V))
    sl, pre, lens, new = _f32(slopes), _int32(prefix_lengths), _int32(lengths), _int32(new_lengths)
    lib, P = _lib.lib(), _ptr
    nbytes = lib.flare_qattn_workspace_size(B, T, S, H, G, D, code, bits)
    ws = torch.empty(nbytes, device=device, dtype=torch.uint8) if nbytes else None
    with _on(device):
        rc = lib.flare_qattn(
            P(q), P(k), P(v), _strides(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3]), code, bits, B, T, S, H, G, D,
            scale, cap, P(sl), P(pre), P(lens), P(new), *(cache[n].data_ptr() for n in _PARTS), P(y), P(ws), nbytes,
            _raw_stream(device.index))
    _lib.check(rc, "flare_qattn")
    return y
