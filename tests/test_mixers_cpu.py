"""Token mixers without a GPU: argument checks, refusals and the C entry points' own checks."""
import ctypes

import pytest
import torch

import causal_flare as cf
from causal_flare import _lib

CPU = "requires GPU tensors"


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("call, error, message", [
    (lambda: cf.short_convolution(t(2, 5), t(5, 4)), ValueError, r"expects x \[B, N, C\]"),
    (lambda: cf.short_convolution(t(2, 5, 6), t(5, 4)), ValueError, "expects weight"),
    (lambda: cf.short_convolution(t(2, 5, 6), t(6, 5)), ValueError, "2, 3 or 4 tokens. Got W=5"),
    (lambda: cf.short_convolution(t(2, 5, 6), t(6, 1)), ValueError, "2, 3 or 4 tokens"),
    (lambda: cf.short_convolution(t(2, 5, 6), t(6, 4), t(5)), ValueError, "expects bias"),
    (lambda: cf.short_convolution(t(2, 5, 6), t(6, 4), activation="gelu"), ValueError, "activation"),
    (lambda: cf.short_convolution(t(2, 5, 6), t(6, 4), document_ids=ints(2, 4)), ValueError, "document_ids"),
    (lambda: cf.short_convolution(t(2, 5, 6), t(6, 4), document_ids=t(2, 5)), ValueError, "integers"),
    (lambda: cf.short_convolution(ints(2, 5, 6), t(6, 4)), ValueError, "floating-point"),
    (lambda: cf.short_convolution(t(2, 5, 6), t(6, 4)), RuntimeError, CPU),
    (lambda: cf.short_convolution_prefill(t(2, 5, 6), t(6, 4), lengths=ints(3)), ValueError, "lengths"),
    (lambda: cf.short_convolution_prefill(t(2, 5, 6), t(6, 4)), RuntimeError, CPU),
    (lambda: cf.short_convolution_decode(t(2, 2, 6), t(6, 4)), ValueError, r"\[B, C\] or \[B, 1, C\]"),
    (lambda: cf.short_convolution_decode(t(2, 6), t(6, 4)), RuntimeError, CPU),
    (lambda: cf.state_space_scan(t(2, 6), t(2, 6), t(6, 4), t(2, 4), t(2, 4)), ValueError, r"x \[B, N, C\]"),
    (lambda: cf.state_space_scan(t(2, 5, 6), t(2, 5, 7), t(6, 4), t(2, 5, 4), t(2, 5, 4)), ValueError, "expects dt"),
    (lambda: cf.state_space_scan(t(2, 5, 6), t(2, 5, 6), t(5, 4), t(2, 5, 4), t(2, 5, 4)), ValueError, "expects A"),
    (lambda: cf.state_space_scan(t(2, 5, 6), t(2, 5, 6), t(6, 65), t(2, 5, 65), t(2, 5, 65)), ValueError, "1 to 64"),
    (lambda: cf.state_space_scan(t(2, 5, 6), t(2, 5, 6), t(6, 4), t(2, 5, 3), t(2, 5, 4)), ValueError, "expects B"),
    (lambda: cf.state_space_scan(t(2, 5, 6), t(2, 5, 6), t(6, 4), t(2, 5, 4), t(2, 5, 2, 4)), ValueError, "expects C"),
    (lambda: cf.state_space_scan(t(2, 5, 6), t(2, 5, 6), t(6, 4), t(2, 5, 4, 4), t(2, 5, 4, 4)), ValueError, "groups"),
    (lambda: cf.state_space_scan(t(2, 5, 6), t(2, 5, 6), t(6, 4), t(2, 5, 4), t(2, 5, 4), t(5)), ValueError, "expects D"),
    (lambda: cf.state_space_scan(t(2, 5, 6), t(2, 5, 6), t(6, 4), t(2, 5, 4), t(2, 5, 4), z=t(2, 5, 5)), ValueError,
     "expects z"),
    (lambda: cf.state_space_scan(t(2, 5, 6), t(2, 5, 6), t(6, 4), t(2, 5, 4), t(2, 5, 4)), RuntimeError, CPU),
    (lambda: cf.state_space_scan_prefill(t(2, 5, 6), t(2, 5, 6), t(6, 4), t(2, 5, 4), t(2, 5, 4), lengths=t(2)),
     ValueError, "integers"),
    (lambda: cf.state_space_scan_prefill(t(2, 5, 6), t(2, 5, 6), t(6, 4), t(2, 5, 4), t(2, 5, 4)), RuntimeError, CPU),
    (lambda: cf.state_space_scan_decode(t(2, 5, 6), t(2, 5, 6), t(6, 4), t(2, 5, 4), t(2, 5, 4)), ValueError, "one token"),
    (lambda: cf.state_space_scan_decode(t(2, 6), t(2, 6), t(6, 4), t(2, 4), t(2, 4)), RuntimeError, CPU),
    (lambda: cf.softmax_attention(t(2, 5, 4, 32), t(2, 5, 32), t(2, 5, 32)), ValueError, "expects Q"),
    (lambda: cf.softmax_attention(t(2, 5, 4, 32), t(2, 6, 4, 32), t(2, 6, 4, 32)), ValueError, "K and V"),
    (lambda: cf.softmax_attention(t(2, 5, 4, 32), t(2, 5, 3, 32), t(2, 5, 3, 32)), ValueError, "divide"),
    (lambda: cf.softmax_attention(t(2, 5, 4, 40), t(2, 5, 4, 40), t(2, 5, 4, 40)), ValueError, "multiples of 16"),
    (lambda: cf.softmax_attention(t(2, 5, 4, 144), t(2, 5, 4, 144), t(2, 5, 4, 144)), ValueError, "multiples of 16"),
    (lambda: cf.softmax_attention(*[t(2, 5, 4, 32)] * 3, softcap=0.0), ValueError, "softcap"),
    (lambda: cf.softmax_attention(*[t(2, 5, 4, 32)] * 3, softcap=float("inf")), ValueError, "softcap"),
    (lambda: cf.softmax_attention(*[t(2, 5, 4, 32)] * 3, slopes=t(3)), ValueError, "slopes"),
    (lambda: cf.softmax_attention(*[t(2, 5, 4, 32)] * 3, slopes=t(4).requires_grad_()), NotImplementedError, "slopes"),
    (lambda: cf.softmax_attention(*[t(2, 5, 4, 32)] * 3, document_ids=ints(2, 6)), ValueError, "document_ids"),
    (lambda: cf.softmax_attention(*[t(2, 5, 4, 32)] * 3, prefix_lengths=ints(3)), ValueError, "prefix_lengths"),
    (lambda: cf.softmax_attention(*[t(2, 5, 4, 32)] * 3, prefix_lengths=ints(2), causal=False), ValueError, "causal"),
    (lambda: cf.softmax_attention(*[t(2, 5, 4, 32)] * 3), RuntimeError, CPU),
    (lambda: cf.softmax_attention_prefill(*[t(2, 5, 4, 32)] * 3, {"k": t(2, 9, 4, 32)}, ints(2)), ValueError, "cache"),
    (lambda: cf.softmax_attention_prefill(*[t(2, 5, 4, 32)] * 3, {"k": t(2, 9, 4, 32), "v": t(2, 8, 4, 32)}, ints(2)),
     ValueError, "cache"),
    (lambda: cf.softmax_attention_prefill(*[t(2, 5, 4, 32)] * 3, {x: t(2, 9, 4, 32, dtype=torch.float16) for x in "kv"},
                                          ints(2)), ValueError, "one type"),
    (lambda: cf.softmax_attention_prefill(*[t(2, 5, 4, 32)] * 3, {x: t(2, 4, 9, 32).transpose(1, 2) for x in "kv"},
                                          ints(2)), ValueError, "contiguous"),
    (lambda: cf.softmax_attention_prefill(*[t(2, 5, 4, 32)] * 3, {x: t(2, 9, 4, 32) for x in "kv"}, ints(3)),
     ValueError, "lengths"),
    (lambda: cf.softmax_attention_prefill(*[t(2, 5, 4, 32)] * 3, {x: t(2, 9, 4, 32) for x in "kv"}, ints(2)),
     RuntimeError, CPU),
    (lambda: cf.softmax_attention_decode(*[t(2, 5, 4, 32)] * 3, {x: t(2, 9, 4, 32) for x in "kv"}, ints(2)),
     ValueError, "one token"),
    (lambda: cf.softmax_attention_decode(*[t(2, 4, 32)] * 3, {x: t(2, 9, 4, 32) for x in "kv"}, ints(2)),
     RuntimeError, CPU),
])
def test_refusals(call, error, message):
    with pytest.raises(error, match=message):
        call()


def _refused(rc, message):
    lib = _lib.lib()
    return rc == -1 and message in lib.flare_last_error()


def test_c_entry_points_check_before_they_launch():
    lib = _lib.lib()
    P = ctypes.c_void_p(4096)
    six, nine, twelve = ((ctypes.c_int64 * n)(*[8] * n) for n in (6, 9, 12))
    assert _refused(lib.flare_conv_forward(None, 1, 1, P, None, 0, 1, 1, 1, 8, 4, None, None, None, P, None, None),
                    b"null pointer")
    assert _refused(lib.flare_conv_forward(P, 1, 1, P, None, 0, 1, 1, 1, 8, 5, None, None, None, P, None, None), b"W must be")
    assert _refused(lib.flare_conv_forward(P, 1, 1, P, None, 0, 7, 1, 1, 8, 4, None, None, None, P, None, None), b"dtype")
    assert _refused(lib.flare_conv_forward(P, 1, 1, P, None, 0, 1, 1, 0, 8, 4, None, None, None, P, None, None), b"positive")
    assert _refused(lib.flare_conv_forward(P, 1, 1, P, None, 0, 1, 1, 4, 8, 4, P, P, None, P, None, None), b"exclude")
    assert _refused(lib.flare_conv_forward(P, 1, 1, P, None, 0, 1, 1 << 30, 1 << 30, 1 << 20, 4, None, None, None, P, None,
                                           None), b"too large")
    assert lib.flare_conv_backward(P, 1, 1, P, None, 0, 1, 1, 4, 8, 4, None, P, P, P, None, P, 8, None) == -3
    assert _refused(lib.flare_conv_step(P, 1, P, None, 0, 1, 1, 8, 4, None, None, P, None), b"null pointer")
    scan = [P] * 5 + [None] * 3 + [0, 1]
    assert _refused(lib.flare_scan_forward(*scan, 1, 4, 8, 65, 1, twelve, None, None, None, P, None, 4, None, P, 0, None),
                    b"1 to 64")
    assert _refused(lib.flare_scan_forward(*scan, 1, 4, 8, 16, 3, twelve, None, None, None, P, None, 4, None, P, 0, None),
                    b"groups")
    assert _refused(lib.flare_scan_forward(*scan, 1, 4, 8, 16, 1, twelve, None, None, None, P, None, 48, P, P, 0, None),
                    b"multiples")
    assert lib.flare_scan_forward(*scan, 1, 4, 8, 16, 1, twelve, None, None, None, P, None, 4, None, P, 8, None) == -3
    assert _refused(lib.flare_scan_forward(*scan, 1, 4, 8, 16, 1, twelve, P, None, P, P, None, 4, None, P, 0, None), b"exclude")
    for chunk in (160, 48, 0):
        assert _refused(lib.flare_scan_backward(*scan, 1, 400, 8, 16, 1, twelve, None, P, chunk, P, *[P] * 5, None, None,
                                                None, P, 0, None), b"chunks of up to 128")
    assert lib.flare_scan_backward(*scan, 1, 4, 8, 16, 1, twelve, None, P, 32, P, *[P] * 5, None, None, None, P, 0, None) == -3
    assert _refused(lib.flare_scan_step(*scan, 1, 8, 16, 1, twelve, None, None, P, None), b"null pointer")
    assert lib.flare_scan_chunk(1, 4, 8, 65, 1, 0) == 0
    for states in (4, 16, 32, 64):
        chunk = lib.flare_scan_chunk(1, 10 ** 7, 64, states, 1, 1)
        assert 1 <= chunk <= 128 and chunk % lib.flare_scan_kept_tokens(states) == 0
    attn = [P, P, P, nine, 1]
    assert _refused(lib.flare_attn_forward(*attn, 1, 4, 4, 4, 3, 64, 1.0, 0.0, None, 1, None, None, None, None, P, None, None, None,
                                           0, None), b"divide")
    assert _refused(lib.flare_attn_forward(*attn, 1, 4, 4, 4, 4, 24, 1.0, 0.0, None, 1, None, None, None, None, P, None, None, None,
                                           0, None), b"multiple of 16")
    assert _refused(lib.flare_attn_forward(*attn, 1, 4, 5, 4, 4, 64, 1.0, 0.0, None, 1, None, None, None, None, P, None, None, None,
                                           0, None), b"without a cache")
    assert _refused(lib.flare_attn_forward(*attn, 1, 4, 4, 4, 4, 64, 1.0, -1.0, None, 1, None, None, None, None, P, None,
                                           None, None, 0, None), b"cap")
    assert _refused(lib.flare_attn_forward(P, P, ctypes.c_void_p(4098), nine, 1, 1, 4, 4, 4, 4, 64, 1.0, 0.0, None, 1, None,
                                           None, None, None, P, None, None, None, 0, None), b"16-byte")
    assert lib.flare_attn_forward(*attn, 1, 4, 4, 4, 4, 64, 1.0, 0.0, None, 1, P, None, None, None, P, None, None, None,
                                  0, None) == -3
    assert lib.flare_attn_forward(*attn, 1, 4000, 4000, 1, 1, 64, 1.0, 0.0, None, 1, None, None, None, None, P, None, None, P,
                                  4096, None) == -3
    assert lib.flare_attn_backward(*attn, 1, 4, 4, 4, 64, 1.0, 0.0, None, 1, None, None, P, None, P, P, P, P, P, P, 0,
                                   None) == -3
    assert _refused(lib.flare_attn_append(P, P, six, 1, 1, 4, 8, 4, 64, None, None, P, P, None), b"null pointer")
    assert lib.flare_attn_step(P, P, P, six, 1, 1, 4096, 4, 4, 64, 1.0, 0.0, None, P, P, P, P, None, 0, None) == -3


def test_names():
    for name in ("short_convolution", "state_space_scan", "softmax_attention"):
        for face in ("", "_prefill", "_decode"):
            assert getattr(cf, name + face) is getattr(cf.mixers, name + face)
            assert name + face in cf.__all__ and name + face in cf.mixers.__all__


# The 64-bit forms that the GPU tests measure against: their gradients against differences of
# their values.
def _difference(f, leaves, dy, seed):
    g = torch.Generator().manual_seed(seed)
    way = [torch.randn(x.shape, generator=g, dtype=torch.float64) for x in leaves]
    e = 1e-5
    hi, lo = (f(*[x + s * e * w for x, w in zip(leaves, way)]) for s in (1, -1))
    return float(((hi - lo) * dy).sum() / (2 * e)), way


def _normal(g, *shape):
    return torch.randn(shape, generator=g, dtype=torch.float64)


def test_oracle_gradients_against_differences():
    import _mixers as M
    g = torch.Generator().manual_seed(3)
    ids = torch.tensor([[0, 0, 0, 1, 1, 1, 1, -1, -1], [2, 2, 2, 2, 2, 2, 2, 2, 2]])
    for silu in (False, True):
        x, w, b, dy = _normal(g, 2, 9, 3), _normal(g, 3, 4), _normal(g, 3), _normal(g, 2, 9, 3)
        got = M.conv(x, w, b, silu, ids, dy=dy)
        want, way = _difference(lambda *a: M.conv(*a, silu, ids)["y"][0], (x, w, b), dy, 4)
        have = sum(float((got[n][0] * v).sum()) for n, v in zip(("dx", "dweight", "dbias"), way))
        assert abs(have - want) < 1e-7 * (1 + abs(want))
    names = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")
    leaves = (_normal(g, 2, 9, 4), _normal(g, 2, 9, 4), -_normal(g, 4, 3).abs(), _normal(g, 2, 9, 2, 3),
              _normal(g, 2, 9, 2, 3), _normal(g, 4), _normal(g, 2, 9, 4), _normal(g, 4))
    dy = _normal(g, 2, 9, 4)
    got = M.scan(*leaves, softplus=True, ids=ids, dy=dy)
    want, way = _difference(lambda *a: M.scan(*a, softplus=True, ids=ids)["y"][0], leaves, dy, 5)
    have = sum(float((got["d" + n][0] * v).sum()) for n, v in zip(names, way))
    assert abs(have - want) < 1e-7 * (1 + abs(want))
    for cap, prefix in ((None, None), (2.0, torch.tensor([5, 0]))):
        q, k, v, dy = _normal(g, 2, 9, 4, 16), _normal(g, 2, 9, 2, 16), _normal(g, 2, 9, 2, 16), _normal(g, 2, 9, 4, 16)
        more = dict(softcap=cap, prefix=prefix, slopes=torch.tensor([0.1, 0.2, 0.5, 1.0]), ids=ids)
        got = M.attention(q, k, v, **more, dy=dy)
        want, way = _difference(lambda *a: M.attention(*a, **more)["y"][0], (q, k, v), dy, 6)
        have = sum(float((got[n][0] * w).sum()) for n, w in zip(("dq", "dk", "dv"), way))
        assert abs(have - want) < 1e-7 * (1 + abs(want))
