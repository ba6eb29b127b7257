"""Quantised caches and rotary positions without a GPU: refusals, the C entry points' checks, and the 64-bit forms."""
import ctypes
import math

import pytest
import torch

import _quantized as Q
import causal_flare as cf
from causal_flare import _lib

CPU = "requires GPU tensors"


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def cache(bits=4, **other):
    return dict(cf.quantized_cache(2, 9, 4, 32, bits, device="cpu"), **other)


F = cf.rotary_frequencies(32)
QKV = [t(2, 5, 4, 32)] * 3


@pytest.mark.parametrize("call, error, message", [
    (lambda: cf.rotary_frequencies(7), ValueError, "even number"),
    (lambda: cf.rotary_frequencies(0), ValueError, "even number"),
    (lambda: cf.rotary_frequencies(8, base=0.0), ValueError, "positive base"),
    (lambda: cf.rotary_frequencies(8, factor=math.inf), ValueError, "positive base and factor"),
    (lambda: cf.rotary_frequencies(8, original_length=0), ValueError, "original_length"),
    (lambda: cf.rotary_frequencies(8, original_length=64, low_turns=4, high_turns=4), ValueError, "low_turns"),
    (lambda: cf.rotary_positions(t(2, 32), None, F), ValueError, "expects Q"),
    (lambda: cf.rotary_positions(t(2, 5, 4, 32), t(2, 4, 32), F), ValueError, "expects Q"),
    (lambda: cf.rotary_positions(t(2, 5, 4, 32), t(2, 6, 4, 32), F), ValueError, "expects K"),
    (lambda: cf.rotary_positions(t(2, 5, 4, 32), t(2, 5, 4, 16), F), ValueError, "expects K"),
    (lambda: cf.rotary_positions(t(2, 5, 0, 32), None, F), ValueError, "expects heads"),
    (lambda: cf.rotary_positions(ints(2, 5, 4, 32), None, F), ValueError, "floating-point"),
    (lambda: cf.rotary_positions(t(2, 5, 4, 32), None, F.float()), ValueError, "float64"),
    (lambda: cf.rotary_positions(t(2, 5, 4, 32), None, F.tolist()), ValueError, "float64"),
    (lambda: cf.rotary_positions(t(2, 5, 4, 32), None, F[None]), ValueError, "float64"),
    (lambda: cf.rotary_positions(t(2, 5, 4, 16), None, F), ValueError, "turns 2 to D"),
    (lambda: cf.rotary_positions(t(2, 5, 4, 32), None, F[:0]), ValueError, "turns 2 to D"),
    (lambda: cf.rotary_positions(t(2, 5, 4, 264), None, F), ValueError, "heads of up to 256"),
    (lambda: cf.rotary_positions(t(2, 5, 4, 32), None, F, positions=ints(2, 4)), ValueError, "positions"),
    (lambda: cf.rotary_positions(t(2, 5, 4, 32), None, F, positions=t(2, 5)), ValueError, "integers"),
    (lambda: cf.rotary_positions(t(2, 5, 4, 32), None, F, lengths=ints(3)), ValueError, "lengths"),
    (lambda: cf.rotary_positions(t(2, 5, 4, 32), None, F, ints(2, 5), ints(2)), ValueError, "not both"),
    (lambda: cf.rotary_positions(t(2, 5, 4, 32), None, F), RuntimeError, CPU),
    (lambda: cf.quantized_cache(1, 2, 3, 32, bits=5, device="cpu"), ValueError, "8 or 4 bits"),
    (lambda: cf.quantized_cache(1, 2, 3, 40, device="cpu"), ValueError, "multiples of 16"),
    (lambda: cf.quantized_cache(1, 0, 3, 32, device="cpu"), ValueError, "positive sizes"),
    (lambda: cf.quantized_cache_write({}, *QKV[1:], ints(2)), ValueError, "expects a cache"),
    (lambda: cf.quantized_cache_write(cache(k_scale=None), *QKV[1:], ints(2)), ValueError, "expects a cache"),
    (lambda: cf.quantized_cache_write(cache(k=t(2, 9, 4, 32)), *QKV[1:], ints(2)), ValueError, "expects codes"),
    (lambda: cf.quantized_cache_write(cache(k=t(2, 9, 4, dtype=torch.uint8)), *QKV[1:], ints(2)), ValueError, r"cache\['k'\]"),
    (lambda: cf.quantized_cache_write(cache(k=t(2, 9, 4, 4, dtype=torch.uint8)), *QKV[1:], ints(2)), ValueError, "multiples of 16"),
    (lambda: cf.quantized_cache_write(cache(v=t(2, 9, 4, 32, dtype=torch.uint8)), *QKV[1:], ints(2)), ValueError, "'v'"),
    (lambda: cf.quantized_cache_write(cache(8, v=t(2, 9, 4, 32, dtype=torch.uint8)), *QKV[1:], ints(2)), ValueError, "'v'"),
    (lambda: cf.quantized_cache_write(cache(k_scale=t(2, 9, 4, 2, dtype=torch.uint8)), *QKV[1:], ints(2)), ValueError, "k_scale"),
    (lambda: cf.quantized_cache_write(cache(v_scale=t(2, 9, 4, 1)), *QKV[1:], ints(2)), ValueError, "v_scale"),
    (lambda: cf.quantized_cache_write(cache(k=t(2, 4, 9, 16, dtype=torch.uint8).transpose(1, 2)), *QKV[1:], ints(2)), ValueError,
     "contiguous"),
    (lambda: cf.quantized_cache_write(cache(), t(2, 5, 3, 32), t(2, 5, 3, 32), ints(2)), ValueError, "expects K and V"),
    (lambda: cf.quantized_cache_write(cache(), t(2, 5, 4, 32), t(2, 6, 4, 32), ints(2)), ValueError, "expects K and V"),
    (lambda: cf.quantized_cache_write(cache(), t(2, 5, 4, 32), t(2, 5, 4, 32).half(), ints(2)), ValueError, "one type"),
    (lambda: cf.quantized_cache_write(cache(), *[t(2, 5, 4, 32).double()] * 2, ints(2)), ValueError, "unsupported dtype"),
    (lambda: cf.quantized_cache_write(cache(), *QKV[1:], ints(3)), ValueError, "lengths"),
    (lambda: cf.quantized_cache_write(cache(), *QKV[1:], [0, 0]), ValueError, "tensor in lengths"),
    (lambda: cf.quantized_cache_write(cache(), *QKV[1:], ints(2), t(2)), ValueError, "integers"),
    (lambda: cf.quantized_cache_write(cache(), *QKV[1:], ints(2)), RuntimeError, CPU),
    (lambda: cf.quantized_cache_read(cache(), first=ints(3)), ValueError, "first"),
    (lambda: cf.quantized_cache_read(cache(), count=-1), ValueError, "count"),
    (lambda: cf.quantized_cache_read(cache(), dtype=torch.float64), ValueError, "unsupported dtype"),
    (lambda: cf.quantized_cache_read(cache()), RuntimeError, CPU),
    (lambda: cf.softmax_attention_prefill(*QKV, cache(), ints(3)), ValueError, "lengths"),
    (lambda: cf.softmax_attention_prefill(*QKV, cache(), None), ValueError, "tensor in lengths"),
    (lambda: cf.softmax_attention_prefill(*[t(2, 5, 4, 64)] * 3, cache(), ints(2)), ValueError, "expects a cache of"),
    (lambda: cf.softmax_attention_prefill(*[t(2, 5, 2, 32)] * 3, cache(), ints(2)), ValueError, "expects a cache of"),
    (lambda: cf.softmax_attention_prefill(QKV[0].half(), *QKV[1:], cache(), ints(2)), ValueError, "one type"),
    (lambda: cf.softmax_attention_prefill(*[x.double() for x in QKV], cache(), ints(2)), ValueError, "unsupported dtype"),
    (lambda: cf.softmax_attention_prefill(*QKV, cache(v=None), ints(2)), ValueError, "expects a cache"),
    (lambda: cf.softmax_attention_prefill(*QKV, cache(), ints(2), softcap=-1.0), ValueError, "softcap"),
    (lambda: cf.softmax_attention_prefill(*QKV, cache(), ints(2), prefix_lengths=ints(3)), ValueError, "prefix_lengths"),
    (lambda: cf.softmax_attention_prefill(*QKV, cache(), ints(2), new_lengths=t(2)), ValueError, "integers"),
    (lambda: cf.softmax_attention_prefill(*QKV, cache(), ints(2)), RuntimeError, CPU),
    (lambda: cf.softmax_attention_decode(*QKV, cache(), ints(2)), ValueError, "one token"),
    (lambda: cf.softmax_attention_decode(*[t(32)] * 3, cache(), ints(2)), ValueError, "expects Q"),
    (lambda: cf.softmax_attention_decode(t(), t(), t(), cache(), ints(2)), ValueError, "expects Q"),
    (lambda: cf.softmax_attention_prefill(*[t(2, 4, 32)] * 3, cache(), ints(2)), ValueError, "expects Q"),
    (lambda: cf.softmax_attention_decode(*[t(2, 4, 32)] * 3, cache(8), ints(3)), ValueError, "lengths"),
    (lambda: cf.softmax_attention_decode(*[t(2, 4, 32)] * 3, cache(8), ints(2)), RuntimeError, CPU),
])
def test_refusals(call, error, message):
    with pytest.raises(error, match=message):
        call()


def _refused(rc, message):
    return rc == -1 and message in _lib.lib().flare_last_error()


def test_c_entry_points_check_before_they_launch():
    lib = _lib.lib()
    P, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4100)
    six, nine = ((ctypes.c_int64 * n)(*[16] * n) for n in (6, 9))
    f = (ctypes.c_double * 16)(*[0.5] * 16)

    def rotary(q=P, k=P, dtype=1, B=1, N=4, H=4, G=4, D=64, R=32, freq=f, at=None, lens=None, out=P, out_k=P):
        return lib.flare_rotary(q, k, six, dtype, B, N, H, G, D, R, freq, at, lens, 0, 0, out, out_k, None)
    assert _refused(rotary(q=None), b"null pointer") and _refused(rotary(out_k=None), b"null pointer")
    assert _refused(rotary(dtype=5), b"dtype") and _refused(rotary(N=0), b"positive") and _refused(rotary(G=0), b"positive")
    assert _refused(rotary(R=31), b"even number") and _refused(rotary(R=66), b"even number")
    assert _refused(rotary(D=512), b"256") and _refused(rotary(at=P, lens=P), b"exclude")
    assert _refused(rotary(N=1 << 31), b"too large") and _refused(rotary(H=1 << 20), b"too large")
    assert _refused(rotary(freq=(ctypes.c_double * 16)(*[0.5] * 15, math.nan)), b"frequency 15 is not finite")
    assert _refused(rotary(freq=(ctypes.c_double * 16)(*[math.inf] * 16)), b"frequency 0 is not finite")

    def write(k=P, kc=P, bits=4, dtype=1, B=1, N=4, M=8, G=4, D=64, lens=P):
        return lib.flare_qcache_write(k, P, six, dtype, bits, B, N, M, G, D, lens, None, kc, P, P, P, None)
    assert _refused(write(k=None), b"null pointer") and _refused(write(lens=None), b"null pointer")
    assert _refused(write(bits=3), b"3 bits") and _refused(write(dtype=9), b"dtype") and _refused(write(D=24), b"multiple of 16")
    assert _refused(write(D=144), b"multiple of 16") and _refused(write(M=0), b"positive") and _refused(write(N=1 << 28), b"too large")
    assert _refused(write(B=1 << 17), b"too large") and _refused(write(kc=odd), b"16-byte") and _refused(write(k=odd), b"16-byte")

    def read(kc=P, out=P, bits=8, N=4, D=64):
        return lib.flare_qcache_read(kc, P, P, P, 1, bits, 1, N, 8, 4, D, None, out, P, None)
    assert _refused(read(kc=None), b"null pointer") and _refused(read(out=odd), b"16-byte") and _refused(read(bits=16), b"16 bits")
    assert _refused(read(N=0), b"positive") and _refused(read(D=8), b"multiple of 16")

    def attend(q=P, bits=4, B=1, N=1, M=4096, H=4, G=4, D=64, cap=0.0, ws=None, size=0, kc=P):
        return lib.flare_qattn(q, P, P, nine, 1, bits, B, N, M, H, G, D, 1.0, cap, None, None, P, None, kc, P, P, P, P, ws, size, None)
    assert _refused(attend(q=None), b"null pointer") and _refused(attend(bits=2), b"2 bits") and _refused(attend(H=6), b"divide")
    assert _refused(attend(D=200), b"multiple of 16") and _refused(attend(cap=-1.0), b"cap") and _refused(attend(kc=odd), b"16-byte")
    for n in (1, 9, 200):
        need = lib.flare_qattn_workspace_size(1, n, 4096, 4, 4, 64, 1, 4)
        assert need > 0 and need % 16 == 0
        assert attend(N=n) == -3 and attend(N=n, ws=P, size=need - 1) == -3 and attend(N=n, ws=odd, size=need) == -3
    assert lib.flare_qattn_workspace_size(1, 4096, 8, 4, 4, 0, 1, 4) == 0
    assert lib.flare_qattn_workspace_size(0, 1, 8, 4, 4, 64, 1, 4) == 0 and lib.flare_qattn_workspace_size(1, 1, 8, 4, 3, 64, 1, 8) == 0


def test_names():
    for name in ("quantized_cache", "quantized_cache_read", "quantized_cache_write", "rotary_frequencies", "rotary_positions"):
        assert getattr(cf, name) is getattr(cf.mixers, name)
        assert name in cf.__all__ and name in cf.mixers.__all__


def test_layout():
    c = cf.quantized_cache(2, 9, 4, 80, 4, device="cpu")
    assert c["k"].shape == (2, 9, 4, 40) and c["k"].dtype is torch.uint8 and c["v_scale"].shape == (2, 9, 4, 3)
    c = cf.quantized_cache(2, 9, 4, 80, device="cpu")
    assert c["v"].shape == (2, 9, 4, 80) and c["v"].dtype is torch.float8_e4m3fn and c["k_scale"].dtype is torch.uint8


# The 64-bit forms that the GPU tests measure against.
@pytest.mark.parametrize("bits", [4, 8])
def test_the_plain_form_rounds_to_the_nearest(bits):
    """Against every code there is, at every scale that the block's largest value allows."""
    g = torch.Generator().manual_seed(bits)
    codes = torch.arange(16 if bits == 4 else 256)
    if bits == 4:
        table = Q.held((codes[:8] * 2 + 16 * (codes[:8] * 2 + 1)).to(torch.uint8)[:, None], torch.full((8, 1), 127, dtype=torch.uint8)).flatten()
    else:
        codes = codes[(codes & 127) != 127]
        table = Q.held(codes.to(torch.uint8).view(torch.float8_e4m3fn)[:, None], torch.full((254, 1), 127, dtype=torch.uint8)).flatten()
    assert table.max() == (6.0 if bits == 4 else 448.0) and len(set(table.tolist())) == len(codes) - 1     # 0 and -0
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        x = (torch.randn(40, 48, generator=g) * 2.0 ** torch.randint(-8, 8, (40, 1), generator=g)).to(dt)
        value, byte = Q.rounded(x, bits)
        assert byte.shape == (40, 2)
        for d in (0, 32):
            scale = 2.0 ** (byte[:, d // 32].double() - 127)
            block = x[:, d:d + 32].double()
            best = (block[..., None] - table * scale[:, None, None]).abs().amin(-1)
            got = (block - value[:, d:d + 32]).abs()
            # the largest may have been cut, by no more than the half step that it would round by
            assert torch.equal(got, best)
            top = block.abs().amax(1)
            assert (top <= Q.FORMS[bits][3] * scale).all()
            # a scale half as large would not do, or is none of the type (fp16: 464 2^-16 is 0.007)
            least = 2.0 ** Q.FORMS[bits][4 if dt is torch.float16 else 5][0]
            assert ((top > Q.FORMS[bits][3] * scale / 2) | (scale == least)).all()
        assert torch.equal(value.to(dt).double(), value)


def test_rotary_gradients_against_differences():
    g = torch.Generator().manual_seed(1)
    f = cf.rotary_frequencies(12, base=100.0)
    at = torch.randint(-50, 5000, (2, 7), generator=g)
    for interleaved in (False, True):
        x, dy, way = (torch.randn((2, 7, 3, 16), generator=g, dtype=torch.float64) for _ in range(3))
        hi, lo = (Q.rotary(x + e * way, f, at, interleaved)[0] for e in (1e-5, -1e-5))
        want = float(((hi - lo) * dy).sum() / 2e-5)
        have = float((Q.rotary(dy, f, at, interleaved, inverse=True)[0] * way).sum())
        assert abs(have - want) < 1e-7 * (1 + abs(want))


@pytest.mark.parametrize("token", [False, True])
def test_frequencies_have_no_gradient(token):
    f, q = F.clone().requires_grad_(), t(2, 4, 32) if token else t(2, 5, 4, 32)
    for k in (None, q):
        with pytest.raises(NotImplementedError, match="no gradient for frequencies"):
            cf.rotary_positions(q, k, f)
        with torch.no_grad(), pytest.raises(RuntimeError, match=CPU):
            cf.rotary_positions(q, k, f)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_other_entries_of_a_cache_are_the_callers(dtype):
    """Keys and values of the queries' type stay such a cache, whatever else its dict holds."""
    qkv = [t(2, 5, 4, 32, dtype=dtype)] * 3
    plain = {n: t(2, 9, 4, 32, dtype=dtype) for n in ("k", "v")}
    for more in ({}, {"k_scale": t(4)}, {"k_scale": None, "v_scale": 1.0}):
        with pytest.raises(RuntimeError, match=CPU):
            cf.softmax_attention_prefill(*qkv, dict(plain, **more), ints(2))
        with pytest.raises(RuntimeError, match=CPU):
            cf.softmax_attention_decode(*(x[:, 0] for x in qkv), dict(plain, **more), ints(2))


def test_grids_that_cannot_be_launched_are_refused_first():
    """2^32 threads and more in a dimension of a grid, which a launch does not take: nothing may be written before."""
    lib, P = _lib.lib(), ctypes.c_void_p(4096)
    six, nine = ((ctypes.c_int64 * n)(*[16] * n) for n in (6, 9))
    f = (ctypes.c_double * 128)(*[0.5] * 128)

    def attend(dtype, B, N, M, H, G, D=16, bits=4):
        size = lib.flare_qattn_workspace_size(B, N, M, H, G, D, dtype, bits)
        return lib.flare_qattn(P, P, P, nine, dtype, bits, B, N, M, H, G, D, 1.0, 0.0, None, None, P, None, P, P, P, P, P, P, size, None)
    assert _refused(attend(0, 32, 1 << 24, 1 << 25, 8, 1), b"too large")               # rows: 2^28 workgroups
    assert _refused(attend(0, 1, 1 << 24, 1 << 25, 16, 1), b"too large")               # 2^24
    assert _refused(attend(1, 1 << 14, 1024, 4096, 256, 256, bits=8), b"too large")    # prompts, by codes: 2^25
    assert _refused(attend(2, 8192, 1 << 16, 16, 8, 1), b"too large")                  # over values of 16 bits: 2^25

    def rotary(N, H=32, D=256, R=256):
        return lib.flare_rotary(P, P, six, 1, 1, N, H, H, D, R, f, None, None, 0, 0, P, P, None)
    assert _refused(rotary(1 << 24), b"too large") and _refused(rotary((1 << 25) - 1, R=32), b"too large")


@pytest.mark.parametrize("bits", [4, 8])
def test_workspace_of_large_rooms(bits):
    """Values turned into 16 bits take 1 GiB at most, whatever a cache has room for; the rest is what parts of rows leave."""
    size, B, N, H, G, D = _lib.lib().flare_qattn_workspace_size, 3, 4096, 16, 4, 128
    parts = 2 * 4 * B * N * H * (D + 4)
    some = 0
    for room in (1 << 14, 1 << 17, (1 << 19) - 1, 1 << 19, (1 << 19) + 1, 1 << 20, 1 << 21, 1 << 22, 1 << 24, 1 << 30):
        need = size(B, N, room, H, G, D, 1, bits)
        assert need <= (1 << 30) + parts, room
        some = max(some, need)
        if room > 1 << 19:
            assert need <= parts
    assert some >= 1 << 30
