"""Caches of 8 and 4 bits and attention over them, against plain 64-bit forms."""
import math

import pytest
import torch

import _mixers as M
import _quantized as Q
import causal_flare as cf

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
PARTS = ("k", "k_scale", "v", "v_scale")


def rng(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, dtype=torch.float64) * std).to(dtype)


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def raw(cache):
    return {n: cache[n].view(torch.uint8).cpu().clone() for n in PARTS}


def filled(g, B, S, G, D, bits):
    """A cache of arbitrary codes: finite ones, with scales about 1 and here and there a block that is NaN."""
    cache = cf.quantized_cache(B, S, G, D, bits)
    for n in ("k", "v"):
        shape = cache[n].shape
        codes = torch.randint(0, 256, shape, generator=g).to(torch.uint8)
        if bits == 8:
            codes = torch.where((codes & 127) == 127, codes - 1, codes)      # no NaN among them
        cache[n].view(torch.uint8).copy_(codes)
        scale = torch.randint(115, 122, cache[n + "_scale"].shape, generator=g).to(torch.uint8)
        cache[n + "_scale"].copy_(torch.where(torch.rand(scale.shape, generator=g) < 0.05, 255, scale))
    return cache


def odd_values(x):
    """Rows of `x` [B, T, G, D] with values that a format may stumble over."""
    info = torch.finfo(x.dtype)
    flat = x.flatten(0, 2)
    specials = [0.0, -0.0, info.max, -info.max, info.tiny, info.tiny / 4, 7.0, 464.0, 6.0, 448.0, 0.25, 5.0, 1.75, 1.8125,
                math.inf, -math.inf, math.nan]
    for i, s in enumerate(specials):
        if i < flat.shape[0]:
            flat[i, (5 * i) % flat.shape[1]] = s
    if flat.shape[0] > 40:
        flat[30] = 0.0
        flat[31] = -0.0
        flat[32] = info.max
        flat[33] = info.tiny
        flat[34] = torch.linspace(-7, 7, flat.shape[1]).to(x.dtype)
        flat[35] = torch.linspace(-464, 464, flat.shape[1]).to(x.dtype)
    return x


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D", [16, 48, 64, 80, 96, 112, 128])
def test_write_and_read(dtype, bits, D):
    dt, g = TYPES[dtype], rng(D + bits)
    B, T, G, S = 5, 9, 3, 21
    # spread over the exponents that a type has
    spread = torch.randint(-20, 14, (B, T, G, 1), generator=g).double() if dt is torch.float16 else \
        torch.randint(-130, 125, (B, T, G, 1), generator=g).double()
    k, v = ((torch.randn((B, T, G, D), generator=g, dtype=torch.float64) * 2.0 ** spread).clamp(
        -torch.finfo(dt).max, torch.finfo(dt).max).to(dt) for _ in range(2))
    k = odd_values(k)
    cache = filled(g, B, S, G, D, bits)
    before = raw(cache)
    # in place, with nothing real, idle, past the end by one, and filling the cache to its end
    lengths, new = (3, 7, -1, S - T + 1, S - T), (T, 0, T, T, T)
    wide = torch.empty((B, T, G, 2 * D), dtype=dt, device="cuda")          # rows that are slices
    wide[..., :D] = k.cuda()
    assert cf.quantized_cache_write(cache, wide[..., :D], v.cuda(), ints(*lengths), ints(*new)) is cache
    after = raw(cache)
    for n, x in (("k", k), ("v", v)):
        value, scale = Q.rounded(x, bits)
        got = Q.held(cache[n], cache[n + "_scale"])
        for b in range(B):
            writes = new[b] if lengths[b] >= 0 and lengths[b] + new[b] <= S else 0
            at = slice(max(lengths[b], 0), max(lengths[b], 0) + writes)
            assert torch.equal(after[n + "_scale"][b, at], scale[b, :writes]), (n, b)
            assert torch.equal(torch.nan_to_num(got[b, at], nan=7e77), torch.nan_to_num(value[b, :writes], nan=7e77)), (n, b)
            # what a type wrote it holds
            back = value[b, :writes].to(dt).double()
            assert torch.equal(torch.nan_to_num(back, nan=7e77), torch.nan_to_num(value[b, :writes], nan=7e77))
            keep = torch.ones(S, dtype=torch.bool)
            keep[at] = False
            for part in (n, n + "_scale"):
                assert torch.equal(after[part][b, keep], before[part][b, keep]), (part, b)
    # read back, whole and in windows that reach outside
    for kind in TYPES.values():
        for first, count in ((None, None), (ints(0, -2, S - 3, 2 * S, 5), 6)):
            got = cf.quantized_cache_read(cache, first, count, kind)
            for n, x in zip(("k", "v"), got):
                assert x.dtype is kind
                all_ = Q.held(cache[n], cache[n + "_scale"])
                ref = all_
                if first is not None:
                    ref = torch.zeros((B, count, G, D), dtype=torch.float64)
                    for b in range(B):
                        for i in range(count):
                            if 0 <= int(first[b]) + i < S:
                                ref[b, i] = all_[b, int(first[b]) + i]
                ref = ref.float().to(kind)
                assert torch.equal(torch.nan_to_num(x.cpu().float(), nan=7e37), torch.nan_to_num(ref.float(), nan=7e37))


def check_attention(dtype, bits, H, G, D, S, T, lengths, new=None, cap=None, slopes=None, prefix=None, seed=0, scale=None,
                    q_std=2.0, decode=False):
    dt, g = TYPES[dtype], rng(seed)
    B = len(lengths)
    k, v, q = normal(g, B, T, G, D, dtype=dt), normal(g, B, T, G, D, dtype=dt), normal(g, B, T, H, D, dtype=dt, std=q_std)
    cache = filled(g, B, S, G, D, bits)
    # what the sequences hold has no NaN; what lies behind may
    old = {n: normal(g, B, S, G, D, dtype=dt) for n in ("k", "v")}
    cf.quantized_cache_write(cache, old["k"].cuda(), old["v"].cuda(), torch.zeros(B, dtype=torch.int32, device="cuda"),
                             ints(*[max(0, n) for n in lengths]))
    lens = ints(*lengths)
    sl = None if slopes is None else torch.tensor(slopes, dtype=torch.float32)
    fresh = [T] * B if new is None else list(new)
    before = raw(cache)
    more = dict(scale=scale, softcap=cap, slopes=None if sl is None else sl.cuda())
    if decode:
        y, same = cf.softmax_attention_decode(q[:, 0].cuda(), k[:, 0].cuda(), v[:, 0].cuda(), cache, lens, **more)
    else:
        y, same = cf.softmax_attention_prefill(q.cuda(), k.cuda(), v.cuda(), cache, lens, **more,
                                               prefix_lengths=None if prefix is None else ints(*prefix),
                                               new_lengths=None if new is None else ints(*new))
    assert same is cache and y.dtype is dt and y.shape == (B, T, H, D)
    after = raw(cache)
    assert torch.equal(lens.cpu(), torch.tensor(lengths, dtype=torch.int32))
    unit = 0.0 if dt is torch.float32 else M.U[dt]
    tiny = 2.0 ** -25 if dt is torch.float16 else 2.0 ** -126
    for b in range(B):
        off, n = lengths[b], fresh[b]
        fits = off >= 0 and off + n <= S
        writes = n if fits else 0
        at = slice(max(off, 0), max(off, 0) + writes)
        for name, x in (("k", k), ("v", v)):
            value, byte = Q.rounded(x[b:b + 1, :writes], bits)
            assert torch.equal(Q.held(cache[name][b:b + 1, at], cache[name + "_scale"][b:b + 1, at]), value)
            keep = torch.ones(S, dtype=torch.bool)
            keep[at] = False
            for part in (name, name + "_scale"):
                assert torch.equal(after[part][b, keep], before[part][b, keep]), (part, b)
        if off < 0:
            assert (y[b] == 0).all(), b
        elif not fits:
            assert torch.isnan(y[b]).all(), b
        else:
            assert (y[b, n:] == 0).all(), b
            if n == 0:
                continue
            kk, vv = (Q.held(cache[name][b:b + 1, :off + n], cache[name + "_scale"][b:b + 1, :off + n]) for name in ("k", "v"))
            ref, tol = M.attention(q[b:b + 1, :n], kk, vv, scale, softcap=cap, slopes=sl, offset=[off],
                                   prefix=None if prefix is None else [min(prefix[b], off + n)], unit=unit, tiny=tiny)["y"]
            M.check(y[b:b + 1, :n], ref, tol + M.U[dt] * ref.abs(), f"y of sequence {b}", dt)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("H, G, D", [(4, 4, 16), (6, 2, 48), (8, 2, 64), (5, 5, 80), (8, 1, 96), (20, 1, 112), (16, 4, 128)])
def test_decode(dtype, bits, H, G, D):
    # empty, idle, one short of full, full, the ends of a wave's and of a workgroup's tiles, and several shares
    check_attention(dtype, bits, H, G, D, 700, 1, [0, -1, 699, 700, 31, 32, 63, 64, 65, 255, 256, 511, 1], seed=D + bits,
                    decode=True)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cap, slopes", [(15.0, False), (400.0, False), (None, True), (20.0, True)])
def test_decode_scores(dtype, bits, cap, slopes):
    check_attention(dtype, bits, 8, 4, 64, 400, 1, [399, 0, 150], cap=cap, slopes=[2.0 ** -i for i in range(8)] if slopes else None,
                    seed=bits, decode=True)
    check_attention(dtype, bits, 8, 4, 128, 300, 1, [257], cap=cap, slopes=[2.0 ** -i for i in range(8)] if slopes else None,
                    seed=bits, decode=True, scale=-0.2)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("H, G, D, B, S", [(16, 4, 64, 36, 500), (8, 8, 48, 17, 300), (12, 6, 96, 30, 300), (4, 4, 128, 33, 70),
                                           (4, 4, 32, 800, 40), (2, 2, 16, 800, 37)])
def test_decode_of_many_sequences(dtype, bits, H, G, D, B, S):
    # key heads side by side in a workgroup, with their keys in one share and in several
    at = torch.randint(-1, S + 1, (B,), generator=rng(B)).tolist()
    check_attention(dtype, bits, H, G, D, S, 1, at, seed=D, decode=True, cap=30.0 if D == 64 else None,
                    slopes=[2.0 ** -(1 + h % 8) for h in range(H)] if D == 96 else None)
    if H // G > 1:
        check_attention(dtype, bits, H, G, D, S, 2, at[:32] if B > 32 else at, seed=D)


@pytest.mark.parametrize("bits, dtype", [(4, "bf16"), (8, "fp32")])
def test_decode_of_many_long_caches(bits, dtype):
    """As many sequences as fill the card alone: key heads side by side, each sequence's keys in one workgroup."""
    dt, g = TYPES[dtype], rng(21)
    B, G, D, S = 256, 16, 16, 4100
    cache = cf.quantized_cache(B, S, G, D, bits)
    k, v, q = (normal(g, B, 40, G, D, dtype=dt).cuda() for _ in range(3))
    lens = torch.randint(0, S, (B,), generator=g).int()
    lens[:6] = torch.tensor([0, 1, S - 1, S, -1, 4000])
    cf.quantized_cache_write(cache, k[:, 1:], v[:, 1:], (lens - 39).clamp_min(0).cuda())       # the last ones it holds
    y, _ = cf.softmax_attention_decode(q[:, 0], k[:, 0], v[:, 0], cache, lens.cuda(), softcap=20.0)
    assert torch.isnan(y[3]).all() and (y[4] == 0).all()
    for b in (0, 1, 2, 5, 6, 77, 255):
        n = int(lens[b]) + 1
        kk, vv = (Q.held(cache[x][b:b + 1, :n], cache[x + "_scale"][b:b + 1, :n]) for x in ("k", "v"))
        assert torch.equal(kk[:, n - 1], Q.rounded(k[b:b + 1, 0].cpu(), bits)[0])
        ref, tol = M.attention(q[b:b + 1, :1], kk, vv, softcap=20.0, offset=[n - 1], unit=0.0 if dtype == "fp32" else M.U[dt],
                               tiny=2.0 ** -126)["y"]
        M.check(y[b:b + 1], ref, tol + M.U[dt] * ref.abs(), f"y of sequence {b}", dt)


@pytest.mark.parametrize("bits", [4, 8])
def test_decode_of_large_scores(bits):
    # weights that move the reference again and again, and rows whose first keys count for nothing
    check_attention("bf16", bits, 4, 1, 128, 900, 1, [899, 640], seed=5, decode=True, q_std=60.0)
    check_attention("fp32", bits, 4, 1, 64, 900, 1, [899, 640], seed=5, decode=True, q_std=60.0)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("H, G, D, T", [(4, 4, 64, 2), (4, 4, 128, 16), (4, 4, 80, 17), (8, 2, 128, 4), (8, 2, 48, 5), (8, 2, 96, 8),
                                        (8, 1, 128, 8), (8, 1, 32, 9), (16, 1, 64, 4), (6, 2, 112, 21), (6, 2, 16, 22)])
def test_drafts(dtype, bits, H, G, D, T):
    check_attention(dtype, bits, H, G, D, 333, T, [0, 333 - T, 334 - T, -3, 60, 129], seed=T)
    check_attention(dtype, bits, H, G, D, 333, T, [0, 333 - T, 5, 64 - T], new=[T - 1, T, 0, 1], seed=T,
                    prefix=[T // 2, 333, 2, 0], cap=25.0, slopes=[0.5 / (1 + h) for h in range(H)])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("H, G, D, T", [(4, 4, 128, 65), (4, 2, 64, 150), (3, 1, 96, 129), (2, 2, 80, 190), (2, 1, 32, 70), (2, 2, 16, 66)])
def test_prompts(dtype, bits, H, G, D, T):
    S = T + 90
    check_attention(dtype, bits, H, G, D, S, T, [0, 90, 91, -1, 37], seed=T)
    check_attention(dtype, bits, H, G, D, S, T, [64, 3, 90, 0], new=[T - 7, 1, T, 0], prefix=[100, 3, 0, 5], seed=T)
    check_attention(dtype, bits, H, G, D, S, T, [33], cap=12.0, seed=T)
    check_attention(dtype, bits, H, G, D, S, T, [33], cap=300.0, slopes=[0.25 / (1 + h) for h in range(H)], seed=T)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("H, G, D, T", [(4, 4, 64, 128), (2, 2, 128, 250), (3, 1, 80, 256), (4, 4, 16, 131), (2, 1, 96, 384), (2, 2, 32, 200),
                                        (8, 1, 48, 256), (16, 2, 128, 270), (8, 1, 96, 300), (16, 1, 64, 129), (8, 1, 32, 257)])
def test_longer_prompts(dtype, bits, H, G, D, T):
    S = T + 70
    check_attention(dtype, bits, H, G, D, S, T, [0, 70, 71, -1, 33], seed=T)
    check_attention(dtype, bits, H, G, D, S, T, [64, 3], new=[T - 7, 0], prefix=[100, 3], seed=T, cap=20.0)
    check_attention(dtype, bits, H, G, D, S, T, [70], cap=300.0, slopes=[0.25 / (1 + h) for h in range(H)], seed=T)


@pytest.mark.parametrize("bits", [4, 8])
def test_prompts_of_a_large_cache(bits):
    # long rooms of many sequences: more values than are turned into 16 bits at a time
    check_attention("bf16", bits, 4, 1, 64, 1 << 20, 512, [0, 200, (1 << 20) - 512, 5, (1 << 20) - 511, 31],
                    new=[512, 7, 0, 512, 512, 500], seed=3)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_parts_of_long_caches(dtype):
    # keys split over workgroups, of a token, of drafts and of a prompt
    check_attention(dtype, 4, 4, 1, 64, 5000, 1, [4999, 3000, 0], seed=1, decode=True)
    check_attention(dtype, 4, 4, 1, 64, 5000, 9, [4991, 2500], seed=2)
    check_attention(dtype, 8, 2, 1, 128, 3500, 80, [3420, 1100], new=[80, 33], seed=3)


def _visible_nan(dtype, bits, T, H, G, D, S, off, places):
    """y where the tokens `places` of the new ones have a NaN or an infinite value in v: rows that see one are NaN
    there, in its block, and no others."""
    dt, g = TYPES[dtype], rng(9)
    k, v, q = normal(g, 1, T, G, D, dtype=dt), normal(g, 1, T, G, D, dtype=dt), normal(g, 1, T, H, D, dtype=dt)
    bad = v.clone()
    for t, d, x in places:
        bad[0, t, :, d] = x
    out = []
    for values in (v, bad):
        cache = filled(rng(1), 1, S, G, D, bits)
        cf.quantized_cache_write(cache, normal(rng(2), 1, off, G, D, dtype=dt).cuda(), normal(rng(3), 1, off, G, D, dtype=dt).cuda(),
                                 ints(0))
        out.append(cf.softmax_attention_prefill(q.cuda(), k.cuda(), values.cuda(), cache, ints(off))[0].cpu())
    want = torch.zeros((1, T, H, D), dtype=torch.bool)
    for t, d, x in places:
        want[0, t:, :, d // 32 * 32:(d // 32 + 1) * 32] = True
    assert torch.equal(torch.isnan(out[1]), want)
    # the others' weights are the same; the value of the block's other elements is not theirs to see
    assert torch.equal(out[1][~want], out[0][~want])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("bits", [4, 8])
def test_nan_reaches_the_rows_that_see_it(dtype, bits):
    _visible_nan(dtype, bits, 6, 4, 2, 128, 200, 100, [(3, 40, math.nan), (5, 0, math.inf)])
    _visible_nan(dtype, bits, 16, 2, 2, 80, 200, 60, [(9, 79, -math.inf)])
    _visible_nan(dtype, bits, 150, 2, 1, 64, 400, 130, [(70, 5, math.nan), (149, 63, math.inf)])
    _visible_nan(dtype, bits, 200, 2, 2, 96, 400, 130, [(70, 5, math.nan), (199, 63, math.inf)])
    _visible_nan(dtype, bits, 256, 8, 1, 64, 400, 130, [(70, 5, math.nan), (255, 63, math.inf)])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("T, H, G, D", [(6, 4, 2, 128), (200, 2, 2, 96), (256, 8, 1, 64)])
def test_nan_keys_reach_the_rows_that_see_them(dtype, bits, T, H, G, D):
    dt, g = TYPES[dtype], rng(5)
    off, S = 60, T + 70
    k, v, q = normal(g, 1, T, G, D, dtype=dt), normal(g, 1, T, G, D, dtype=dt), normal(g, 1, T, H, D, dtype=dt)
    at = T - 3
    bad = k.clone()
    bad[0, at, 0, 7] = math.inf
    old = [normal(g, 1, off, G, D, dtype=dt).cuda() for _ in range(2)]
    out = []
    for keys in (k, bad):
        cache = cf.quantized_cache(1, S, G, D, bits)
        cf.quantized_cache_write(cache, *old, ints(0))
        out.append(cf.softmax_attention_prefill(q.cuda(), keys.cuda(), v.cuda(), cache, ints(off))[0].cpu())
    want = torch.zeros((1, T, H, D), dtype=torch.bool)
    want[0, at:, :H // G] = True
    assert torch.equal(torch.isnan(out[1]), want)
    assert torch.equal(out[1][~want], out[0][~want])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T, H, G, D", [(1, 4, 2, 64), (6, 4, 2, 128), (200, 2, 2, 96), (256, 8, 1, 64)])
def test_infinite_queries(dtype, T, H, G, D):
    """A query with an infinite element: its scores are infinite, or of the cap; other rows know nothing of it."""
    dt, g = TYPES[dtype], rng(15)
    off, S = 60, T + 70
    k, v, q = normal(g, 1, T, G, D, dtype=dt), normal(g, 1, T, G, D, dtype=dt), normal(g, 1, T, H, D, dtype=dt)
    old = [normal(g, 1, off, G, D, dtype=dt) for _ in range(2)]
    for x in (k, old[0]):
        x[..., 5] = torch.where(x[..., 5].abs() < 0.25, 0.25, x[..., 5])       # no code of 0 there
    t0, h0 = T // 2, H - 1
    odd = q.clone()
    odd[0, t0, h0, 5] = -math.inf
    for cap in (None, 7.0):
        out = []
        for queries in (q, odd):
            cache = cf.quantized_cache(1, S, G, D, 8)
            cf.quantized_cache_write(cache, *(x.cuda() for x in old), ints(0))
            out.append(cf.softmax_attention_prefill(queries.cuda(), k.cuda(), v.cuda(), cache, ints(off), softcap=cap)[0].cpu())
        rest = torch.ones((1, T, H, D), dtype=torch.bool)
        rest[0, t0, h0] = False
        assert torch.equal(out[0][rest], out[1][rest])
        n = off + t0 + 1
        kk, vv = (Q.held(cache[x][0, :n, -1], cache[x + "_scale"][0, :n, -1]) for x in ("k", "v"))
        assert (kk[:, 5] != 0).all() and (kk[:, 5] < 0).any()
        if cap is None:
            assert torch.isnan(out[1][0, t0, h0]).all()           # one of the scores is +inf
        else:
            w = torch.softmax(-cap * torch.sign(kk[:, 5]), 0)
            ref, mag = w @ vv, w @ vv.abs()
            u = M.U[dt] if dt is not torch.float32 else 0.0
            M.check(out[1][0, t0, h0], ref, (u + 2.0 ** -18) * mag + M.U[dt] * ref.abs(), "y", dt)


@pytest.mark.parametrize("T, pieces", [(150, (70, 1, 9, 66, 4)), (20, (1,) * 20)])
@pytest.mark.parametrize("bits", [4, 8])
def test_a_prompt_in_pieces(bits, T, pieces):
    g = rng(4)
    H, G, D, S = 8, 2, 96, 200
    k, v, q = (normal(g, 2, T, h, D, dtype=torch.bfloat16).cuda() for h in (G, G, H))
    whole, parts = cf.quantized_cache(2, S, G, D, bits), cf.quantized_cache(2, S, G, D, bits)
    y, _ = cf.softmax_attention_prefill(q, k, v, whole, ints(0, 0))
    at, got = 0, []
    for n in pieces:
        now = slice(at, at + n)
        if n == 1:
            out = cf.softmax_attention_decode(q[:, now], k[:, now], v[:, now], parts, ints(at, at))[0]
        else:
            out = cf.softmax_attention_prefill(q[:, now], k[:, now], v[:, now], parts, ints(at, at))[0]
        got.append(out)
        at += n
    for n in PARTS:
        assert torch.equal(whole[n].view(torch.uint8), parts[n].view(torch.uint8)), n
    ref, tol = M.attention(q, *(Q.held(whole[n][:, :T], whole[n + "_scale"][:, :T]) for n in ("k", "v")), unit=M.U[torch.bfloat16],
                           tiny=2.0 ** -126)["y"]
    for out in (y, torch.cat(got, 1)):
        M.check(out, ref, tol + M.U[torch.bfloat16] * ref.abs(), "y", torch.bfloat16)


def test_strides_and_other_integers():
    g = rng(8)
    B, H, G, D, S = 3, 8, 2, 64, 100
    fused = normal(g, B, 7, H + 2 * G, D, dtype=torch.bfloat16).cuda()
    q, k, v = fused[:, :, :H], fused[:, :, H:H + G], fused[:, :, H + G:]
    a, b = cf.quantized_cache(B, S, G, D, 4), cf.quantized_cache(B, S, G, D, 4)
    ya, _ = cf.softmax_attention_prefill(q, k, v, a, ints(0, 5, 93))
    yb, _ = cf.softmax_attention_prefill(*(t.contiguous() for t in (q, k, v)), b, ints(0, 5, 93).long())
    assert torch.equal(ya, yb)
    for n in PARTS:
        assert torch.equal(a[n], b[n])
    # unaligned rows are copied
    odd = torch.empty(B * 7 * (H + 1) * D + 1, dtype=torch.bfloat16, device="cuda")[1:1 + B * 7 * H * D].view(B, 7, H, D)
    odd.copy_(q)
    yc, _ = cf.softmax_attention_prefill(odd, k, v, b, ints(0, 5, 93))
    assert torch.equal(ya, yc)
    # single tokens with and without their dimension of one
    t1, _ = cf.softmax_attention_decode(q[:, 0], k[:, 0], v[:, 0], a, ints(7, 12, -1))
    t2, _ = cf.softmax_attention_decode(q[:, :1], k[:, :1], v[:, :1], b, ints(7, 12, -1))
    assert torch.equal(t1, t2)


def test_empty_calls():
    cache = cf.quantized_cache(2, 8, 2, 32, 8)
    e = torch.empty((2, 0, 4, 32), device="cuda")
    y, _ = cf.softmax_attention_prefill(e, e[:, :, :2], e[:, :, :2], cache, ints(0, 0))
    assert y.shape == (2, 0, 4, 32)
    assert cf.quantized_cache_write(cache, e[:, :, :2], e[:, :, :2], ints(0, 0)) is cache
    assert cf.quantized_cache_read(cache, count=0)[0].shape == (2, 0, 2, 32)
    none = cf.quantized_cache(0, 8, 2, 32, 4)
    z = torch.empty((0, 2, 32), device="cuda")
    assert cf.softmax_attention_decode(z, z, z, none, torch.empty(0, dtype=torch.int32, device="cuda"))[0].shape == (0, 1, 2, 32)
    assert all((cache[n].view(torch.uint8) == 0).all() for n in PARTS)


@pytest.mark.parametrize("bits", [4, 8])
def test_captured_tokens_and_drafts(bits):
    """A graph of decode steps and drafts, replayed with other inputs and lengths, against the calls themselves."""
    g = rng(6)
    B, H, G, D, S = 4, 8, 2, 128, 600
    for T in (1, 3, 40):
        cache, plain = cf.quantized_cache(B, S, G, D, bits), cf.quantized_cache(B, S, G, D, bits)
        q, k, v = (normal(g, B, T, h, D, dtype=torch.bfloat16).cuda() for h in (H, G, G))
        lens = torch.zeros(B, dtype=torch.int32, device="cuda")

        def call(to, at):
            if T == 1:
                return cf.softmax_attention_decode(q, k, v, to, at)[0]
            return cf.softmax_attention_prefill(q, k, v, to, at)[0]

        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            call(cache, lens)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call(cache, lens)
            lens += T
        lens.zero_()
        at = torch.zeros(B, dtype=torch.int32, device="cuda")
        for step in range(5):
            for t, h in ((q, H), (k, G), (v, G)):
                t.copy_(normal(g, B, T, h, D, dtype=torch.bfloat16))
            graph.replay()
            want = call(plain, at)
            at += T
            torch.cuda.synchronize()
            assert torch.equal(y, want), (T, step)
            for n in PARTS:
                assert torch.equal(cache[n].view(torch.uint8), plain[n].view(torch.uint8)), (T, step, n)


@pytest.mark.parametrize("T", [128, 512])
def test_captured_prompts(T):
    """A graph of a prompt, by codes and by values turned into 16 bits, replayed with other inputs and lengths."""
    g = rng(16)
    B, H, G, D, S = 3, 8, 2, 96, 1700
    cache, plain = cf.quantized_cache(B, S, G, D, 4), cf.quantized_cache(B, S, G, D, 4)
    q, k, v = (normal(g, B, T, h, D, dtype=torch.float16).cuda() for h in (H, G, G))
    lens, new = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")

    def call(to):
        return cf.softmax_attention_prefill(q, k, v, to, lens, softcap=30.0, new_lengths=new)[0]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call(cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call(cache)
    for step in range(4):
        for t, h in ((q, H), (k, G), (v, G)):
            t.copy_(normal(g, B, T, h, D, dtype=torch.float16))
        new.copy_(torch.randint(0, T + 1, (B,), generator=g))
        graph.replay()
        want = call(plain)
        torch.cuda.synchronize()
        assert torch.equal(y, want), step
        for n in PARTS:
            assert torch.equal(cache[n].view(torch.uint8), plain[n].view(torch.uint8)), (step, n)
        lens += new


def test_calls_on_two_streams():
    g = rng(7)
    H, G, D, S = 8, 2, 64, 3000
    sets = []
    for i in range(2):
        cache = cf.quantized_cache(2, S, G, D, 4)
        cf.quantized_cache_write(cache, *(normal(g, 2, S - 10, G, D, dtype=torch.bfloat16).cuda() for _ in range(2)), ints(0, 0))
        sets.append((cache, [normal(g, 2, h, D, dtype=torch.bfloat16).cuda() for h in (H, G, G)]))
    lens = ints(S - 10, S - 500)
    alone = [cf.softmax_attention_decode(*x, cache, lens)[0].clone() for cache, x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        out = []
        for s, (cache, x) in zip(streams, sets):
            with torch.cuda.stream(s):
                out.append(cf.softmax_attention_decode(*x, cache, lens)[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(alone, out))


def test_offsets_past_32_bits():
    """A cache whose codes pass 2^32 bytes: its last sequence's rows are found."""
    B, S, G, D = 5, 1 << 20, 8, 128
    cache = cf.quantized_cache(B, S, G, D, 8)
    assert cache["k"].numel() > 2 ** 32
    g = rng(3)
    k, v, q = (normal(g, B, 40, h, D, dtype=torch.bfloat16).cuda() for h in (G, G, 8))
    lens = torch.full((B,), S - 50, dtype=torch.int32, device="cuda")
    # all but the last few tokens are zeros: their weights are equal and they add nothing to y
    y, _ = cf.softmax_attention_prefill(q, k, v, cache, lens)
    t, _ = cf.softmax_attention_decode(q[:, 0], k[:, 0], v[:, 0], cache, lens + 40)
    got = cf.quantized_cache_read(cache, lens, 41, torch.float32)
    for x, new in zip(got, (k, v)):
        want = Q.rounded(torch.cat((new, new[:, :1]), 1).cpu(), 8)[0]
        assert torch.equal(x.double().cpu(), want)
    kk, vv = got[0].double(), got[1].double()
    for b in (0, B - 1):
        for i, (row, n, off) in enumerate(((y[b, 39], 40, S - 50), (t[b, 0], 41, S - 50))):
            qq = (q[b, 39] if i == 0 else q[b, 0]).double()
            s = torch.einsum("hd,nhd->hn", qq.cpu(), kk[b, :n].cpu()) * D ** -0.5
            w = torch.exp(s)
            ref = (w[:, :, None] * vv[b, :n].cpu().transpose(0, 1)).sum(1) / (w.sum(1, keepdim=True) + off)
            # weights and y rounded to bf16, sums over a million terms in 32 bits
            mag = (w[:, :, None] * vv[b, :n].cpu().transpose(0, 1).abs()).sum(1) / (w.sum(1, keepdim=True) + off)
            M.check(row, ref, (2 * M.U[torch.bfloat16] + 2.0 ** -10) * mag, "y", torch.bfloat16)


@pytest.mark.parametrize("bits", [4, 8])
def test_rows_beyond_32_bits_are_outside(bits):
    cache = filled(rng(23), 6, 9, 2, 32, bits)
    at = torch.tensor([2 ** 32, -2 ** 32, 2 ** 32 + 3, 2 ** 31, -2 ** 40 + 1, 4], device="cuda")
    got = cf.quantized_cache_read(cache, at, 3, torch.float32)
    for n, x in zip(("k", "v"), got):
        assert (x[:5] == 0).all()
        want = Q.held(cache[n][5, 4:7], cache[n + "_scale"][5, 4:7]).float()
        assert torch.equal(x[5].cpu().nan_to_num(nan=7e37), want.nan_to_num(nan=7e37))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_prompts_by_codes_of_a_large_room(dtype, bits):
    """As many blocks of queries as have values turned into 16 bits first, in rooms whose values would pass 1 GiB."""
    dt, g = TYPES[dtype], rng(24)
    B, T, H, G, D, S = 2, 200, 8, 1, 128, (1 << 21) + 64
    cache = cf.quantized_cache(B, S, G, D, bits)
    q, k, v = (normal(g, B, T, h, D, dtype=dt) for h in (H, G, G))
    old = [normal(g, B, 70, G, D, dtype=dt).cuda() for _ in range(2)]
    cf.quantized_cache_write(cache, *old, ints(0, 0))
    y, _ = cf.softmax_attention_prefill(q.cuda(), k.cuda(), v.cuda(), cache, ints(33, S - T + 1), new_lengths=ints(T - 3, T),
                                        prefix_lengths=ints(50, 0))
    assert torch.isnan(y[1]).all() and (y[0, T - 3:] == 0).all()
    n = 33 + T - 3
    kk, vv = (Q.held(cache[x][:1, :n], cache[x + "_scale"][:1, :n]) for x in ("k", "v"))
    assert torch.equal(kk[:, 33:], Q.rounded(k[:1, :T - 3], bits)[0])
    ref, tol = M.attention(q[:1, :T - 3], kk, vv, offset=[33], prefix=[50], unit=M.U[dt],
                           tiny=2.0 ** -25 if dtype == "fp16" else 2.0 ** -126)["y"]
    M.check(y[:1, :T - 3], ref, tol + M.U[dt] * ref.abs(), "y", dt)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("T, H, G, D", [(1, 4, 2, 64), (6, 4, 2, 128), (40, 4, 2, 80), (200, 2, 2, 96), (256, 8, 1, 64)])
def test_fp16_attention_over_what_bf16_wrote(bits, T, H, G, D):
    """Queries of fp16 see what a cache holds rounded to fp16, infinite beyond its range, whichever kernel takes them."""
    g = rng(25)
    off, S = 100, T + 110
    old = [normal(g, 3, off, G, D) * 2.0 ** torch.randint(-30, 3, (3, off, G, 1), generator=g) for _ in range(2)]
    old[1][1, 77, 0, 5], old[1][1, 77, 0, 6], old[1][1, 99, G - 1, D - 1] = 1e5, -1e5, 3e38
    old[0][2, 88, 0, 3] = 1e5
    cache = cf.quantized_cache(3, S, G, D, bits)
    cf.quantized_cache_write(cache, *(t.bfloat16().cuda() for t in old), ints(0, 0, 0))
    k, v, q = normal(g, 3, T, G, D).half(), normal(g, 3, T, G, D).half(), normal(g, 3, T, H, D).half()
    y, _ = cf.softmax_attention_prefill(q.cuda(), k.cuda(), v.cuda(), cache, ints(off, off, off))
    y = y.cpu()
    kk, vv = (Q.held(cache[x][:, :off + T], cache[x + "_scale"][:, :off + T]).half().double() for x in ("k", "v"))

    def near(b, heads, keys, values, odd, before):
        ref, tol = M.attention(q[b:b + 1, :, heads], keys[None], values[None], offset=[before], unit=M.U[torch.float16], tiny=2.0 ** -25)["y"]
        M.check(y[b:b + 1, :, heads].masked_fill(odd, 0.0), ref.masked_fill(odd, 0.0), tol + M.U[torch.float16] * ref.abs(),
                f"y of sequence {b}", torch.float16)
    every, no = slice(0, H), torch.zeros(1, dtype=torch.bool)
    near(0, every, kk[0], vv[0], no, off)
    # infinite values: whatever their weight, y is infinite in their dimension, with their sign, and nowhere else
    infinite = torch.isinf(vv[1])
    assert infinite[77, 0, 5] and infinite[77, 0, 6] and infinite[99, G - 1, D - 1]
    odd = infinite.any(0).repeat_interleave(H // G, 0).expand(T, H, D)
    sign = torch.where(infinite, vv[1].sign(), 0.0).sum(0).repeat_interleave(H // G, 0).expand(T, H, D)
    assert (y[1][odd] == sign[odd] * math.inf).all()
    near(1, every, kk[1], vv[1].masked_fill(infinite, 0.0), odd, off)
    # a key's infinite element: a score of +inf (or, of 0 times it, NaN) makes a row NaN; one of -inf has a weight of 0
    assert torch.isinf(kk[2]).nonzero().tolist() == [[88, 0, 3]]
    none = (q[2, :, :H // G, 3] >= 0)[..., None].expand(T, H // G, D)
    assert torch.isnan(y[2, :, :H // G][none]).all()
    rest = torch.arange(off + T) != 88
    near(2, slice(0, H // G), kk[2][rest][:, :1], vv[2][rest][:, :1], none, off - 1)
    if G > 1:
        near(2, slice(H // G, H), kk[2][:, 1:], vv[2][:, 1:], no, off)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype, B, H, G, D, T", [("bf16", 32, 4, 4, 128, 5), ("bf16", 66, 4, 2, 80, 6), ("fp16", 32, 8, 4, 64, 8),
                                                  ("fp32", 32, 8, 4, 128, 16), ("fp32", 64, 2, 2, 48, 9)])
def test_nan_with_key_heads_side_by_side(dtype, bits, B, H, G, D, T):
    """Drafts of as many sequences as let a workgroup's waves take several key heads: NaN keys and values of one head reach the
    rows of its own queries that see them."""
    dt, g = TYPES[dtype], rng(26)
    S = 90
    lens = torch.randint(0, S - T + 1, (B,), generator=g).int()
    old = [normal(g, B, S - T, G, D, dtype=dt).cuda() for _ in range(2)]
    k, v, q = normal(g, B, T, G, D, dtype=dt), normal(g, B, T, G, D, dtype=dt), normal(g, B, T, H, D, dtype=dt)
    bad_k, bad_v = k.clone(), v.clone()
    want = torch.zeros((B, T, H, D), dtype=torch.bool)
    R = H // G
    for b in range(B):
        at, h, d = b % T, b // 2 % G, 7 * b % D
        if b % 3 == 0:
            bad_v[b, at, h, d] = math.nan
            want[b, at:, h * R:(h + 1) * R, d // 32 * 32:(d // 32 + 1) * 32] = True
        if b % 3 == 1:
            bad_k[b, at, h, d] = math.inf
            want[b, at:, h * R:(h + 1) * R] = True
    out = []
    for keys, values in ((k, v), (bad_k, bad_v)):
        cache = cf.quantized_cache(B, S, G, D, bits)
        cf.quantized_cache_write(cache, *old, torch.zeros_like(lens).cuda())
        out.append(cf.softmax_attention_prefill(q.cuda(), keys.cuda(), values.cuda(), cache, lens.cuda())[0].cpu())
    assert torch.equal(torch.isnan(out[1]), want)
    assert torch.equal(out[1][~want], out[0][~want])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype, B, H, G, D, T", [("fp32", 33, 8, 4, 128, 16), ("fp32", 64, 8, 2, 64, 15), ("fp32", 32, 4, 4, 80, 11),
                                                  ("bf16", 64, 2, 2, 96, 16), ("fp16", 32, 8, 4, 112, 8)])
def test_drafts_with_key_heads_side_by_side(dtype, bits, B, H, G, D, T):
    S = 140
    g = rng(27)
    at = torch.randint(-1, S - T + 2, (B,), generator=g).tolist()
    check_attention(dtype, bits, H, G, D, S, T, at, seed=D)
    check_attention(dtype, bits, H, G, D, S, T, at, new=torch.randint(0, T + 1, (B,), generator=g).tolist(), seed=D, cap=25.0,
                    prefix=torch.randint(0, S, (B,), generator=g).tolist(), slopes=[0.5 / (1 + h) for h in range(H)])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("T, H, G, D", [(5, 8, 4, 128), (16, 2, 2, 80), (40, 4, 2, 64), (150, 2, 1, 96), (256, 8, 1, 64)])
def test_padding_holds_anything(dtype, bits, T, H, G, D):
    """Rows behind new_lengths, and all of a sequence that sits out, are NaN; lengths of new tokens and prefixes beyond their
    ends count as these."""
    dt, g = TYPES[dtype], rng(28)
    B, S = 5, T + 60
    lens, new = ints(0, 50, 60, -7, 33), (T - 2, 0, T + 9, T, 1)
    q, k, v = normal(g, B, T, H, D, dtype=dt), normal(g, B, T, G, D, dtype=dt), normal(g, B, T, G, D, dtype=dt)
    old = [normal(g, B, 60, G, D, dtype=dt).cuda() for _ in range(2)]
    bad = [x.clone() for x in (q, k, v)]
    for b in range(B):
        for x in bad:
            x[b, 0 if b == 3 else min(new[b], T):] = math.nan
    out = []
    for i, tensors in enumerate(((q, k, v), bad)):
        cache = cf.quantized_cache(B, S, G, D, bits)
        cf.quantized_cache_write(cache, *old, torch.zeros_like(lens))
        fresh, prefix = (ints(*(min(n, T) for n in new)), ints(0, 50, S, 0, 20)) if i == 0 else \
            (ints(T - 2, -1, T + 9, T, 1), ints(-4, 2 ** 31 - 1, 2 ** 30, 5, 20))
        y, _ = cf.softmax_attention_prefill(*(x.cuda() for x in tensors), cache, lens, prefix_lengths=prefix, new_lengths=fresh)
        out.append((y, raw(cache)))
    assert torch.isfinite(out[0][0]).all() and torch.equal(out[0][0], out[1][0])
    for n in PARTS:
        assert torch.equal(out[0][1][n], out[1][1][n]), n
