"""Positions and quantised caches for softmax attention: what is measured of them.

Rotary positions of queries and keys, a cache whose keys and values are held in 8 or 4 bits, and
softmax attention over such a cache.  Each is called as a program calls it: in a training step,
over prompts that continue a cache, and for one token or a few drafted ones a sequence while
answering.

A quantised cache holds its values in blocks of 32 along a head (the last one may be shorter):
e4m3 or e2m1 codes times a power of 2 of the block's own, the least by which the block's largest
value rounds to one that the codes have.

``listed`` holds the fixed cases and ``draw`` one more of the same ranges.  With ``own``
false ``run`` computes a case in plain torch operations in 32 bits; with ``own`` true it
calls the package.  ``exact`` gives the same outputs in 64 bits, from the definitions.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 32


# ---------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------
def _rotary(name, kind, dtype, B, N, H, G, D, turned=None, interleaved=False, factor=1.0, parts=False, far=0, docs=0):
    """turned: dimensions of a head that are rotated.  factor: of longer contexts, by parts of the
    frequencies or for all alike.  far: where positions start.  docs: documents that a row is packed from."""
    case = {"op": "rotary", "kind": kind, "dtype": dtype, "B": B, "N": N, "H": H, "G": G, "D": D,
            "turned": turned or D, "interleaved": interleaved, "factor": factor, "parts": parts, "far": far, "docs": docs}
    return dict(case, name=name) if name else case


def _cache(name, kind, dtype, bits, B, N, G, D, S):
    case = {"op": "cache", "kind": kind, "dtype": dtype, "bits": bits, "B": B, "N": N, "G": G, "D": D, "S": S}
    return dict(case, name=name) if name else case


def _attend(name, dtype, bits, B, N, H, G, D, S, cap=0.0, slopes=False, prefix=False):
    case = {"op": "attend", "kind": "decode" if N == 1 else "prefill", "dtype": dtype, "bits": bits, "B": B, "N": N,
            "H": H, "G": G, "D": D, "S": S, "cap": cap, "slopes": slopes, "prefix": prefix}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one token for each sequence of a serving batch: a launch and its latency
        _rotary("rotary_step", "decode", "bf16", 64, 1, 16, 4, 128),
        # the training step of a mid-size layer whose context is being lengthened, shared key heads
        _rotary("rotary_train", "train", "bf16", 4, 4096, 16, 4, 128, factor=8.0, parts=True),
        # full precision over packed documents of an odd total length, half of each head in adjacent pairs
        _rotary("rotary_train_fp32", "train", "fp32", 2, 2011, 8, 8, 64, turned=32, interleaved=True, docs=5),
        # prompts of a padded batch, written into a cache of 4 bits and taken back as the cache holds them
        _cache("cache_prompt", "write", "bf16", 4, 4, 4096, 16, 128, 8192),
        # a whole cache of 8 bits as 16-bit tensors, for operators that read these
        _cache("cache_read", "read", "bf16", 8, 16, 8192, 4, 128, 8192),
        # one token a sequence against a cache of some thousands, shared key heads, capped scores
        _attend("attend_step", "bf16", 4, 64, 1, 16, 4, 128, 8192, cap=30.0),
        # the same with a key head for each query head and a bias on distance
        _attend("attend_step_8", "fp16", 8, 16, 1, 16, 16, 64, 4096, slopes=True),
        # one sequence and a short cache: launches and their latency
        _attend("attend_step_one", "bf16", 4, 1, 1, 16, 4, 128, 1000),
        # a few drafted tokens a sequence against long caches, odd in number
        _attend("attend_drafts", "bf16", 8, 16, 5, 16, 4, 128, 8192),
        # follow-up prompts of odd lengths into caches, with a prefix that sees itself whole
        _attend("attend_prompt", "fp16", 4, 3, 1531, 16, 4, 128, 4096, prefix=True),
        # a long follow-up of one sequence behind a longer cache
        _attend("attend_prompt_long", "bf16", 4, 1, 4096, 16, 4, 128, 16384),
        # full precision, as a check or a small model runs it
        _attend("attend_prompt_fp32", "fp32", 8, 2, 257, 8, 8, 64, 1021),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rotary", "rotary", "cache", "attend", "attend", "attend", "attend"))
    dtype = rng.choice(("bf16", "bf16", "bf16", "fp16", "fp32"))
    bits = rng.choice((4, 4, 8))
    G = rng.choice((1, 2, 4, 8))
    H = G * rng.choice((1, 1, 2, 4, 8) if G <= 2 else (1, 2, 4))
    D = rng.choice((32, 48, 64, 64, 80, 96, 128, 128))
    if op == "rotary":
        kind = rng.choice(("decode", "prefill", "train"))
        B = _log_int(rng, 1, 64) if kind == "decode" else _log_int(rng, 1, 8)
        N = 1 if kind == "decode" else _log_int(rng, 40, max(80, min(16384, 2 ** 18 // (B * H))))
        turned = rng.choice((None, None, D // 2, 16))
        return _rotary(None, kind, dtype, B, N, H, G, D, turned, rng.random() < 0.3, rng.choice((1.0, 1.0, 4.0, 8.0)),
                       rng.random() < 0.5, rng.choice((0, 0, 100000)), rng.choice((0, 1, 3, 8)) if kind == "train" else 0)
    if op == "cache":
        kind = rng.choice(("write", "read"))
        B = _log_int(rng, 1, 16)
        S = _log_int(rng, 40, max(80, min(16384, 2 ** 19 // (B * G))))
        N = _log_int(rng, 1, max(1, S - S // 4)) if kind == "write" else S
        return _cache(None, kind, dtype, bits, B, N, G, D, S)
    cap = rng.choice((0.0, 0.0, 20.0, 50.0))
    slopes = rng.random() < 0.4
    kind = rng.choice(("decode", "decode", "drafts", "prompt"))
    if kind == "prompt":
        B = _log_int(rng, 1, 8)
        N = _log_int(rng, 17, max(40, min(4096, 2 ** 16 // (B * H))))
        S = N + _log_int(rng, 1, 8192 // B)
    else:
        B = _log_int(rng, 1, 64)
        N = 1 if kind == "decode" else rng.randint(2, 16)
        S = _log_int(rng, 64, min(8192, 8192 * 16 * 64 // (B * H * N))) + N
    return _attend(None, dtype, bits, B, N, H, G, D, S, cap, slopes, N > 1 and rng.random() < 0.3)


# ---------------------------------------------------------------------------------------
# Codes
# ---------------------------------------------------------------------------------------
# Of each code: the largest value, what a block's largest value may be at a scale of 1 (as a mantissa
# below 1 and a power of 2: 7 and 464), and the exponents that a scale may have for 16-bit floats of 5
# bits of exponent and for wider ones (so that every value a cache holds is one of the type that it was
# written from).
_FORMS = {4: (6.0, 0.875, 3, (-23, 13), (-125, 125)), 8: (448.0, 0.90625, 9, (-15, 7), (-117, 119))}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _power(e):
    """2^e in 32 bits, exactly, for whole e from -126 to 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x, bits):
    """Codes and scales of x [.., D]: e4m3 [.., D] or two e2m1 a byte [.., D / 2] (the lower half first),
    and exponents + 127 [.., blocks]; 255 for a block with a value that is not finite."""
    D = x.shape[-1]
    most, room, room_power, narrow, wide = _FORMS[bits]
    lo, hi = narrow if x.dtype is torch.float16 else wide
    n = -(-D // BLOCK)
    w = torch.nn.functional.pad(x.float(), (0, n * BLOCK - D)).unflatten(-1, (n, BLOCK))
    top = w.abs().amax(-1)
    part, power = torch.frexp(top)                         # the least e with top <= room 2^e
    e = (power - room_power + (part > room).int()).clamp(lo, hi)
    odd = ~torch.isfinite(top)
    e = torch.where(odd | (top == 0), lo, e)
    v = (w * _power(-e)[..., None]).clamp(-most, most)
    v = torch.where(odd[..., None], 0.0, v)
    scale = torch.where(odd, 255, e + 127).to(torch.uint8)
    v = v.flatten(-2)[..., :D]
    if bits == 8:
        return v.to(torch.float8_e4m3fn), scale
    a = v.abs()
    # steps of a half up to 2, of one up to 4 and of two from there, ties to the even code
    code = torch.where(a < 2, (a * 2).round(), torch.where(a < 4, a.round() + 2, (a / 2).round() + 4))
    code = code.to(torch.uint8) + 8 * torch.signbit(v).to(torch.uint8)
    return code[..., ::2] + 16 * code[..., 1::2], scale


def _values(codes, scale, D):
    """What codes and scales stand for, in 32 bits."""
    if codes.dtype is torch.uint8:
        table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=codes.device)
        v = table[torch.stack((codes % 16, codes // 16), -1).flatten(-2).int()]
    else:
        v = codes.float()
    factor = torch.where(scale == 255, math.nan, _power(scale.clamp(1, 254).int() - 127))
    return v * factor.repeat_interleave(BLOCK, -1)[..., :D]


# ---------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------
def _frequencies(case):
    """Radians a token, [turned / 2] in 64 bits on the host."""
    turned, factor = case["turned"], case["factor"]
    f = 10000.0 ** (-torch.arange(0, turned, 2, dtype=torch.float64) / turned)
    if not case["parts"]:
        return f / factor
    # those of 32 turns and more over 2048 tokens stay, those below one are divided
    keep = ((2048 * f / (2 * math.pi) - 1) / (32 - 1)).clamp(0, 1)
    return f * (keep + (1 - keep) / factor)


def _slopes(H):
    """A geometric series over the heads, from 1/2 down to 1/256."""
    return torch.tensor([2.0 ** (-1 - 7.0 * h / max(1, H - 1)) for h in range(H)], device="cuda")


def _keys(g, shape, dtype):
    """Keys as projections leave them: some channels a few times as large as the others."""
    wide = 1 + 4 * (torch.rand(shape[-2:], generator=g, device="cuda") < 0.05)
    return (torch.randn(shape, generator=g, device="cuda") * wide).to(dtype)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[case["dtype"]]
    B, N, G, D = case["B"], case["N"], case["G"], case["D"]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dt)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32)

    x = {}
    if case["op"] == "rotary":
        H = case["H"]
        x["q"], x["k"] = normal(B, N, H, D), normal(B, N, G, D)
        x["frequencies"] = _frequencies(case)
        x["positions"] = x["lengths"] = None
        if case["kind"] == "train":
            x["dq"], x["dk"] = normal(B, N, H, D), normal(B, N, G, D)
            x["q"], x["k"] = x["q"].requires_grad_(True), x["k"].requires_grad_(True)
            if case["docs"] or case["far"]:
                t = torch.arange(N, device="cuda", dtype=torch.int32)
                cuts = torch.cat((whole(0, 0, B, 1), whole(0, N, B, max(0, case["docs"] - 1))), 1)
                start = torch.where(cuts[:, :, None] <= t, cuts[:, :, None], 0).amax(1)
                x["positions"] = (t - start).int() + case["far"]
        else:
            x["lengths"] = whole(0, 8192, B) + case["far"]
        return x
    S, bits = case["S"], case["bits"]
    x["cache"] = {}
    for n in ("k", "v"):
        held = _keys(g, (B, S, G, D), dt) if n == "k" else normal(B, S, G, D)
        x["cache"][n], x["cache"][n + "_scale"] = _quantise(held, bits)
        del held
    x["new"] = None
    if case["kind"] == "read":
        return x
    x["k"], x["v"] = _keys(g, (B, N, G, D), dt), normal(B, N, G, D)
    room = S - N
    x["lengths"] = whole(room - room // 4, room, B)
    if N > 16:
        x["new"] = whole(N - N // 3, N, B)       # right padding, a third of the batch's length at most
    if case["op"] == "attend":
        # scores of a standard deviation of about 2: heads that look at a few places
        x["q"] = normal(B, N, case["H"], D, std=2.0)
        x["slopes"] = _slopes(case["H"]) if case["slopes"] else None
        x["prefix"] = whole(0, S // 2, B) if case["prefix"] else None
    return x


def prepare(case, seed):
    return {"case": case, "x": _inputs(case, seed)}


# ---------------------------------------------------------------------------------------
# The package's calls
# ---------------------------------------------------------------------------------------
def _package():
    root = os.path.join(os.getcwd(), "causal-flare_amd")
    if root not in sys.path:
        sys.path.insert(1, root)
    import causal_flare
    return causal_flare


def _own(case, x):
    cf = _package()
    kind = case["kind"]
    if case["op"] == "rotary":
        y = cf.rotary_positions(x["q"], x["k"], x["frequencies"], positions=x["positions"], lengths=x["lengths"],
                                interleaved=case["interleaved"])
        if kind != "train":
            return list(y)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, (x["q"], x["k"]), (x["dq"], x["dk"])))
    dt = _TYPES[case["dtype"]]
    if kind == "read":
        return list(cf.quantized_cache_read(x["cache"], dtype=dt))
    y = []
    if case["op"] == "cache":
        cache = cf.quantized_cache_write(x["cache"], x["k"], x["v"], x["lengths"], new_lengths=x["new"])
    else:
        more = {"softcap": case["cap"] or None, "slopes": x["slopes"]}
        if kind == "prefill":
            out, cache = cf.softmax_attention_prefill(x["q"], x["k"], x["v"], x["cache"], x["lengths"], **more,
                                                      prefix_lengths=x["prefix"], new_lengths=x["new"])
        else:
            out, cache = cf.softmax_attention_decode(x["q"], x["k"], x["v"], x["cache"], x["lengths"], **more)
        y = [out]
    # what the call wrote, as the values that the cache now holds
    return y + list(cf.quantized_cache_read(cache, first=x["lengths"], count=case["N"], dtype=dt))


# ---------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------
def _turn(x, cos, sin, case):
    """The pairs of x [B, N, heads, D] turned by angles [B, N, 1, turned / 2]."""
    R = case["turned"]
    v = x.float()
    if case["interleaved"]:
        a, b = v[..., 0:R:2], v[..., 1:R:2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = v[..., :R // 2], v[..., R // 2:R]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((y, v[..., R:]), -1).to(x.dtype)


def _plain_rotary(case, x):
    t = torch.arange(case["N"], device="cuda", dtype=torch.float64)
    at = t.expand(case["B"], -1) if x["lengths"] is None else t + x["lengths"][:, None]
    if x["positions"] is not None:
        at = x["positions"].double()
    angle = (at[..., None] * x["frequencies"].to("cuda"))[:, :, None]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q, k = x["q"].detach(), x["k"].detach()
    y = [_turn(q, cos, sin, case), _turn(k, cos, sin, case)]
    if case["kind"] == "train":
        y += [_turn(x["dq"], cos, -sin, case), _turn(x["dk"], cos, -sin, case)]
    return y


def _plain_write(case, x):
    """The new rows to their places, in place; which rows of the cache these are, [B, N], and which are real."""
    B, N = case["B"], case["N"]
    t = torch.arange(N, device="cuda")
    at = x["lengths"].long()[:, None] + t
    real = torch.ones_like(at, dtype=torch.bool) if x["new"] is None else t < x["new"][:, None]
    b = torch.arange(B, device="cuda")[:, None].expand(B, N)
    cache = x["cache"]
    for n in ("k", "v"):
        for name, new in zip((n, n + "_scale"), _quantise(x[n], case["bits"])):
            held, new = cache[name].view(torch.uint8), new.view(torch.uint8)
            held[b, at] = torch.where(real[..., None, None], new, held[b, at])
    return b, at


def _plain_cache(case, x):
    dt = _TYPES[case["dtype"]]
    cache, D = x["cache"], case["D"]
    if case["kind"] == "read":
        return [_values(cache[n], cache[n + "_scale"], D).to(dt) for n in ("k", "v")]
    b, at = _plain_write(case, x)
    return [_values(cache[n][b, at], cache[n + "_scale"][b, at], D).to(dt) for n in ("k", "v")]


def _plain_attend(case, x):
    B, N, H, G, D, S = (case[n] for n in ("B", "N", "H", "G", "D", "S"))
    dt = _TYPES[case["dtype"]]
    b, at = _plain_write(case, x)
    cache = x["cache"]
    k, v = (_values(cache[n], cache[n + "_scale"], D).transpose(1, 2).contiguous() for n in ("k", "v"))   # [B, G, S, D]
    q = x["q"].float().view(B, N, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, H // G * N, D)
    s = (q @ k.transpose(2, 3).contiguous() / math.sqrt(D)).view(B, H, N, S)
    if case["cap"]:
        s = torch.tanh(s / case["cap"]) * case["cap"]
    j = torch.arange(S, device="cuda")
    if x["slopes"] is not None:
        s = s - x["slopes"][:, None, None] * (at[:, :, None] - j).abs()[:, None].float()
    n = torch.full((B,), N, device="cuda") if x["new"] is None else x["new"]
    sees = j <= at[:, :, None]
    if x["prefix"] is not None:
        sees = sees | (j < x["prefix"][:, None, None])
    sees = sees & (j < (x["lengths"] + n)[:, None, None])
    real = (torch.arange(N, device="cuda") < n[:, None])[:, None, :, None]          # [B, 1, N, 1]
    s = s.masked_fill_(~(sees[:, None] & real), -math.inf)
    top = s.amax(-1, keepdim=True)
    s = torch.exp(s.sub_(torch.where(real, top, 0.0)))
    total = s.sum(-1, keepdim=True)
    o = (s.view(B, G, H // G * N, S) @ v).view(B, H, N, D)
    y = torch.where(real, o / total, 0.0).transpose(1, 2)
    return [y.to(dt)] + [_values(cache[n][b, at], cache[n + "_scale"][b, at], D).to(dt) for n in ("k", "v")]


def run(state):
    case, x = state["case"], state["x"]
    if own:
        return _own(case, x)
    with torch.no_grad():
        return {"rotary": _plain_rotary, "cache": _plain_cache, "attend": _plain_attend}[case["op"]](case, x)


# ---------------------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    B, N, G, D = (case[n] for n in ("B", "N", "G", "D"))
    if case["op"] == "rotary":
        values = B * N * (case["H"] + G) * D * (2 if case["kind"] == "train" else 1)
        return {"bytes": 2 * size * values, "flops": 3 * values}
    held = D * case["bits"] // 8 + -(-D // BLOCK)             # bytes of a row of the cache
    if case["kind"] == "read":
        return {"bytes": 2 * B * N * G * (held + size * D), "flops": 2 * B * N * G * D}
    real = N * 5 // 6 if N > 16 else N
    new = 2 * B * G * real * (size * D + held) + 2 * B * G * N * size * D     # written, and read back
    if case["op"] == "cache":
        return {"bytes": new, "flops": 8 * B * real * G * D}
    H, seen = case["H"], (case["S"] - N) * 7 // 8
    pairs = real * seen + real * (real + 1) // 2
    return {"bytes": new + 2 * size * B * N * H * D + 2 * B * G * seen * held, "flops": 4 * B * H * D * pairs}


# ---------------------------------------------------------------------------------------
# The same outputs in 64 bits, from the definitions
# ---------------------------------------------------------------------------------------
def _exact_rotary(case, x):
    R = case["turned"]
    rows = []
    for b in range(case["B"]):
        if x["positions"] is not None:
            at = x["positions"][b].double()
        else:
            at = torch.arange(case["N"], device="cuda").double() + (0 if x["lengths"] is None else int(x["lengths"][b]))
        rows.append(torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                                at[:, None] * x["frequencies"].cuda()[None, :]))
    turn = torch.stack(rows)[:, :, None]

    def apply(v, turn):
        v = v.detach().double()
        out = v.clone()
        first = slice(0, R, 2) if case["interleaved"] else slice(0, R // 2)
        second = slice(1, R, 2) if case["interleaved"] else slice(R // 2, R)
        z = torch.complex(v[..., first], v[..., second]) * turn
        out[..., first], out[..., second] = z.real, z.imag
        return out

    y = [apply(x["q"], turn), apply(x["k"], turn)]
    if case["kind"] == "train":
        y += [apply(x["dq"], turn.conj()), apply(x["dk"], turn.conj())]
    return y


def _power64(e):
    """2^e in 64 bits, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _held(codes, scale):
    """A cache's values, each code taken apart into sign, exponent and mantissa."""
    if codes.dtype is torch.uint8:
        c = torch.empty((*codes.shape[:-1], 2 * codes.shape[-1]), dtype=torch.int64, device=codes.device)
        c[..., 0::2], c[..., 1::2] = codes & 15, codes >> 4
        sign, power, frac, bias, bits = c >> 3, (c >> 1) & 3, c & 1, 1, 1
    else:
        c = codes.view(torch.uint8).long()
        sign, power, frac, bias, bits = c >> 7, (c >> 3) & 15, c & 7, 7, 3
    v = torch.where(power > 0, frac + 2 ** bits, frac).double() * _power64(power.clamp_min(1) - bias - bits)
    at = torch.arange(v.shape[-1], device=codes.device) // BLOCK
    return torch.where(sign > 0, -v, v) * _power64(scale.long() - 127)[..., at]


def _rounded(x, bits):
    """What a cache holds of x [.., D]: the nearest value of the codes at its block's scale."""
    narrow = x.dtype is torch.float16
    x = x.double()
    out = torch.empty_like(x)
    least, frac, most, room = (0, 1, 6.0, 7.0) if bits == 4 else (-6, 3, 448.0, 464.0)
    lo, hi = ((-23, 13) if narrow else (-125, 125)) if bits == 4 else ((-15, 7) if narrow else (-117, 119))
    for d in range(0, x.shape[-1], BLOCK):
        w = x[..., d:d + BLOCK]
        top = w.abs().amax(-1, keepdim=True)
        # a logarithm's guess, put right by comparisons that are exact
        e = torch.ceil(torch.log2(top.clamp_min(1e-300) / room))
        e = torch.where(top > room * _power64(e), e + 1, torch.where(top <= room * _power64(e - 1), e - 1, e)).clamp(lo, hi)
        u = w * _power64(-e)
        at = torch.floor(torch.log2(u.abs().clamp_min(1e-300)))
        at = torch.where(_power64(at + 1) <= u.abs(), at + 1, torch.where(_power64(at) > u.abs(), at - 1, at))
        step = _power64(at.clamp_min(least) - frac)
        out[..., d:d + BLOCK] = (torch.round(u / step) * step).clamp(-most, most) * _power64(e)
    return out


def _exact_cache(case, x):
    cache = x["cache"]
    if case["kind"] == "read":
        return [_held(cache[n], cache[n + "_scale"]) for n in ("k", "v")]
    out = []
    for n in ("k", "v"):
        y = _rounded(x[n], case["bits"])
        for b in range(case["B"]):
            if x["new"] is not None:         # rows behind the real ones are the cache's own still
                real, at = int(x["new"][b]), int(x["lengths"][b])
                y[b, real:] = _held(cache[n][b, at + real:at + case["N"]], cache[n + "_scale"][b, at + real:at + case["N"]])
        out.append(y)
    return out


_ROWS = 2048      # queries of one piece


def _exact_attend(case, x):
    B, N, H, G, D = (case[n] for n in "BNHGD")
    q, cap = x["q"].double(), case["cap"]
    y = torch.zeros_like(q)
    for b in range(B):
        n, off = (N if x["new"] is None else int(x["new"][b])), int(x["lengths"][b])
        pre = 0 if x["prefix"] is None else int(x["prefix"][b])
        seen = {}
        for name in ("k", "v"):
            old = _held(x["cache"][name][b, :off], x["cache"][name + "_scale"][b, :off])
            seen[name] = torch.cat((old, _rounded(x[name][b, :n], case["bits"])))
        j = torch.arange(off + n, device="cuda")
        for i0 in range(0, n, _ROWS):
            i = torch.arange(i0, min(n, i0 + _ROWS), device="cuda")
            hide = (j[None, :] > i[:, None] + off) & (j[None, :] >= pre)
            for h in range(H):
                kk, vv = (seen[name][:, h * G // H].contiguous() for name in ("k", "v"))
                s = q[b, i, h] @ kk.t().contiguous() / math.sqrt(D)
                if cap:
                    s = cap * torch.tanh(s / cap)
                if x["slopes"] is not None:
                    s = s - x["slopes"][h].double() * (i[:, None] + off - j[None, :]).abs()
                y[b, i, h] = torch.softmax(s.masked_fill(hide, -math.inf), dim=1) @ vv
    return [y] + _exact_cache(dict(case, kind="write"), x)


def exact(case, seed):
    x = _inputs(case, seed)
    with torch.no_grad():
        return {"rotary": _exact_rotary, "cache": _exact_cache, "attend": _exact_attend}[case["op"]](case, x)
