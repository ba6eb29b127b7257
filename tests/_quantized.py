"""Plain 64-bit forms of quantised caches and rotary positions."""
import math

import torch

BLOCK = 32
# of each code: exponent of the least normal value, bits of the mantissa, the largest value, what a block's
# largest value may be at a scale of 1, and the exponents of scales by the writer's type
FORMS = {4: (0, 1, 6.0, 7.0, (-23, 13), (-125, 125)), 8: (-6, 3, 448.0, 464.0, (-15, 7), (-117, 119))}


def scale_exponents(x, bits):
    """The exponent of each block of x [.., D], and whether it holds a value that is not finite."""
    lo, hi = FORMS[bits][4 if x.dtype is torch.float16 else 5]
    room = FORMS[bits][3]
    w = x.double()
    blocks = [w[..., d:d + BLOCK] for d in range(0, w.shape[-1], BLOCK)]
    top = torch.stack([b.abs().amax(-1) for b in blocks], -1)
    odd = ~torch.stack([torch.isfinite(b).all(-1) for b in blocks], -1)
    top = torch.where(odd, 0.0, top)
    e = torch.full_like(top, float(lo))
    for step in range(lo, hi):                       # the least e with top <= room 2^e
        e = torch.where(top > room * 2.0 ** step, float(step + 1), e)
    return e, odd


def rounded(x, bits):
    """(values, scale bytes) that a cache holds of x [.., D]; values in 64 bits."""
    least, frac, most = FORMS[bits][:3]
    e, odd = scale_exponents(x, bits)
    at = torch.arange(x.shape[-1]) // BLOCK
    scale = (2.0 ** e)[..., at]
    u = torch.where(odd[..., at], 0.0, x.double()) / scale
    power = torch.floor(torch.log2(u.abs().clamp_min(2.0 ** -60)))
    power = torch.where(2.0 ** (power + 1) <= u.abs(), power + 1, torch.where(2.0 ** power > u.abs(), power - 1, power))
    step = 2.0 ** (power.clamp_min(least) - frac)
    v = (torch.round(u / step) * step).clamp(-most, most) * scale
    return torch.where(odd[..., at], math.nan, v), torch.where(odd, 255, e + 127).to(torch.uint8)


def held(codes, scale):
    """What codes and scale bytes stand for, in 64 bits, code by code."""
    codes, scale = codes.cpu(), scale.cpu()
    if codes.dtype is torch.uint8:
        c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
        sign, power, frac, bias, bits = c >> 3, (c >> 1) & 3, c & 1, 1, 1
    else:
        c = codes.view(torch.uint8).long()
        sign, power, frac, bias, bits = c >> 7, (c >> 3) & 15, c & 7, 7, 3
    v = torch.where(power > 0, frac + 2 ** bits, frac).double() * 2.0 ** (power.clamp_min(1) - bias - bits).double()
    at = torch.arange(v.shape[-1]) // BLOCK
    s = torch.where(scale == 255, math.nan, 2.0 ** (scale.double() - 127))
    return torch.where(sign > 0, -v, v) * s[..., at]


def rotary(x, frequencies, at, interleaved=False, inverse=False):
    """(values, magnitudes) of x [B, N, heads, D] turned by positions at [B, N], in 64 bits."""
    x = x.detach().double().cpu()
    R = 2 * frequencies.shape[0]
    angle = at.double().cpu()[..., None, None] * frequencies.double()
    c, s = torch.cos(angle), torch.sin(angle) * (-1 if inverse else 1)
    first, second = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    a, b = x[..., first], x[..., second]
    y, mag = x.clone(), x.abs()
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    mag[..., first], mag[..., second] = a.abs() + b.abs(), a.abs() + b.abs()
    mag[..., R:] = 0.0                                # these stay as they are
    return y, mag
