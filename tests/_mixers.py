"""Plain 64-bit forms of the token mixers, with the size of the terms each result is summed from.

Every function returns values and magnitudes: what the same formula gives when each term enters
with its absolute value.  A tolerance is then `u |value| + k 2^-24 magnitude` (plus what a
rounding inside costs, where there is one): u is half a step of the output's type, and k counts
the fp32 roundings on the longest way from an input to the result.
"""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# Halves of the smallest fp16 step: results below its normal range are rounded absolutely.
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}


def check(got, ref, tol, what, dtype=torch.float32):
    limit = torch.finfo(got.dtype).max
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    tol = tol + TINY[dtype]
    bad = ~((got - ref).abs() <= tol)
    # a value past the largest of its type is an infinite one there
    bad &= ~((ref.abs() > limit) & (got == torch.sign(ref) * math.inf))
    bad &= ~((got == ref) | (torch.isnan(got) & torch.isnan(ref)))
    if bad.any():
        i = int(torch.where(bad, ((got - ref).abs() / tol).nan_to_num(1e30, 1e30, 1e30), 0.0).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, worst at {i}: "
                             f"{got.flatten()[i]:.9g} for {ref.flatten()[i]:.9g}, tolerance {tol.flatten()[i]:.3g}")


def wide(*tensors):
    return [None if t is None else t.detach().double().cpu() for t in tensors]


def silu_parts(z):
    s = torch.sigmoid(z)
    return z * s, s * (1 + z * (1 - s))


def back_steps(ids, B, N, most):
    """How many earlier tokens of its own run each token has, at most `most`: [B, N]."""
    out = torch.full((B, N), most)
    if ids is not None:
        for b in range(B):
            n = 0
            for t in range(N):
                n = n + 1 if t and ids[b, t] == ids[b, t - 1] else 0
                out[b, t] = min(n, most)
    return out


# ---------------------------------------------------------------------------------------
def conv(x, weight, bias, silu, ids=None, lengths=None, window=None, dy=None):
    """{name: (value, magnitude)} of y, window and, with dy, dx, dweight and dbias."""
    x, weight, bias, window, dy = wide(x, weight, bias, window, dy)
    ids = None if ids is None else ids.cpu()
    B, N, C = x.shape
    W = weight.shape[1]
    live = torch.ones((B, N), dtype=torch.bool)
    if lengths is not None:
        live = torch.arange(N)[None] < lengths.cpu()[:, None]
    if ids is not None:
        live = ids >= 0
    x = torch.where(live[..., None], x, 0.0)
    head = torch.zeros((B, W - 1, C), dtype=torch.float64) if window is None else window
    line = torch.cat((head, x), 1)
    reach = back_steps(ids, B, N, W - 1)
    pre = torch.zeros_like(x) if bias is None else bias.expand(B, N, C).clone()
    mag = pre.abs()
    for k in range(W):
        tap = torch.where((reach >= k)[..., None], line[:, W - 1 - k:W - 1 - k + N], 0.0)
        pre = pre + tap * weight[:, W - 1 - k]
        mag = mag + (tap * weight[:, W - 1 - k]).abs()
    val, slope = silu_parts(pre)
    y = val if silu else pre
    out = {"y": (torch.where(live[..., None], y, 0.0), mag)}
    n = torch.full((B,), N) if lengths is None else lengths.cpu().clamp(0, N)
    rows = torch.stack([line[b, int(n[b]):int(n[b]) + W - 1] for b in range(B)])
    out["window"] = (rows, rows.abs())
    if dy is None:
        return out
    d = torch.where(live[..., None], dy, 0.0)
    # silu'' is at most 1/2: an error of the pre-activation enters through it
    dmag = d.abs() * (1 + mag) if silu else d.abs()
    d = d * slope if silu else d
    dline, dlmag = torch.zeros_like(line), torch.zeros_like(line)
    dw, dwm = torch.zeros_like(weight), torch.zeros_like(weight)
    for k in range(W):
        on = (reach >= k)[..., None]
        dline[:, W - 1 - k:W - 1 - k + N] += torch.where(on, d * weight[:, W - 1 - k], 0.0)
        dlmag[:, W - 1 - k:W - 1 - k + N] += torch.where(on, dmag * weight[:, W - 1 - k].abs(), 0.0)
        tap = torch.where(on, line[:, W - 1 - k:W - 1 - k + N], 0.0)
        dw[:, W - 1 - k] = (d * tap).sum((0, 1))
        dwm[:, W - 1 - k] = (dmag * tap.abs()).sum((0, 1))
    out["dx"] = dline[:, W - 1:], dlmag[:, W - 1:]
    out["dweight"] = dw, dwm
    out["dbias"] = d.sum((0, 1)), dmag.sum((0, 1))
    return out


# ---------------------------------------------------------------------------------------
def _past(mag):
    """Magnitudes along dimension 1, infinite from where one passes fp32: such a state stays so."""
    return torch.where(mag.cummax(1).values > 1e38, math.inf, mag)


def scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=False, ids=None, lengths=None, h0=None, dy=None):
    """{name: (value, magnitude)} of y, h and, with dy, every gradient; B, C [nb, n, g, s]."""
    x, dt, A, B, C, D, z, dt_bias, h0, dy = wide(x, dt, A, B, C, D, z, dt_bias, h0, dy)
    nb, n, c = x.shape
    s, g = A.shape[1], B.shape[2]
    live = torch.ones((nb, n), dtype=torch.bool)
    if lengths is not None:
        live = torch.arange(n)[None] < lengths.cpu()[:, None]
    if ids is not None:
        ids = ids.cpu()
        live = ids >= 0
    on = live[..., None]
    x, dt = torch.where(on, x, 0.0), torch.where(on, dt, 0.0)
    raw = dt if dt_bias is None else dt + dt_bias
    delta = torch.nn.functional.softplus(raw, threshold=700) if softplus else raw
    delta = torch.where(on, delta, 0.0)
    Bw, Cw = (torch.where(on[..., None], t, 0.0).repeat_interleave(c // g, 2) for t in (B, C))
    cut = torch.zeros((nb, n), dtype=torch.bool)
    if ids is not None:
        cut[:, 1:] = ids[:, 1:] != ids[:, :-1]
    a = torch.exp(delta[..., None] * A)
    a = torch.where(cut[..., None, None], 0.0, a)
    u = (delta * x)[..., None] * Bw
    h = torch.zeros((nb, c, s), dtype=torch.float64) if h0 is None else h0
    hm = h.abs()
    hs, hms = [], []
    for t in range(n):
        h, hm = a[:, t] * h + u[:, t], a[:, t] * hm + u[:, t].abs()
        hs.append(h)
        hms.append(hm)
    H, HM = torch.stack(hs, 1), _past(torch.stack(hms, 1))
    skip = torch.zeros_like(x) if D is None else D * x
    lin, linm = (Cw * H).sum(-1) + skip, (Cw.abs() * HM).sum(-1) + skip.abs()
    gate, slope = (torch.ones_like(x), None) if z is None else silu_parts(torch.where(on, z, 0.0))
    out = {"y": (torch.where(on, lin * gate, 0.0), linm * gate.abs()), "h": (h, hm)}
    # the roundings a term can pass through: every step of the recurrence, each with an exponent
    # of size |delta A|
    out["k"] = 8 * (n + s + 16) * (1 + float((delta[..., None] * A).abs().max()))
    if dy is None:
        return out
    dy = torch.where(on, dy, 0.0)
    gy = dy * gate
    prev = torch.cat((torch.zeros_like(H[:, :1]), H[:, :-1]), 1)
    prevm = torch.cat((torch.zeros_like(H[:, :1]), HM[:, :-1]), 1)
    r, rm = torch.zeros_like(h), torch.zeros_like(h)
    rs, rms = [], []
    for t in range(n - 1, -1, -1):
        r, rm = r + gy[:, t, :, None] * Cw[:, t], rm + (gy[:, t, :, None] * Cw[:, t]).abs()
        rs.append(r)
        rms.append(rm)
        r, rm = r * a[:, t], rm * a[:, t]
    Rg, RM = torch.stack(rs[::-1], 1), _past(torch.stack(rms, 1)).flip(1)
    p, pm = Rg * a * prev, RM * a * prevm
    sB, sBm = (Rg * Bw).sum(-1), (RM * Bw.abs()).sum(-1)
    step = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    ddt, ddtm = ((p * A).sum(-1) + x * sB) * step, ((pm * A.abs()).sum(-1) + x.abs() * sBm) * step
    ddt, ddtm = torch.where(on, ddt, 0.0), torch.where(on, ddtm, 0.0)
    out["dx"] = (torch.where(on, delta * sB + (0 if D is None else gy * D), 0.0),
                 delta.abs() * sBm + (0 if D is None else (gy * D).abs()))
    out["ddt"] = ddt, ddtm
    out["dA"] = (p * delta[..., None]).sum((0, 1)), (pm * delta[..., None].abs()).sum((0, 1))
    du = (delta * x)[..., None]
    out["dB"] = (Rg * du).view(nb, n, g, c // g, s).sum(3), (RM * du.abs()).view(nb, n, g, c // g, s).sum(3)
    gh = gy[..., None]
    out["dC"] = (gh * H).view(nb, n, g, c // g, s).sum(3), (gh.abs() * HM).view(nb, n, g, c // g, s).sum(3)
    out["dD"] = (gy * x).sum((0, 1)), (gy * x).abs().sum((0, 1))
    out["ddt_bias"] = ddt.sum((0, 1)), ddtm.sum((0, 1))
    if z is not None:
        out["dz"] = torch.where(on, dy * lin * slope, 0.0), (dy * slope).abs() * linm + dy.abs() * linm
    return out


# ---------------------------------------------------------------------------------------
def attention(q, k, v, scale=None, causal=True, softcap=None, slopes=None, ids=None, prefix=None, offset=None,
              dy=None, unit=0.0, tiny=0.0):
    """{name: (value, tolerance)} of y and, with dy, dq, dk and dv.

    unit: half a step of the type that weights and score gradients are rounded to (0: none), tiny:
    half its smallest step, 2^-25 for fp16, by which a weight or score gradient below 2^-14 is
    off; 2^-126 for the others, below which an exponential is 0.  (Weights are at most that much off after the division by their sum, which is at least 1.)
    offset [B]: position of query 0 (k and v then hold positions 0 ..).  The tolerances hold the
    inner roundings; the caller adds that of the result.
    """
    q, k, v, slopes, dy = wide(q, k, v, slopes, dy)
    B, N, H, D = q.shape
    M, G = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    y, ty = torch.zeros_like(q), torch.zeros_like(q)
    dq, tq = torch.zeros_like(q), torch.zeros_like(q)
    dk, tk, dv, tv = (torch.zeros_like(k) for _ in range(4))
    e32 = 2.0 ** -24
    for b in range(B):
        off = 0 if offset is None else int(offset[b])
        i, j = torch.arange(N)[:, None] + off, torch.arange(M)[None]
        see = torch.ones((N, M), dtype=torch.bool)
        if causal:
            see = j <= i
            if prefix is not None:
                see = see | (j < int(prefix[b]))
        if ids is not None:
            d = ids[b].cpu()
            see = see & (d[:, None] == d[None]) & (d[:, None] >= 0)
        rows, cols = see.any(1)[:, None], see.any(0)[:, None]
        for h in range(H):
            m = h // (H // G)
            # what no one sees has no part in anything, whatever it holds
            qq, kk, vv = torch.where(rows, q[b, :, h], 0.0), torch.where(cols, k[b, :, m], 0.0), v[b, :, m]
            vv = torch.where(cols, vv, 0.0)
            x = qq @ kk.t() * scale
            size = qq.abs() @ kk.abs().t() * abs(scale)
            th = torch.tanh(x / softcap) if softcap else None
            s = softcap * th if softcap else x
            if slopes is not None:
                s = s - slopes[h] * (i - j).abs()
                size = size + slopes[h].abs() * (i - j).abs()
            s = torch.where(see, s, -math.inf)
            top = s.amax(1, keepdim=True)
            p = torch.exp(s - torch.where(top.isinf(), 0.0, top))
            p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
            # absolute error of a score: a product over D, the cap (two units of 1 of tanh), the bias
            es = e32 * (torch.where(see, size, 0.0).amax(1, keepdim=True) * (8 + D / 4) + 16 + 8 * (softcap or 0.0))
            o = p @ vv
            y[b, :, h] = o
            pv = p @ vv.abs()
            ty[b, :, h] = (unit + 2 * es + e32 * 64) * pv + tiny * (see.double() @ vv.abs())
            if dy is None:
                continue
            do = torch.where(rows, dy[b, :, h], 0.0)
            dp = do @ vv.t()
            delta = (do * o).sum(1, keepdim=True)
            cut = (1 - th * th) if softcap else torch.ones_like(p)
            ds = p * (dp - delta) * cut
            # errors of dP and delta (the latter from the rounded y), of p, and of the cut
            edp = e32 * (16 + D) * (do.abs() @ vv.abs().t()) + (do.abs() * ((unit * 2 + 2 * es + e32 * 64) * pv
                                                                          + unit * o.abs())).sum(1, keepdim=True)
            eds = p * cut * edp + (2 * es + e32 * 64) * p * (dp - delta).abs() * (cut + (4 if softcap else 0))
            eds = eds + unit * ds.abs() + tiny * see * (1 + (dp - delta).abs())
            dq[b, :, h] = ds @ kk * scale
            tq[b, :, h] = (eds @ kk.abs() + e32 * 64 * (ds.abs() @ kk.abs())) * abs(scale)
            dk[b, :, m] += ds.t() @ qq * scale
            tk[b, :, m] += (eds.t() @ qq.abs() + e32 * 64 * (ds.abs().t() @ qq.abs())) * abs(scale)
            dv[b, :, m] += p.t() @ do
            tv[b, :, m] += ((unit + 2 * es + e32 * 64) * p + tiny * see).t() @ do.abs()
    out = {"y": (y, ty)}
    if dy is not None:
        out.update(dq=(dq, tq), dk=(dk, tk), dv=(dv, tv))
    return out
