"""The token mixers a hybrid stack sets beside its FLARE layers: what is measured of them.

A short causal convolution, a selective state space scan and exact softmax attention (its
scores capped by a tanh, biased by distance, masked by documents or by a prefix).  Each is
called as a program calls it: over packed documents in a training step, over prompts that
continue a cached state, and for one token a sequence while answering.

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


# ---------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------
def _conv(name, kind, dtype, B, N, C, W, silu=True, docs=0):
    case = {"op": "conv", "kind": kind, "dtype": dtype, "B": B, "N": N, "C": C, "W": W, "silu": silu, "docs": docs}
    return dict(case, name=name) if name else case


def _scan(name, kind, dtype, B, N, C, S, G=1, gate=True, docs=0):
    case = {"op": "scan", "kind": kind, "dtype": dtype, "B": B, "N": N, "C": C, "S": S, "G": G, "gate": gate,
            "docs": docs}
    return dict(case, name=name) if name else case


def _attend(name, kind, dtype, B, N, H, G, D, cap=0.0, slopes=False, docs=0, prefix=False, cache=0):
    case = {"op": "attend", "kind": kind, "dtype": dtype, "B": B, "N": N, "H": H, "G": G, "D": D, "cap": cap,
            "slopes": slopes, "docs": docs, "prefix": prefix, "cache": cache}
    return dict(case, name=name) if name else case


def listed():
    return [
        # prompts of a padded batch that continue earlier ones, 16 heads of 128
        _conv("conv_prompt", "prefill", "bf16", 4, 4096, 2048, 4),
        # a training step over packed documents of an odd total length, 16 heads of 64
        _conv("conv_train", "train", "bf16", 4, 2011, 1024, 4, docs=7),
        # one token for each sequence of a serving batch: a launch and its latency
        _conv("conv_step", "decode", "bf16", 64, 1, 2048, 4),
        # one token for each sequence of a serving batch: the states stream through
        _scan("scan_step", "decode", "bf16", 64, 1, 2048, 16),
        # a short odd prompt in full precision, as a CPU-side check or a small model runs it
        _scan("scan_prompt_small", "prefill", "fp32", 1, 257, 512, 16, gate=False),
        # one long document as a prompt, when the tokens are the only parallel axis
        _scan("scan_prompt_long", "prefill", "bf16", 1, 16384, 2048, 16),
        # the training step of a mid-size layer
        _scan("scan_train", "train", "bf16", 4, 4096, 2048, 16, docs=5),
        # one token a sequence against a cache of some thousands, shared key heads, capped scores
        _attend("attend_step", "decode", "bf16", 64, 1, 16, 4, 128, cap=30.0, cache=8192),
        # full precision with a bias on distance at an odd length, forward and backward
        _attend("attend_train_fp32", "train", "fp32", 2, 1021, 8, 8, 64, slopes=True),
        # the training step of a mid-size layer with capped scores
        _attend("attend_train", "train", "bf16", 4, 4096, 16, 16, 64, cap=30.0),
        # a long packed batch of documents, shared key heads and a bias on distance
        _attend("attend_train_packed", "train", "bf16", 1, 16384, 16, 4, 128, slopes=True, docs=6),
        # follow-up prompts of odd lengths into caches, with a prefix that sees itself whole
        _attend("attend_prompt", "prefill", "fp16", 3, 1531, 16, 4, 128, prefix=True, cache=4096),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("conv", "scan", "scan", "attend", "attend", "attend"))
    kind = rng.choice(("prefill", "train", "decode"))
    dtype = rng.choice(("bf16", "bf16", "bf16", "fp16", "fp32"))
    if kind == "decode":
        B, N = _log_int(rng, 1, 64), 1
    else:
        B = _log_int(rng, 1, 8)
    docs = rng.choice((0, 0, 1, 3, 8)) if kind == "train" else 0
    if op in ("conv", "scan"):
        C = rng.choice((64, 200, 512, 768, 1000, 1024, 1536, 2048))
        if kind != "decode":
            # no drawn call costs more than the largest listed one
            N = _log_int(rng, 40, max(80, min(16384, 2 ** 24 // (B * C))))
        if op == "conv":
            return _conv(None, kind, dtype, B, N, C, rng.choice((2, 3, 4, 4)), rng.random() < 0.7, docs)
        G = rng.choice((1, 1, 1, 2, 4))
        return _scan(None, kind, dtype, B, N, C, rng.choice((8, 16, 16, 16, 24, 32)) if C <= 1024 else 16, G,
                     rng.random() < 0.7, docs)
    G = rng.choice((1, 2, 4, 8))
    H = G * rng.choice((1, 1, 2, 4, 8) if G <= 2 else (1, 2, 4))
    D = rng.choice((32, 48, 64, 64, 80, 96, 128, 128))
    cap = rng.choice((0.0, 0.0, 20.0, 50.0))
    slopes = rng.random() < 0.4
    if kind == "decode":
        return _attend(None, kind, dtype, B, 1, H, G, D, cap, slopes, cache=_log_int(rng, 64, 8192 * 16 * 64 // (B * H)
                                                                                  if B * H > 1024 else 8192))
    most = 2 ** 16 if dtype != "fp32" else 2 ** 13
    N = _log_int(rng, 40, max(80, min(8192, most * 2 // (B * H))))
    cache = N + _log_int(rng, 1, 2048) if kind == "prefill" else 0
    return _attend(None, kind, dtype, B, N, H, G, D, cap, slopes, docs, rng.random() < 0.3, cache)


# ---------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------
def _documents(case, g):
    """Ids of packed documents: random cuts, and the row's last few tokens padding (-1)."""
    B, N = case["B"], case["N"]
    if not case["docs"]:
        return None
    cuts = torch.rand((B, case["docs"] - 1), generator=g, device="cuda").mul(N).long()
    starts = torch.zeros((B, N + 1), dtype=torch.int64, device="cuda")
    starts.scatter_add_(1, cuts, torch.ones_like(cuts))
    ids = starts.cumsum(1)[:, :N].to(torch.int32)
    pad = torch.randint(0, 1 + N // 50, (B,), generator=g, device="cuda")
    ids[torch.arange(N, device="cuda")[None, :] >= (N - pad)[:, None]] = -1
    return ids


def _slopes(H):
    """A geometric series over the heads, from 1/2 down to 1/256."""
    return torch.tensor([2.0 ** (-1 - 7.0 * h / max(1, H - 1)) for h in range(H)], device="cuda")


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[case["dtype"]]
    B, N, kind = case["B"], case["N"], case["kind"]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    def lengths():
        # right padding, a third of the batch's length at most
        return torch.randint(N - N // 3, N + 1, (B,), generator=g, device="cuda", dtype=torch.int32)

    f32 = torch.float32
    x = {}
    if case["op"] == "conv":
        C, W = case["C"], case["W"]
        x["x"] = normal(B, N, C)
        x["weight"] = normal(C, W, std=W ** -0.5, dtype=f32)
        x["bias"] = normal(C, std=0.1, dtype=f32)
        if kind != "train":
            x["state"] = normal(B, W - 1, C)
        leaves = ("x", "weight", "bias")
        shape = (B, N, C)
    elif case["op"] == "scan":
        C, S, G = case["C"], case["S"], case["G"]
        x["x"] = normal(B, N, C)
        x["dt"] = normal(B, N, C, std=0.5)
        x["A"] = -torch.arange(1, S + 1, device="cuda", dtype=f32).expand(C, S).mul(1 + normal(C, 1, std=0.05, dtype=f32))
        x["B"] = normal(B, N, G, S)
        x["C"] = normal(B, N, G, S)
        x["D"] = 1 + normal(C, std=0.1, dtype=f32)
        # steps of 1e-3 to 1e-1 where dt is 0: the softplus' inverse of them
        step = torch.exp(torch.rand((C,), generator=g, device="cuda") * math.log(100.0) + math.log(1e-3))
        x["dt_bias"] = step + torch.log(-torch.expm1(-step))
        x["z"] = normal(B, N, C) if case["gate"] else None
        if kind != "train":
            x["state"] = normal(B, C, S, std=0.3, dtype=f32)
        leaves = ("x", "dt", "A", "B", "C", "D", "dt_bias") + (("z",) if case["gate"] else ())
        shape = (B, N, C)
    else:
        H, G, D = case["H"], case["G"], case["D"]
        # scores of a standard deviation of 2: heads that look at a few places
        x["q"], x["k"], x["v"] = normal(B, N, H, D, std=2.0), normal(B, N, G, D), normal(B, N, G, D)
        x["slopes"] = _slopes(H) if case["slopes"] else None
        S = case["cache"]
        if kind != "train":
            x["cache_k"], x["cache_v"] = normal(B, S, G, D), normal(B, S, G, D)
            room = S - N
            x["lengths"] = torch.randint(room - room // 4, room + 1, (B,), generator=g, device="cuda",
                                         dtype=torch.int32)
        x["prefix"] = None
        if case["prefix"]:
            top = N if kind == "train" else S
            x["prefix"] = torch.randint(0, top // 2 + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        leaves = ("q", "k", "v")
        shape = (B, N, H, D)
    x["docs"] = _documents(case, g)
    x["new"] = lengths() if kind == "prefill" else None
    if kind == "train":
        x["dy"] = normal(*shape)
        for name in leaves:
            x[name] = x[name].detach().requires_grad_(True)
        x["leaves"] = leaves
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
    if case["op"] == "conv":
        act = "silu" if case["silu"] else None
        if kind == "train":
            y = cf.short_convolution(x["x"], x["weight"], x["bias"], activation=act, document_ids=x["docs"])
        elif kind == "prefill":
            y, state = cf.short_convolution_prefill(x["x"], x["weight"], x["bias"], activation=act,
                                                    state={"window": x["state"]}, lengths=x["new"])
            return [y, state["window"]]
        else:
            y, state = cf.short_convolution_decode(x["x"], x["weight"], x["bias"], activation=act,
                                                   state={"window": x["state"]})
            return [y, state["window"]]
    elif case["op"] == "scan":
        args = (x["x"], x["dt"], x["A"], x["B"], x["C"])
        more = {"D": x["D"], "z": x["z"], "dt_bias": x["dt_bias"], "dt_softplus": True}
        if kind == "train":
            y = cf.state_space_scan(*args, **more, document_ids=x["docs"])
        elif kind == "prefill":
            y, state = cf.state_space_scan_prefill(*args, **more, state={"h": x["state"]}, lengths=x["new"])
            return [y, state["h"]]
        else:
            y, state = cf.state_space_scan_decode(*args, **more, state={"h": x["state"]})
            return [y, state["h"]]
    else:
        more = {"softcap": case["cap"] or None, "slopes": x["slopes"]}
        if kind == "train":
            y = cf.softmax_attention(x["q"], x["k"], x["v"], **more, document_ids=x["docs"],
                                     prefix_lengths=x["prefix"])
        else:
            cache = {"k": x["cache_k"], "v": x["cache_v"]}
            if kind == "prefill":
                y, cache = cf.softmax_attention_prefill(x["q"], x["k"], x["v"], cache, x["lengths"], **more,
                                                        prefix_lengths=x["prefix"], new_lengths=x["new"])
            else:
                y, cache = cf.softmax_attention_decode(x["q"], x["k"], x["v"], cache, x["lengths"], **more)
            return [y, cache["k"], cache["v"]]
    return [y.detach(), *torch.autograd.grad(y, [x[n] for n in x["leaves"]], x["dy"])]


# ---------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------
def _runs(case, x):
    """Which tokens begin a document, and which are no padding: [B, N] each, or None."""
    ids = x["docs"]
    if ids is not None:
        first = torch.ones_like(ids, dtype=torch.bool)
        first[:, 1:] = ids[:, 1:] != ids[:, :-1]
        return first, ids >= 0
    if x["new"] is not None:
        t = torch.arange(case["N"], device="cuda")
        return None, t[None, :] < x["new"][:, None]
    return None, None


def _plain_conv(case, x):
    B, N, W, kind = case["B"], case["N"], case["W"], case["kind"]
    xf, w, bias = x["x"].float(), x["weight"].float(), x["bias"].float()
    first, keep = _runs(case, x)
    before = x["state"].float() if kind != "train" else xf.new_zeros((B, W - 1, case["C"]))
    xs = torch.cat((before, xf), dim=1)
    reach = None
    if first is not None:
        run = first.cumsum(1)
        reach = torch.cat((run.new_zeros((B, W - 1)), run), dim=1)
    pre = bias.expand(B, N, -1)
    taps = []
    for k in range(W):                       # the tap k tokens back
        tap = xs[:, W - 1 - k:W - 1 - k + N]
        if reach is not None:
            tap = tap * (reach[:, W - 1 - k:W - 1 - k + N] == run)[..., None]
        taps.append(tap)
        pre = pre + tap * w[:, W - 1 - k]
    gate = torch.sigmoid(pre)
    y = pre * gate if case["silu"] else pre
    if keep is not None:
        y = y * keep[..., None]
    out = [y.to(x["x"].dtype)]
    if kind != "train":
        n = torch.full((B,), N, device="cuda") if x["new"] is None else x["new"].long()
        at = n[:, None] + torch.arange(W - 1, device="cuda")[None, :]
        window = torch.gather(xs, 1, at[..., None].expand(-1, -1, case["C"])).to(x["x"].dtype)
        if kind == "decode":
            x["state"].copy_(window)
            window = x["state"]
        return out + [window]
    d = x["dy"].float()
    if case["silu"]:
        d = d * gate * (1 + pre * (1 - gate))
    if keep is not None:
        d = d * keep[..., None]
    dx = torch.zeros_like(xs)
    dw = []
    for k in range(W):
        dk = d * w[:, W - 1 - k]
        if reach is not None:
            dk = dk * (reach[:, W - 1 - k:W - 1 - k + N] == run)[..., None]
        dx[:, W - 1 - k:W - 1 - k + N] += dk
        dw.append((d * taps[k]).sum((0, 1)))
    return out + [dx[:, W - 1:].to(x["x"].dtype), torch.stack(dw[::-1], dim=1), d.sum((0, 1))]


def _carry(a, b):
    """h_t = a_t h_{t-1} + b_t over dimension 1 from h = 0, by doubling; `b` is replaced."""
    step, n = 1, a.shape[1]
    while step < n:
        b = torch.cat((b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]), dim=1)
        if 2 * step < n:
            a = torch.cat((a[:, :step], a[:, step:] * a[:, :-step]), dim=1)
        step *= 2
    return b


def _plain_scan(case, x):
    B, N, C, S, G, kind = (case[k] for k in ("B", "N", "C", "S", "G", "kind"))
    xf, A, D = x["x"].float(), x["A"].float(), x["D"].float()
    Bm, Cm = (x[k].float().repeat_interleave(C // G, dim=2) if G > 1 else x[k].float() for k in ("B", "C"))
    raw = x["dt"].float() + x["dt_bias"].float()
    delta = raw.clamp_min(0) + torch.log1p(torch.exp(-raw.abs()))
    first, keep = _runs(case, x)
    if keep is not None:
        keep = keep[..., None]
        delta = torch.where(keep, delta, 0.0)     # a token that is no token leaves the state alone
    a = torch.exp(delta[..., None] * A)
    if first is not None:
        a = torch.where(first[..., None, None], 0.0, a)
    u = (delta * xf)[..., None] * Bm
    if kind != "train":
        u[:, 0] += a[:, 0] * x["state"]
    h = _carry(a, u)
    lin = (Cm * h).sum(-1) + D * xf
    zf = x["z"].float() if case["gate"] else None
    gate = torch.sigmoid(zf) if case["gate"] else None
    y = lin * zf * gate if case["gate"] else lin
    if keep is not None:
        y = torch.where(keep, y, 0.0)
    out = [y.to(x["x"].dtype)]
    if kind != "train":
        h = h[:, -1].contiguous()
        if kind == "decode":
            x["state"].copy_(h)
            h = x["state"]
        return out + [h]
    dy = x["dy"].float()
    if keep is not None:
        dy = torch.where(keep, dy, 0.0)
    dz = None
    if case["gate"]:
        dz = dy * lin * gate * (1 + zf * (1 - gate))
        dy = dy * zf * gate
    # dh_t = C_t dy_t + a_{t+1} dh_{t+1}: the same carry over the reversed tokens
    nxt = torch.cat((a[:, 1:], torch.zeros_like(a[:, :1])), dim=1)
    dh = _carry(nxt.flip(1), (dy[..., None] * Cm).flip(1)).flip(1)
    del nxt
    prev = torch.cat((torch.zeros_like(h[:, :1]), h[:, :-1]), dim=1)
    da = dh * prev * a                           # d/d(delta A); a = 0 where a document begins
    del prev, a
    s = (dh * Bm).sum(-1)
    ddelta = (da * A).sum(-1) + s * xf
    draw_ = ddelta * torch.sigmoid(raw)
    if keep is not None:
        draw_ = torch.where(keep, draw_, 0.0)
    dA = (da * delta[..., None]).sum((0, 1))
    dB = (dh * (delta * xf)[..., None]).view(B, N, G, C // G, S).sum(3)
    dC = (dy[..., None] * h).view(B, N, G, C // G, S).sum(3)
    grads = [s * delta + dy * D, draw_, dA, dB, dC, (dy * xf).sum((0, 1)), draw_.sum((0, 1))]
    if case["gate"]:
        grads.append(dz)
    return out + [t.to(x[n].dtype) for t, n in zip(grads, x["leaves"])]


def _visible(case, x, b, rows, cols, at):
    """Which keys `cols` the queries at positions `rows` of sequence b may see."""
    see = cols[None, :] <= rows[:, None]
    if x["prefix"] is not None:
        see |= cols[None, :] < x["prefix"][b]
    if case["kind"] != "train":
        n = x["lengths"][b] + (x["new"][b] if x["new"] is not None else 1)
        see &= (cols < n)[None, :] & (rows < n)[:, None]
    elif x["docs"] is not None:
        ids = x["docs"][b]
        see &= (ids[at][:, None] == ids[None, :]) & (ids[at] >= 0)[:, None]
    return see


def _plain_attend(case, x):
    B, N, H, G, D, kind, cap = (case[k] for k in ("B", "N", "H", "G", "D", "kind", "cap"))
    scale = D ** -0.5
    dt = x["q"].dtype
    train = kind == "train"
    k_all, v_all = x["k"], x["v"]
    if not train:
        t = torch.arange(N, device="cuda")[None, :]
        ok = t < (x["new"] if x["new"] is not None else torch.full((B,), N, device="cuda"))[:, None]
        bi = torch.arange(B, device="cuda")[:, None].expand(B, N)
        to = (x["lengths"].long()[:, None] + t)
        k_all, v_all = x["cache_k"], x["cache_v"]
        for cache, new in ((k_all, x["k"]), (v_all, x["v"])):
            at = torch.where(ok, to, 0)
            old = cache[bi, at]
            # the rows behind a prompt's end keep what the cache held
            vals = torch.where(ok[..., None, None], new.detach(), old)
            first = cache[:, 0].clone()
            cache[bi, at] = vals
            cache[:, 0] = torch.where((x["lengths"] == 0)[:, None, None] & ok[:, :1, None], new.detach()[:, 0], first)
    M = k_all.shape[1]
    if kind == "decode":
        return [_plain_step(case, x).to(dt), k_all, v_all]
    y = torch.zeros((B, N, H, D), device="cuda", dtype=torch.float32)
    if train:
        dq, dk, dv = torch.zeros_like(y), torch.zeros((B, N, G, D), device="cuda"), torch.zeros((B, N, G, D), device="cuda")
    cols = torch.arange(M, device="cuda")
    at = torch.arange(N, device="cuda")
    for b in range(B):
        rows = at if train else at + x["lengths"][b]
        see = _visible(case, x, b, rows, cols, at)
        far = (rows[:, None] - cols[None, :]).abs().float() if case["slopes"] else None
        for h in range(H):
            j = h // (H // G)
            q, k, v = x["q"][b, :, h].float(), k_all[b, :, j].float(), v_all[b, :, j].float()
            s = (q @ k.t()) * scale
            if cap:
                tanh = torch.tanh(s / cap)
                s = cap * tanh
            if far is not None:
                s = s - x["slopes"][h] * far
            s = torch.where(see, s, -math.inf)
            top = s.amax(1, keepdim=True)
            p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            total = p.sum(1, keepdim=True)
            p = p / torch.where(total == 0, 1.0, total)
            y[b, :, h] = p @ v
            if train:
                dy = x["dy"][b, :, h].float()
                ds = p * (dy @ v.t() - (dy * y[b, :, h]).sum(1, keepdim=True))
                if cap:
                    ds = ds * (1 - tanh * tanh)
                dq[b, :, h] = (ds @ k) * scale
                dk[b, :, j] += (ds.t() @ q) * scale
                dv[b, :, j] += p.t() @ dy
    if train:
        return [t.to(dt) for t in (y, dq, dk, dv)]
    return [y.to(dt), x["cache_k"], x["cache_v"]]


def _plain_step(case, x):
    """One query a sequence against its cache: the heads that share keys as one product."""
    B, H, G, D, cap = (case[k] for k in ("B", "H", "G", "D", "cap"))
    M = case["cache"]
    q = x["q"].float().view(B, G, H // G, D)
    k = x["cache_k"].float().permute(0, 2, 3, 1).contiguous()
    v = x["cache_v"].float().permute(0, 2, 1, 3).contiguous()
    s = (q @ k) * D ** -0.5
    if cap:
        s = cap * torch.tanh(s / cap)
    far = (x["lengths"][:, None] - torch.arange(M, device="cuda")[None, :])[:, None, None, :]
    if case["slopes"]:
        s = s - x["slopes"].view(1, G, H // G, 1) * far
    s = torch.where(far >= 0, s, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return ((p / p.sum(-1, keepdim=True)) @ v).view(B, 1, H, D)


def run(state):
    case, x = state["case"], state["x"]
    if own:
        if case["kind"] == "train":
            return _own(case, x)
        with torch.no_grad():
            return _own(case, x)
    with torch.no_grad():
        return {"conv": _plain_conv, "scan": _plain_scan, "attend": _plain_attend}[case["op"]](case, x)


# ---------------------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------------------
def work(case):
    B, N, kind = case["B"], case["N"], case["kind"]
    size = _TYPES[case["dtype"]].itemsize
    if case["op"] == "conv":
        C, W = case["C"], case["W"]
        tokens = B * N * C
        if kind == "train":          # x and dy in, y and dx out
            return {"bytes": size * 4 * tokens + 8 * C * (W + 1), "flops": tokens * (6 * W + 12)}
        state = 2 * B * (W - 1) * C * size
        return {"bytes": size * 2 * tokens + state + 4 * C * (W + 1), "flops": tokens * (2 * W + 6)}
    if case["op"] == "scan":
        C, S, G = case["C"], case["S"], case["G"]
        wide = 4 if case["gate"] else 3                # x, dt, (z) in and y out
        tokens = B * N
        moved = size * tokens * (C * wide + 2 * G * S) + 4 * C * (S + 2)
        flops = 7 * tokens * C * S
        if kind == "train":                            # dy in and the gradients out
            moved += size * tokens * (C * wide + 2 * G * S) + 4 * C * (S + 2)
            flops += 18 * tokens * C * S
        else:
            moved += 8 * B * C * S
        return {"bytes": moved, "flops": flops}
    H, G, D = case["H"], case["G"], case["D"]
    row = size * D
    if kind == "decode":
        seen = case["cache"] * 7 // 8
        return {"bytes": row * (2 * B * H + 2 * B * G * (seen + 2)), "flops": 4 * B * H * D * seen}
    if kind == "prefill":
        real, seen = N * 5 // 6, (case["cache"] - N) * 7 // 8
        pairs = real * seen + real * real // 2
        return {"bytes": row * B * (2 * N * H + 2 * G * (seen + 2 * real)), "flops": 4 * B * H * D * pairs}
    # random cuts: the mean of the summed squares of d documents is 2 N^2 / (d + 1)
    pairs = N * N // (max(1, case["docs"]) + 1)
    return {"bytes": row * B * N * (4 * H + 4 * G), "flops": 14 * B * H * D * pairs}


# ---------------------------------------------------------------------------------------
# The same outputs in 64 bits, token by token and pair by pair
# ---------------------------------------------------------------------------------------
def _exact_conv(case, x):
    B, N, C, W = (case[k] for k in "BNCW")
    train = case["kind"] == "train"
    wide = {n: x[n].detach().double().requires_grad_(train) for n in ("x", "weight", "bias")}
    rows = []
    windows = []
    for b in range(B):
        n = N if x["new"] is None else int(x["new"][b])
        ids = None if x["docs"] is None else x["docs"][b].tolist()
        # back[t]: how many earlier tokens of its own document token t has
        back = torch.full((N,), 10 ** 6, device="cuda")
        if ids is not None:
            count = []
            for t in range(N):
                count.append(count[-1] + 1 if t and ids[t] == ids[t - 1] else 0)
            back = torch.tensor(count, device="cuda")
        head = torch.zeros((W - 1, C), dtype=torch.float64, device="cuda") if train else x["state"][b].double()
        line = torch.cat((head, wide["x"][b]))
        pre = wide["bias"].expand(N, C)
        for k in range(W):
            tap = line[W - 1 - k:W - 1 - k + N] * wide["weight"][:, W - 1 - k]
            pre = pre + torch.where((back >= k)[:, None], tap, 0.0)
        y = pre / (1 + torch.exp(-pre)) if case["silu"] else pre
        live = torch.arange(N, device="cuda") < n
        if ids is not None:
            live = live & (x["docs"][b] >= 0)
        rows.append(torch.where(live[:, None], y, 0.0))
        windows.append(line.detach()[n:n + W - 1])
    y = torch.stack(rows)
    if not train:
        return [y.detach(), torch.stack(windows)]
    return [y.detach(), *torch.autograd.grad(y, [wide[n] for n in ("x", "weight", "bias")], x["dy"].double())]


def _exact_scan(case, x):
    B, N, C, S, G = (case[k] for k in "BNCSG")
    train = case["kind"] == "train"
    w = {n: (None if x[n] is None else x[n].detach().double()) for n in
         ("x", "dt", "A", "B", "C", "D", "dt_bias", "z")}
    per = C // G
    raw = w["dt"] + w["dt_bias"]
    delta = torch.where(raw > 40, raw, torch.log1p(torch.exp(raw.clamp_max(40))))
    live = torch.ones((B, N), dtype=torch.bool, device="cuda")
    if x["new"] is not None:
        live = torch.arange(N, device="cuda")[None, :] < x["new"][:, None]
    ids = x["docs"]
    if ids is not None:
        live = ids >= 0
    h = torch.zeros((B, C, S), dtype=torch.float64, device="cuda") if train else x["state"].double()
    before = []                                   # the state each token finds, for the way back
    lin = torch.zeros((B, N, C), dtype=torch.float64, device="cuda")
    chan = torch.arange(C, device="cuda") // per
    for t in range(N):
        if ids is not None and t:
            h = torch.where((ids[:, t] == ids[:, t - 1])[:, None, None], h, 0.0)
        if train:
            before.append(h)
        new = torch.exp(delta[:, t, :, None] * w["A"]) * h \
            + (delta[:, t] * w["x"][:, t])[..., None] * w["B"][:, t][:, chan]
        h = torch.where(live[:, t, None, None], new, h)
        lin[:, t] = (h * w["C"][:, t][:, chan]).sum(-1) + w["D"] * w["x"][:, t]
    sig = None if w["z"] is None else 1 / (1 + torch.exp(-w["z"]))
    y = lin if sig is None else lin * w["z"] * sig
    y = torch.where(live[..., None], y, 0.0)
    if not train:
        return [y, h]
    dy = torch.where(live[..., None], x["dy"].double(), 0.0)
    dz = None
    if sig is not None:
        dz = dy * lin * (sig + w["z"] * sig * (1 - sig))
        dy = dy * w["z"] * sig
    del lin, y
    out = {n: torch.zeros_like(w[n]) for n in ("x", "dt", "A", "B", "C", "D")}
    dh = torch.zeros_like(h)
    for t in range(N - 1, -1, -1):
        prev = before.pop()
        on = live[:, t, None, None]
        a = torch.exp(delta[:, t, :, None] * w["A"])
        Bt, Ct = w["B"][:, t][:, chan], w["C"][:, t][:, chan]
        dx_ = (delta[:, t] * w["x"][:, t])[..., None]
        now = a * prev + dx_ * Bt
        dh = dh + torch.where(on, dy[:, t, :, None] * Ct, 0.0)
        g = torch.where(on, dh, 0.0)
        out["C"][:, t] = torch.where(on, dy[:, t, :, None] * now, 0.0).view(B, G, per, S).sum(2)
        out["B"][:, t] = (g * dx_).view(B, G, per, S).sum(2)
        s = (g * Bt).sum(-1)
        p = g * a * prev
        out["A"] += (p * delta[:, t, :, None]).sum(0)
        out["dt"][:, t] = ((p * w["A"]).sum(-1) + s * w["x"][:, t]) / (1 + torch.exp(-raw[:, t]))
        out["x"][:, t] = s * delta[:, t] + dy[:, t] * w["D"]
        out["D"] += (dy[:, t] * w["x"][:, t]).sum(0)
        dh = torch.where(on, dh * a, dh)
        if ids is not None and t:
            dh = torch.where((ids[:, t] == ids[:, t - 1])[:, None, None], dh, 0.0)
    x = {n: x[n] for n in x}
    y = _exact_scan(dict(case, kind="values"), dict(x, state=torch.zeros_like(h), new=None))[0]
    grads = [out["x"], out["dt"], out["A"], out["B"], out["C"], out["D"], out["dt"].sum((0, 1))]
    return [y, *grads, *([] if dz is None else [dz])]


_ROWS = 2048      # queries of one piece


def _exact_attend(case, x):
    B, N, H, G, D = (case[k] for k in "BNHGD")
    kind, cap = case["kind"], case["cap"]
    train = kind == "train"
    q = x["q"].detach().double()
    if train:
        k, v = x["k"].detach().double(), x["v"].detach().double()
    else:
        k, v = x["cache_k"].double(), x["cache_v"].double()
        for b in range(B):
            n, at = (N if x["new"] is None else int(x["new"][b])), int(x["lengths"][b])
            k[b, at:at + n] = x["k"][b, :n].double()
            v[b, at:at + n] = x["v"][b, :n].double()
    y = torch.zeros_like(q)
    gq, gk, gv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        n = N if (train or x["new"] is None) else int(x["new"][b])
        off = 0 if train else int(x["lengths"][b])
        m = N if train else off + n
        j = torch.arange(m, device="cuda")
        pre = 0 if x["prefix"] is None else int(x["prefix"][b])
        for i0 in range(0, n, _ROWS):
            i = torch.arange(i0, min(n, i0 + _ROWS), device="cuda")
            hide = (j[None, :] > i[:, None] + off) & (j[None, :] >= pre)
            if x["docs"] is not None:
                ids = x["docs"][b]
                hide |= (ids[i][:, None] != ids[None, :]) | (ids[i] < 0)[:, None]
            none = hide.all(1)
            for h in range(H):
                c = h * G // H
                kk, vv = k[b, :m, c].contiguous(), v[b, :m, c].contiguous()
                qq = q[b, i, h]
                s = qq @ kk.t() / math.sqrt(D)
                if cap:
                    t = torch.tanh(s / cap)
                    s = t * cap
                if x["slopes"] is not None:
                    s = s - x["slopes"][h].double() * (i[:, None] + off - j[None, :]).abs()
                s = s.masked_fill(hide, -math.inf)
                s[none] = 0.0
                w = torch.softmax(s, dim=1)
                w[none] = 0.0
                o = w @ vv
                y[b, i, h] = o
                if not train:
                    continue
                d = x["dy"][b, i, h].double()
                ds = w * (d @ vv.t() - (d * o).sum(1, keepdim=True))
                if cap:
                    ds = ds * (1 - t * t)
                ds = ds / math.sqrt(D)
                gq[b, i, h] = ds @ kk
                gk[b, :m, c] += ds.t().contiguous() @ qq
                gv[b, :m, c] += w.t().contiguous() @ d
    return [y, gq, gk, gv] if train else [y, k, v]


def exact(case, seed):
    x = _inputs(case, seed)
    with torch.set_grad_enabled(case["op"] == "conv" and case["kind"] == "train"):
        return {"conv": _exact_conv, "scan": _exact_scan, "attend": _exact_attend}[case["op"]](case, x)
