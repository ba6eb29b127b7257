"""The token mixers on the GPU against their plain 64-bit forms (_mixers.py), at the sizes, masks
and layouts where they can go wrong."""
import functools
import math

import pytest
import torch

import causal_flare as cf
from _mixers import U, attention, check, conv, scan

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E32 = 2.0 ** -24


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, dtype=F32, std=1.0):
    return (torch.randn(shape, generator=g) * std).to(dtype).to(DEV)


def documents(g, B, N, most=4, pad=True):
    """Runs of random lengths, each row's last tokens padding; and the second row one document."""
    ids = torch.randint(0, N, (B, most), generator=g)
    ids = (torch.arange(N)[None, :, None] >= ids[:, None]).sum(-1).to(torch.int32)
    if pad:
        for b in range(B):
            ids[b, N - int(torch.randint(0, N // 3 + 1, (1,), generator=g)):] = -1
    if B > 1:
        ids[1] = 7
    return ids.to(DEV)


def close(got, ref, what, dtype, k):
    """`ref`: (value, magnitude) of fp32 arithmetic with k roundings on the way.  Where the terms'
    magnitudes pass the largest number of the type or of fp32, a term may be infinite: those
    entries are not looked at."""
    value, mag = ref
    over = ~(mag < torch.finfo(dtype).max / 4)
    if over.any():
        got = torch.where(over.to(got.device), 0.0, got.float()).to(got.dtype)
        value, mag = torch.where(over, 0.0, value), torch.where(over, 0.0, mag)
    check(got, value, U[dtype] * value.abs() + k * E32 * mag, what, dtype)


def sliced(x, extra=16):
    """The same values as a slice of a wider tensor."""
    wide = torch.full((*x.shape[:-1], x.shape[-1] + 2 * extra), float("nan"), dtype=x.dtype, device=x.device)
    wide[..., extra:-extra] = x
    return wide[..., extra:-extra]


# ---------------------------------------------------------------------------------------
# Short convolution
# ---------------------------------------------------------------------------------------
# W taps, the bias, two exponentials and a quotient of the gate: some 16 roundings; the
# exponential's argument is of the size of the magnitude itself
CONV_K = 64


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B, N, C, W, docs", [
    (1, 1, 8, 4, False), (2, 2, 16, 4, False), (3, 3, 24, 3, False), (2, 33, 40, 2, False), (1, 67, 7, 4, False),
    (2, 131, 64, 4, True), (3, 40, 5, 3, True), (2, 64, 48, 2, True), (1, 1030, 512, 4, False), (9, 65, 1024, 4, True),
])
def test_conv(dtype, B, N, C, W, docs):
    g = gen(100 * N + C)
    x, w, b = normal(g, B, N, C, dtype=dtype), normal(g, C, W, std=0.5), normal(g, C, std=0.3)
    dy = normal(g, B, N, C, dtype=dtype)
    ids = documents(g, B, N) if docs else None
    for silu, bias in ((True, b), (False, None)):
        leaves = [t.clone().requires_grad_() for t in (x, w)] + ([bias.clone().requires_grad_()] if silu else [])
        y = cf.short_convolution(leaves[0], leaves[1], leaves[2] if silu else None,
                                 activation="silu" if silu else None, document_ids=ids)
        grads = torch.autograd.grad(y, leaves, dy)
        ref = conv(x, w, bias, silu, ids, dy=dy)
        close(y, ref["y"], "y", dtype, CONV_K)
        close(grads[0], ref["dx"], "dx", dtype, CONV_K)
        # the sums over tokens: each partial sum of 32 tokens and then their column sums
        close(grads[1], ref["dweight"], "dweight", F32, CONV_K + 32 + B * N / 8)
        if silu:
            close(grads[2], ref["dbias"], "dbias", F32, CONV_K + 32 + B * N / 8)


@pytest.mark.parametrize("B, N, C, W, docs", [(1, 2101, 2050, 4, 3), (2, 4099, 2052, 3, 0)])
def test_conv_of_longer_runs(B, N, C, W, docs):
    test_conv(BF16, B, N, C, W, docs)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B, N, C, W", [(4, 1, 16, 4), (5, 2, 24, 4), (6, 9, 10, 3), (8, 70, 64, 2)])
def test_conv_prefill_and_decode(dtype, B, N, C, W):
    g = gen(N + C)
    x, w, b = normal(g, B, N, C, dtype=dtype), normal(g, C, W, std=0.5), normal(g, C, std=0.3)
    window = normal(g, B, W - 1, C, dtype=dtype)
    lengths = torch.arange(B, dtype=torch.int64, device=DEV).clamp(max=N)
    x[torch.arange(N, device=DEV)[None] >= lengths[:, None]] = float("nan")   # behind the end
    before = window.clone()
    y, state = cf.short_convolution_prefill(x, w, b, "silu", {"window": window}, lengths)
    ref = conv(x, w, b, True, lengths=lengths, window=window)
    close(y, ref["y"], "y", dtype, CONV_K)
    assert torch.equal(state["window"].double().cpu(), ref["window"][0])
    assert torch.equal(window, before)
    # lengths out of range are taken as 0 and N
    y2, s2 = cf.short_convolution_prefill(x, w, b, "silu", {"window": window},
                                          torch.where(lengths == 0, -5, lengths).to(torch.int32))
    assert torch.equal(y2, y) and torch.equal(s2["window"], state["window"])
    x = x.nan_to_num(0.0)
    y_all, s_all = cf.short_convolution_prefill(x, w, b, "silu")
    ref = conv(x, w, b, True)
    close(y_all, ref["y"], "y from nothing", dtype, CONV_K)
    st = {"window": torch.zeros((B, W - 1, C), dtype=dtype, device=DEV)}
    held = st["window"]
    for t in range(N):
        step, st = cf.short_convolution_decode(x[:, t], w, b, "silu", st)
        close(step[:, 0], (ref["y"][0][:, t], ref["y"][1][:, t]), f"step {t}", dtype, CONV_K)
    assert st["window"] is held and torch.equal(held, s_all["window"])
    mask = torch.arange(B, device=DEV) % 2
    old = held.clone()
    step, st = cf.short_convolution_decode(x[:, :1], w, b, None, st, attention_mask=mask)
    assert torch.equal(st["window"][0::2], old[0::2]) and not step[0::2].any()
    assert torch.equal(st["window"][1::2, -1], x[1::2, 0])


def test_conv_reads_slices_and_other_types_in_place():
    g = gen(1)
    x, w, b = normal(g, 2, 50, 64, dtype=BF16), normal(g, 64, 4), normal(g, 64)
    y = cf.short_convolution(x, w, b, "silu")
    assert torch.equal(cf.short_convolution(sliced(x), w, b, "silu"), y)
    assert torch.equal(cf.short_convolution(sliced(x, 3), w, b, "silu"), y)                 # no 16-byte rows
    assert torch.equal(cf.short_convolution(x.transpose(0, 1).contiguous().transpose(0, 1), w, b, "silu"), y)
    assert torch.equal(cf.short_convolution(x.transpose(1, 2).contiguous().transpose(1, 2), w, b, "silu"), y)
    assert torch.equal(cf.short_convolution(x, w.double(), b.double(), "silu"), y)
    one = cf.short_convolution(x[:1].expand(3, 50, 64), w, b, "silu")
    assert torch.equal(one[2], y[0])
    w16 = w.to(BF16).requires_grad_()
    assert torch.autograd.grad(cf.short_convolution(x, w16).sum(), w16)[0].dtype is BF16
    assert cf.short_convolution(x[:, :0], w, b).shape == (2, 0, 64)
    assert cf.short_convolution(x[:0], w, b).shape == (0, 50, 64)


# ---------------------------------------------------------------------------------------
# State space scan
# ---------------------------------------------------------------------------------------
def scan_inputs(g, B, N, C, S, G, dtype, gate=True, extras=True):
    x = {"x": normal(g, B, N, C, dtype=dtype), "dt": normal(g, B, N, C, dtype=dtype, std=0.7),
         "A": -torch.rand((C, S), generator=g).mul(4).to(DEV), "B": normal(g, B, N, G, S, dtype=dtype),
         "C": normal(g, B, N, G, S, dtype=dtype)}
    x["D"] = normal(g, C) if extras else None
    x["z"] = normal(g, B, N, C, dtype=dtype) if gate else None
    x["dt_bias"] = normal(g, C) - 1.5 if extras else None
    return x


SCANS = [
    # B, N, C, S, G, documents, gate and extras
    (1, 1, 3, 1, 1, False, False), (2, 2, 64, 16, 1, False, True), (1, 15, 70, 16, 1, False, True),
    (2, 33, 130, 16, 2, False, True), (1, 129, 20, 8, 1, False, True), (2, 257, 48, 4, 1, False, False),
    (1, 300, 260, 16, 4, True, True), (3, 100, 32, 24, 1, True, True), (2, 131, 66, 33, 2, True, True),
    (1, 70, 16, 64, 1, False, True), (2, 64, 128, 32, 1, True, False), (2, 257, 48, 4, 1, False, "positive"),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B, N, C, S, G, docs, more", SCANS)
def test_scan(dtype, B, N, C, S, G, docs, more):
    g = gen(N * 7 + C)
    t = scan_inputs(g, B, N, C, S, G, dtype, more, more)
    if more == "positive":                                     # steps as they are, and no growing states
        t["dt"], t["dt_bias"], more = t["dt"].abs(), None, False
    ids = documents(g, B, N) if docs else None
    dy = normal(g, B, N, C, dtype=dtype)
    names = [n for n in t if t[n] is not None]
    leaves = {n: t[n].clone().requires_grad_() for n in names}
    y = cf.state_space_scan(*[leaves.get(n) for n in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")],
                            dt_softplus=more, document_ids=ids)
    grads = torch.autograd.grad(y, [leaves[n] for n in names], dy)
    ref = scan(**t, softplus=more, ids=ids, dy=dy)
    k = ref["k"]
    close(y, ref["y"], "y", dtype, k)
    with torch.no_grad():                                      # chunks of another length
        close(cf.state_space_scan(*[t[n] for n in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")], dt_softplus=more,
                                  document_ids=ids), ref["y"], "y without gradients", dtype, k)
    for n, got in zip(names, grads):
        # dB and dC add up channels, the parameters' gradients all tokens
        far = C / G if n in "BC" else B * N if n in ("A", "D", "dt_bias") else 0
        close(got, ref["d" + n], "d" + n, F32 if n in ("A", "D", "dt_bias") else dtype, 2 * k + far)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B, N, C, S, G", [(4, 1, 16, 16, 1), (5, 33, 70, 16, 2), (3, 260, 40, 8, 1), (4, 90, 64, 20, 1),
                                           (3, 65, 16, 64, 1)])
def test_scan_prefill_and_decode(dtype, B, N, C, S, G):
    g = gen(N + C)
    t = scan_inputs(g, B, N, C, S, G, dtype)
    names = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")
    lengths = torch.tensor([N, 0, N // 2, max(0, N - 1), 1][:B], device=DEV).clamp(max=N)
    h0 = normal(g, B, C, S)
    gone = torch.arange(N, device=DEV)[None] >= lengths[:, None]
    for n in ("x", "dt", "B", "C", "z"):
        t[n][gone] = float("nan")
    before = h0.clone()
    y, state = cf.state_space_scan_prefill(*[t[n] for n in names], dt_softplus=True, state={"h": h0}, lengths=lengths)
    ref = scan(**t, softplus=True, lengths=lengths, h0=h0)
    close(y, ref["y"], "y", dtype, ref["k"])
    close(state["h"], ref["h"], "h", F32, ref["k"])
    assert torch.equal(h0, before)
    t = {n: v.nan_to_num(0.0) for n, v in t.items()}
    ref = scan(**t, softplus=True, h0=h0)
    st = {"h": h0.clone()}
    held = st["h"]
    for i in range(min(N, 40)):
        step, st = cf.state_space_scan_decode(t["x"][:, i], t["dt"][:, i], t["A"], t["B"][:, i], t["C"][:, i], t["D"],
                                              t["z"][:, i], t["dt_bias"], True, st)
        value, mag = ref["y"]
        close(step[:, 0], (value[:, i], mag[:, i]), f"step {i}", dtype, ref["k"])
    assert st["h"] is held
    if N <= 40:
        close(held, ref["h"], "h after steps", F32, ref["k"])
    old = held.clone()
    mask = (torch.arange(B, device=DEV) % 2)[:, None]
    i = slice(0, 1)
    step, st = cf.state_space_scan_decode(t["x"][:, i], t["dt"][:, i], t["A"], t["B"][:, i], t["C"][:, i], state=st,
                                          attention_mask=mask)
    assert torch.equal(st["h"][0::2], old[0::2]) and not step[0::2].any()
    one = {n: t[n][1::2, i] for n in ("x", "dt", "B", "C")}
    ref = scan(**one, A=t["A"], h0=old[1::2])
    close(step[1::2], ref["y"], "y of the others", dtype, ref["k"])
    close(st["h"][1::2], ref["h"], "h of the others", F32, ref["k"])


def test_scan_of_growing_states_that_are_zero():
    """A decay past fp32 over a chunk (2^180) leaves a state of 0, and one of 2^-100, what it is."""
    B, N, C, S = 1, 400, 64, 16
    z = lambda *s: torch.zeros(s, device=DEV)
    x, dt, A = z(B, N, C), z(B, N, C) + 1, z(C, S) + math.log(2.0) * 180 / 300
    h0 = z(B, C, S)
    h0[:, 0] = 2.0 ** -150 * 2.0 ** 50
    y, st = cf.state_space_scan_prefill(x, dt, A, z(B, N, S), z(B, N, S) + 1, state={"h": h0}, lengths=torch.tensor([300], device=DEV))
    assert not st["h"][:, 1:].any() and not y[:, :, 1:].any()
    assert torch.allclose(st["h"][:, 0], torch.full((B, S), 2.0 ** 80, device=DEV), rtol=1e-3)


def test_scan_reads_slices_and_promotes():
    g = gen(5)
    t = scan_inputs(g, 2, 50, 64, 16, 1, BF16)
    order = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")
    y = cf.state_space_scan(*[t[n] for n in order], dt_softplus=True)
    s = {n: sliced(v, 3) if n in ("x", "dt", "B", "C", "z") else v for n, v in t.items()}
    assert torch.equal(cf.state_space_scan(*[s[n] for n in order], dt_softplus=True), y)
    s = dict(t, B=t["B"][:, :, 0], C=t["C"][:, :, 0])
    assert torch.equal(cf.state_space_scan(*[s[n] for n in order], dt_softplus=True), y)
    s = dict(t, dt=t["dt"].float())
    assert cf.state_space_scan(*[s[n] for n in order], dt_softplus=True).dtype is BF16
    assert cf.state_space_scan(*[t[n][:, :0] if n in ("x", "dt", "B", "C", "z") else t[n] for n in order]).shape == (2, 0, 64)
    # B and C broadcast over the batch: their gradients add up over it
    one = {n: t[n][:1].clone().requires_grad_() for n in ("B", "C")}
    wide = {n: t[n][:1].expand_as(t[n]).clone().requires_grad_() for n in ("B", "C")}
    for leaf in (one, wide):
        s = dict(t, **{n: leaf[n].expand(2, 50, 1, 16) for n in leaf})
        cf.state_space_scan(*[s[n] for n in order], dt_softplus=True).sum().backward()
    assert torch.allclose(one["B"].grad.float(), wide["B"].grad.float().sum(0, keepdim=True), rtol=2 ** -6, atol=2 ** -4)


# ---------------------------------------------------------------------------------------
# Softmax attention
# ---------------------------------------------------------------------------------------
ATTENTION = [
    # B, N, H, G, D, options
    (1, 1, 1, 1, 16, ""), (2, 2, 2, 1, 32, "cap"), (1, 15, 4, 2, 48, "slopes"), (2, 63, 2, 2, 64, "docs"),
    (1, 64, 4, 1, 64, "cap slopes"), (2, 65, 2, 2, 80, "full"), (2, 130, 4, 2, 96, "prefix"),
    (3, 200, 3, 1, 128, "docs slopes"), (2, 257, 2, 1, 128, "cap docs prefix"), (1, 191, 2, 2, 112, "full docs slopes"),
    (2, 300, 1, 1, 64, "prefix slopes"), (1, 513, 2, 2, 64, "docs"), (1, 100, 2, 1, 64, "negative"),
    (1, 140, 2, 2, 128, "wide-cap slopes negative"), (1, 1100, 1, 1, 32, "docs slopes"), (1, 1537, 2, 1, 48, "cap"),
    (1, 200, 2, 2, 64, "cap rising slopes"),
]


def attention_options(g, what, B, N, H):
    o = {}
    if "cap" in what:
        o["softcap"] = 50.0 if "wide-cap" in what else 3.0
    if "negative" in what:
        o["scale"] = -0.2
    if "slopes" in what:
        o["slopes"] = torch.tensor([2.0 ** -(h + 1) for h in range(H)]).to(DEV) * (-1 if "rising" in what else 1)
    if "docs" in what:
        o["document_ids"] = documents(g, B, N)
    if "prefix" in what:
        o["prefix_lengths"] = torch.tensor([N // 2, N + 3, 0][:B], device=DEV)
    if "full" in what:
        o["causal"] = False
    return o


def plain(o):
    o = dict(o)
    return dict(scale=o.get("scale"), softcap=o.get("softcap"), slopes=o.get("slopes"), ids=o.get("document_ids"),
                prefix=o.get("prefix_lengths"), causal=o.get("causal", True))


def close_attention(got, ref, what, dtype):
    value, tol = ref
    check(got, value, U[dtype] * (value.abs() + tol) + tol, what, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B, N, H, G, D, what", ATTENTION)
def test_attention(dtype, B, N, H, G, D, what):
    g = gen(N + D)
    q, k, v, dy = (normal(g, B, N, n, D, dtype=dtype, std=s) for n, s in ((H, 2.0), (G, 1.0), (G, 1.0), (H, 1.0)))
    o = attention_options(g, what, B, N, H)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    y = cf.softmax_attention(*leaves, **o)
    grads = torch.autograd.grad(y, leaves, dy)
    unit, tiny = (0.0 if dtype is F32 else U[dtype]), (2.0 ** -25 if dtype is F16 else 2.0 ** -126)
    ref = attention(q, k, v, **plain(o), dy=dy, unit=unit, tiny=tiny)
    close_attention(y, ref["y"], "y", dtype)
    with torch.no_grad():
        assert torch.equal(cf.softmax_attention(q, k, v, **o), y)
    for n, got in zip(("dq", "dk", "dv"), grads):
        close_attention(got, ref[n], n, dtype)


@pytest.mark.parametrize("dtype, B, N, H, G", [(BF16, 34, 150, 16, 4), (F32, 20, 130, 16, 16), (F16, 36, 129, 16, 1)])
def test_attention_of_many_documents_in_order_of_cost(dtype, B, N, H, G):
    """More workgroups than run at once: blocks start in the order of what they cost."""
    g = gen(N)
    D = 32
    q, k, v, dy = (normal(g, B, N, n, D, dtype=dtype) for n in (H, G, G, H))
    ids = documents(g, B, N)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    y = cf.softmax_attention(*leaves, document_ids=ids)
    grads = torch.autograd.grad(y, leaves, dy)
    unit, tiny = (0.0 if dtype is F32 else U[dtype]), (2.0 ** -25 if dtype is F16 else 2.0 ** -126)
    ref = attention(q, k, v, ids=ids, dy=dy, unit=unit, tiny=tiny)
    close_attention(y, ref["y"], "y", dtype)
    for n, got in zip(("dq", "dk", "dv"), grads):
        close_attention(got, ref[n], n, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B, T, H, G, D, S, what", [
    (4, 1, 2, 1, 64, 70, ""), (5, 7, 4, 2, 128, 200, "cap"), (5, 130, 2, 2, 48, 400, "slopes"),
    (5, 150, 4, 1, 96, 300, "prefix slopes"), (5, 64, 2, 2, 32, 129, "prefix"),
    (5, 3, 4, 2, 64, 2500, "slopes"), (3, 140, 2, 1, 128, 1300, "cap prefix"), (5, 1, 1, 1, 16, 1100, "wide-cap")])
def test_attention_prefill(dtype, B, T, H, G, D, S, what):
    g = gen(T + D)
    q, k, v = (normal(g, B, T, n, D, dtype=dtype) for n in (H, G, G))
    ck, cv = (normal(g, B, S, G, D, dtype=dtype) for _ in range(2))
    held = torch.tensor([0, S - T, (S - T) // 2, -1, S - T + 1][:B], device=DEV)
    new = torch.tensor([T, T, T // 2, T, T][:B], device=DEV)
    o = attention_options(g, what, B, S, H)
    if "prefix_lengths" in o:
        o["prefix_lengths"] = torch.tensor([T // 2, S, 5, 0, 0][:B], device=DEV)
    ck[2, int(held[2]) + int(new[2]):] = float("nan")             # what a cache holds behind its end
    cv[2, int(held[2]) + int(new[2]):] = float("inf")
    cache = {"k": ck.clone(), "v": cv.clone()}
    y, same = cf.softmax_attention_prefill(q, k, v, cache, held, **o, new_lengths=new)
    assert same is cache
    unit, tiny = (0.0 if dtype is F32 else U[dtype]), (2.0 ** -25 if dtype is F16 else 2.0 ** -126)
    for b in range(B):
        n, at = int(new[b]), int(held[b])
        want_k, want_v = ck[b].clone(), cv[b].clone()
        if at >= 0 and at + n <= S:
            want_k[at:at + n], want_v[at:at + n] = k[b, :n], v[b, :n]
            ref = attention(q[b:b + 1, :n], want_k[None, :at + n], want_v[None, :at + n], softcap=o.get("softcap"),
                            slopes=o.get("slopes"), offset=[at], unit=unit, tiny=tiny,
                            prefix=o["prefix_lengths"][b:b + 1] if "prefix_lengths" in o else None)
            close_attention(y[b:b + 1, :n], ref["y"], f"y of {b}", dtype)
            assert not y[b, n:].any()
        elif at < 0:
            assert not y[b].any()
        else:
            assert y[b].isnan().all()
        assert torch.equal(cache["k"][b].nan_to_num(9.0), want_k.nan_to_num(9.0))
        assert torch.equal(cache["v"][b].nan_to_num(9.0), want_v.nan_to_num(9.0))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B, H, G, D, S, what", [
    (6, 1, 1, 16, 5, ""), (6, 4, 2, 64, 130, "cap"), (6, 16, 1, 128, 1100, "slopes"), (6, 24, 1, 48, 300, "cap slopes"),
    (6, 8, 8, 96, 257, ""), (40, 8, 4, 128, 700, "cap"), (2, 34, 2, 32, 5000, "slopes")])
def test_attention_decode(dtype, B, H, G, D, S, what):
    g = gen(S + D)
    q, k, v = (normal(g, B, n, D, dtype=dtype) for n in (H, G, G))
    ck, cv = (normal(g, B, S, G, D, dtype=dtype) for _ in range(2))
    held = torch.tensor(([0, S - 1, S // 2, -1, S, min(127, S - 1)] + [(37 * b) % S for b in range(B)])[:B], device=DEV)
    o = attention_options(g, what, B, S, H)
    for b in range(B):
        ck[b, max(0, int(held[b])):] = float("nan")
        cv[b, max(0, int(held[b])):] = float("inf")
    cache = {"k": ck.clone(), "v": cv.clone()}
    y, same = cf.softmax_attention_decode(q, k, v, cache, held, **o)
    assert same is cache and y.shape == (B, 1, H, D)
    unit, tiny = (0.0 if dtype is F32 else U[dtype]), (2.0 ** -25 if dtype is F16 else 2.0 ** -126)
    for b in range(B):
        at = int(held[b])
        want_k, want_v = ck[b].clone(), cv[b].clone()
        if 0 <= at < S:
            want_k[at], want_v[at] = k[b], v[b]
            ref = attention(q[b:b + 1, None], want_k[None, :at + 1], want_v[None, :at + 1], softcap=o.get("softcap"),
                            slopes=o.get("slopes"), offset=[at], unit=unit, tiny=tiny)
            close_attention(y[b:b + 1], ref["y"], f"y of {b}", dtype)
        else:
            assert y[b].isnan().all() if at >= S else not y[b].any()
        assert torch.equal(cache["k"][b].nan_to_num(9.0), want_k.nan_to_num(9.0))
        assert torch.equal(cache["v"][b].nan_to_num(9.0, posinf=9.0), want_v.nan_to_num(9.0, posinf=9.0))


@pytest.mark.parametrize("cap", [3.0, 30.0, 200.0])
def test_capped_scores_of_fp32_keep_their_digits(cap):
    """As near to 64 bits as elementary fp32 operations, whose scores are off by the same few roundings
    (2.5 times their error leaves room for the order of the sums and exponentials of one unit)."""
    g = gen(int(cap))
    q, k, v, dy = (normal(g, 2, 300, 2, 64, std=s) for s in (2.0, 1.0, 1.0, 1.0))

    def whole(dtype):
        a, b, c = (t.to(dtype).transpose(1, 2).contiguous().requires_grad_() for t in (q, k, v))
        x = cap * torch.tanh((a @ b.transpose(-1, -2).contiguous()) * 0.125 / cap)
        x = x.masked_fill(torch.ones(300, 300, device=DEV, dtype=torch.bool).triu(1), float("-inf"))
        y = torch.softmax(x, -1) @ c
        grads = torch.autograd.grad(y, (a, b, c), dy.to(dtype).transpose(1, 2))
        return [t.detach().double().transpose(1, 2) for t in (y, *grads)]

    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    y = cf.softmax_attention(*leaves, softcap=cap)
    got = [y.detach().double(), *(t.double() for t in torch.autograd.grad(y, leaves, dy))]
    cache = {n: torch.cat([t[:, :299], torch.zeros_like(t[:, :1])], 1) for n, t in (("k", k), ("v", v))}
    held = torch.full((2,), 299, device=DEV, dtype=torch.int32)
    last = cf.softmax_attention_decode(q[:, 299], k[:, 299], v[:, 299], cache, held, softcap=cap)[0].double()
    want, plain32 = whole(torch.float64), whole(torch.float32)
    for name, a, b, c in zip(("y", "dq", "dk", "dv"), got, plain32, want):
        assert (a - c).norm() <= 2.5 * (b - c).norm(), (name, float((a - c).norm() / c.norm()), float((b - c).norm() / c.norm()))
    a, b, c = last, plain32[0][:, 299:], want[0][:, 299:]
    assert (a - c).norm() <= 2.5 * (b - c).norm(), ("token", float((a - c).norm() / c.norm()), float((b - c).norm() / c.norm()))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_attention_decode_of_many_parts(dtype):
    # 128 keys a workgroup: one sequence with nothing, one with all and one with half of 86 parts
    test_attention_decode(dtype, 3, 4, 2, 48, 20011, "cap slopes")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B, N, H, G, D, what", [
    (1, 2900, 6, 2, 80, "docs slopes"), (2, 1300, 4, 4, 128, "prefix"), (1, 2100, 1, 1, 64, "full cap"), (1, 1800, 5, 1, 32, "")])
def test_attention_of_few_rows_in_parts(dtype, B, N, H, G, D, what):
    test_attention(dtype, B, N, H, G, D, what)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("H, G, D, sloped", [(4, 2, 64, False), (16, 4, 128, True), (3, 3, 16, True)])
def test_attention_decode_of_any_integer_lengths(dtype, H, G, D, sloped):
    """Slices of one projection, rows that sit out and a full cache: the same for int32 lengths and others."""
    g = gen(D)
    qkv = normal(g, 5, 1, H + 2 * G, D, dtype=dtype)
    cache = {n: normal(g, 5, 300, G, D, dtype=dtype) for n in "kv"}
    held = torch.tensor([0, 299, 300, -1, 7], device=DEV, dtype=torch.int32)
    o = dict(softcap=20, slopes=normal(g, H).abs() if sloped else None)
    runs = []
    for rows in (qkv, qkv[:, 0], qkv.clone()[:, 0]):
        for lens in (held, held.long(), held.to(torch.int16)):
            c = {n: t.clone() for n, t in cache.items()}
            y, _ = cf.softmax_attention_decode(*rows.split((H, G, G), -2), c, lens, **o)
            runs.append([y.nan_to_num(7.0), c["k"], c["v"]])
    assert all(same(r, runs[0]) for r in runs)
    assert runs[0][0][2].eq(7.0).all() and not runs[0][0][3].any() and runs[0][0][4].ne(7.0).any()


def test_attention_reads_slices_and_promotes():
    g = gen(8)
    qkv = normal(g, 2, 70, 8, 64, dtype=BF16)
    q, k, v = qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:]
    y = cf.softmax_attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(cf.softmax_attention(q, k, v), y)
    assert torch.equal(cf.softmax_attention(*[sliced(t, 3) for t in (q, k, v)]), y)
    assert torch.equal(cf.softmax_attention(*[t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]), y)
    assert cf.softmax_attention(q.float(), k, v).dtype is F32
    assert cf.softmax_attention(q[:, :0], k[:, :0], v[:, :0]).shape == (2, 0, 4, 64)
    # one key head for a batch of sequences: its gradient adds up over them
    kk = k[:1].clone().requires_grad_()
    wide = k[:1].expand_as(k).clone().requires_grad_()
    a = torch.autograd.grad(cf.softmax_attention(q, kk.expand_as(k), v).float().sum(), kk)[0]
    b = torch.autograd.grad(cf.softmax_attention(q, wide, v).float().sum(), wide)[0]
    assert torch.allclose(a.float(), b.float().sum(0, keepdim=True), rtol=2 ** -6, atol=2 ** -7)


# ---------------------------------------------------------------------------------------
# What is masked may hold anything
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
def test_padding_and_other_documents_may_hold_anything(dtype, poison):
    g = gen(11)
    B, N, C, S, H, D = 1, 150, 32, 16, 2, 64
    ids = torch.zeros((B, N), dtype=torch.int32)
    ids[:, 60:110], ids[:, 110:] = 1, -1
    ids = ids.to(DEV)
    bad = torch.arange(N, device=DEV) >= 110

    def both(make, run):
        """Results with finite values behind the mask, and with the poison there."""
        clean = make()
        dirty = [t.clone() for t in clean]
        for t in dirty:
            if t.dim() > 2 and t.shape[1] == N:
                t[:, bad] = poison
        return run(clean), run(dirty)

    def of_conv(t):
        leaves = [v.clone().requires_grad_() for v in t[:3]]
        y = cf.short_convolution(*leaves, activation="silu", document_ids=ids)
        return [y, *torch.autograd.grad(y, leaves, t[3])]

    def of_scan(t):
        leaves = [v.clone().requires_grad_() for v in t[:8]]
        y = cf.state_space_scan(*leaves, dt_softplus=True, document_ids=ids)
        return [y, *torch.autograd.grad(y, leaves, t[8])]

    def of_attention(t):
        leaves = [v.clone().requires_grad_() for v in t[:3]]
        y = cf.softmax_attention(*leaves, document_ids=ids)
        return [y, *torch.autograd.grad(y, leaves, t[3])]

    cases = (
        (lambda: [normal(g, B, N, C, dtype=dtype), normal(g, C, 4), normal(g, C), normal(g, B, N, C, dtype=dtype)], of_conv),
        (lambda: [*scan_inputs(g, B, N, C, S, 1, dtype).values(), normal(g, B, N, C, dtype=dtype)], of_scan),
        (lambda: [normal(g, B, N, H, D, dtype=dtype) for _ in range(4)], of_attention),
    )
    for make, run in cases:
        a, b = both(make, run)
        for x, y in zip(a, b):
            assert torch.equal(x, y)
            if x.dim() > 2 and x.shape[1] == N:
                assert not x[:, bad].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("where", ["k", "v", "q"])
def test_attention_keeps_infinite_values_to_who_sees_them(dtype, where):
    """A later token, or one of another document, that holds an infinite value or NaN."""
    g = gen(12)
    N, H, D, at = 140, 2, 64, 70
    t = {n: normal(g, 1, N, H, D, dtype=dtype) for n in ("q", "k", "v")}
    ids = torch.zeros((1, N), dtype=torch.int32, device=DEV)
    ids[:, 100:] = 1
    dy = normal(g, 1, N, H, D, dtype=dtype)
    apart = [*range(at), *range(100, N)]                             # who does not see token 70
    for poison in (float("inf"), float("nan")):
        dirty = {n: v.clone() for n, v in t.items()}
        dirty[where][0, at, 0, 5] = poison
        outs = []
        for x in (t, dirty):
            leaves = [x[n].clone().requires_grad_() for n in ("q", "k", "v")]
            y = cf.softmax_attention(*leaves, document_ids=ids)
            outs.append([y, *torch.autograd.grad(y, leaves, dy)])
        y0, y1 = outs[0][0], outs[1][0]
        assert torch.equal(y0[:, apart], y1[:, apart])
        assert torch.equal(y0[:, :, 1], y1[:, :, 1])                 # the other head
        # gradients of queries that do not see it, and of keys that only such queries see
        assert torch.equal(outs[0][1][:, apart], outs[1][1][:, apart])
        assert torch.equal(outs[0][2][:, 100:], outs[1][2][:, 100:])
        assert torch.equal(outs[0][3][:, 100:], outs[1][3][:, 100:])
        if where == "v":
            sees = y1[0, at:100, 0, 5]
            assert sees.isnan().all() if math.isnan(poison) else (sees == poison).all()
        else:
            assert not y1[0, at, 0].isfinite().all()
    # a gradient that is infinite in one row stays with the keys that row sees, and reaches them all
    leaves = [t[n].clone().requires_grad_() for n in ("q", "k", "v")]
    dirty = dy.clone()
    dirty[0, at, 0, 5] = float("inf")
    for o in ({"document_ids": ids}, {}):
        y = cf.softmax_attention(*leaves, **o)
        clean, got = torch.autograd.grad(y, leaves, dy, retain_graph=True), torch.autograd.grad(y, leaves, dirty)
        rows = [i for i in range(N) if i != at]
        assert torch.equal(clean[0][:, rows], got[0][:, rows])
        for i in (1, 2):
            assert torch.equal(clean[i][:, at + 1:], got[i][:, at + 1:])
            assert not got[i][0, :at + 1, 0].isfinite().all(-1).any()
    # without documents a key that is infinite is seen by every later query
    if where != "v":
        dirty = {n: v.clone() for n, v in t.items()}
        dirty[where][0, at, 0, 5] = float("inf")
        leaves = [dirty[n].requires_grad_() for n in ("q", "k", "v")]
        grads = torch.autograd.grad(cf.softmax_attention(*leaves), leaves, dy)
        seen = range(at + 1) if where == "q" else range(N)
        assert not grads[1][0, [*seen][:at + 1], 0].isfinite().all(-1).any()
        assert all(x[:, :, 1].isfinite().all() for x in grads)


def test_a_query_that_sees_nothing():
    q, k, v = (normal(gen(i), 2, 80, 2, 32).requires_grad_() for i in range(3))
    ids = torch.full((2, 80), -1, dtype=torch.int64, device=DEV)
    y = cf.softmax_attention(q, k, v, document_ids=ids)
    assert not y.any()
    assert all(not t.any() for t in torch.autograd.grad(y, (q, k, v), torch.ones_like(y)))


# ---------------------------------------------------------------------------------------
# Streams, graphs, repeats
# ---------------------------------------------------------------------------------------
def _calls():
    """{name: (inputs, function of them)}: one call of each entry point."""
    g = gen(21)
    B, N, C, S, H, G, D = 2, 200, 96, 16, 4, 2, 64
    ids = documents(g, B, N)
    t = scan_inputs(g, B, N, C, S, 1, BF16)
    xs, w, b, dy = normal(g, B, N, C, dtype=BF16), normal(g, C, 4), normal(g, C), normal(g, B, N, C, dtype=BF16)
    q, k, v = (normal(g, B, N, n, D, dtype=BF16) for n in (H, G, G))
    do = normal(g, B, N, H, D, dtype=BF16)
    lens = torch.tensor([150, 90], device=DEV, dtype=torch.int32)
    cache = {n: normal(g, B, 400, G, D, dtype=BF16) for n in "kv"}

    def train(f, leaves, d):
        y = f(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, d)]

    def leaves(*ts):
        return [x.clone().requires_grad_() for x in ts]

    conv_leaves, scan_leaves, attn_leaves = leaves(xs, w, b), leaves(*t.values()), leaves(q, k, v)
    window, h = normal(g, B, 3, C, dtype=BF16), normal(g, B, C, S)
    step = {n: x[:, 0] if x.dim() > 2 and x.shape[1] == N else x for n, x in t.items()}

    def conv_step():
        y, s = cf.short_convolution_decode(xs[:, 0], w, b, "silu", {"window": window.clone()})
        return [y, s["window"]]

    def scan_step():
        y, s = cf.state_space_scan_decode(**step, dt_softplus=True, state={"h": h.clone()})
        return [y, s["h"]]

    def prefill_attention():
        y, c = cf.softmax_attention_prefill(q, k, v, {n: x.clone() for n, x in cache.items()}, lens, softcap=20.0)
        return [y, c["k"], c["v"]]

    def decode_attention():
        y, c = cf.softmax_attention_decode(q[:, 0], k[:, 0], v[:, 0], {n: x.clone() for n, x in cache.items()}, lens)
        return [y, c["k"], c["v"]]

    return {
        "conv": lambda: train(lambda *a: cf.short_convolution(*a, activation="silu", document_ids=ids), conv_leaves, dy),
        "conv_prefill": lambda: [cf.short_convolution_prefill(xs, w, b, "silu", {"window": window}, lens)[0]],
        "conv_decode": conv_step,
        "scan": lambda: train(lambda *a: cf.state_space_scan(*a, dt_softplus=True, document_ids=ids), scan_leaves, dy),
        "scan_prefill": lambda: list(cf.state_space_scan_prefill(**t, dt_softplus=True, state={"h": h}, lengths=lens)[1].values()),
        "scan_decode": scan_step,
        "attention": lambda: train(lambda *a: cf.softmax_attention(*a, softcap=20.0, document_ids=ids), attn_leaves, do),
        "attention_prefill": prefill_attention,
        "attention_decode": decode_attention,
    }


NAMES = ("conv", "conv_prefill", "conv_decode", "scan", "scan_prefill", "scan_decode", "attention", "attention_prefill",
         "attention_decode")


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b)) and len(a) == len(b)


@pytest.mark.parametrize("name", NAMES)
def test_repeats_streams_and_graphs(name):
    call = _calls()[name]
    want = call()
    assert same(call(), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = call()
        call()
    here = call()                                              # two at once
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert same(there, want) and same(here, want)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = call()
        graphs.append((g, out))
    for i in range(3):
        for g, out in graphs:
            for x in out:
                x.fill_(1.0)
            g.replay()
        assert same(call(), want)
        torch.cuda.synchronize()
        for g, out in graphs:
            assert same(out, want), i


def test_graphs_of_the_largest_head_dimension():
    """128 dimensions take more LDS than a workgroup has by default, rows in parts a workspace."""
    g = gen(77)
    q, k, v, dy = (normal(g, 1, 700, n, 128, dtype=BF16) for n in (4, 2, 2, 4))
    ids = documents(g, 1, 700)
    cache = {n: normal(g, 1, 1500, 2, 128, dtype=BF16) for n in "kv"}
    lens = torch.tensor([650], device=DEV)

    def call():
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        y = cf.softmax_attention(*leaves, document_ids=ids)
        out = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
        for f, n in ((cf.softmax_attention_prefill, 700), (cf.softmax_attention_decode, 1)):
            y, c = f(q[:, :n], k[:, :n], v[:, :n], {n: t.clone() for n, t in cache.items()}, lens)
            out += [y, c["k"], c["v"]]
        return out

    want = call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(3):
        for x in out:
            x.fill_(1.0)
        graph.replay()
        assert same(call(), want)
        torch.cuda.synchronize()
        assert same(out, want), i


def test_differences():
    """Directional derivatives of the fp32 calls.  f is of order 1 per output and changes by e d1 +
    e^3 d3 / 6; with e = 2^-7 the rounding of f (2^-22 of the sum of its terms) over e and the
    third derivative leave less than 1e-2 of the gradient's length."""
    calls = {
        "conv": ([normal(gen(1), 1, 40, 16), normal(gen(2), 16, 4), normal(gen(3), 16)],
                 lambda *a: cf.short_convolution(*a, activation="silu")),
        "scan": (list(scan_inputs(gen(4), 1, 70, 24, 16, 1, F32).values()),
                 lambda *a: cf.state_space_scan(*a, dt_softplus=True)),
        "attention": ([normal(gen(i), 1, 70, 2, 32) for i in (5, 6, 7)],
                      lambda *a: cf.softmax_attention(*a, softcap=5.0)),
    }
    for name, (inputs, f) in calls.items():
        leaves = [t.clone().requires_grad_() for t in inputs]
        y = f(*leaves)
        dy = normal(gen(9), *y.shape)
        grads = torch.autograd.grad(y, leaves, dy)
        for i, (leaf, grad) in enumerate(zip(inputs, grads)):
            way = grad / grad.norm()
            e = 2.0 ** -7
            moved = [[t + s * e * way if j == i else t for j, t in enumerate(inputs)] for s in (1, -1)]
            with torch.no_grad():
                diff = float(((f(*moved[0]) - f(*moved[1])).double() * dy.double()).sum() / (2 * e))
            assert abs(diff - float(grad.norm())) <= 1e-2 * float(grad.norm()), (name, i, diff, float(grad.norm()))


# ---------------------------------------------------------------------------------------
# A stack of them with a FLARE layer, as they are used together
# ---------------------------------------------------------------------------------------
class Stack:
    """Convolution, scan, attention and FLARE over one width, with seeded weights."""

    def __init__(self, C=128, S=16, H=4, M=32):
        g = gen(31)
        self.C, self.S, self.H, self.D = C, S, H, C // H
        self.w = {"conv": normal(g, C, 4, std=0.5), "bias": normal(g, C, std=0.1),
                  "in": normal(g, C, 3 * C + 2 * S, std=C ** -0.5), "qkv": normal(g, C, 3 * C, std=C ** -0.5),
                  "A": -torch.arange(1, S + 1, device=DEV).float().expand(C, S).clone(), "D": normal(g, C),
                  "dt": normal(g, C) - 2, "latents": normal(g, H, M, C // H), "kv": normal(g, C, 2 * C, std=C ** -0.5)}

    def split(self, x):
        w, C, S = self.w, self.C, self.S
        x, dt, z, b, c = (x @ w["in"]).split((C, C, C, S, S), -1)
        return x, dt, w["A"], b, c, w["D"], z, w["dt"], True

    def heads(self, x, name, n):
        return (x @ self.w[name]).view(*x.shape[:-1], n, self.H, self.D).unbind(-3)

    def whole(self, x, ids=None):
        w = self.w
        x = x + cf.short_convolution(x, w["conv"], w["bias"], "silu", ids)
        x = x + cf.state_space_scan(*self.split(x), document_ids=ids)
        x = x + cf.softmax_attention(*self.heads(x, "qkv", 3), softcap=10.0, document_ids=ids).flatten(-2)
        if ids is None:
            x = x + cf.flare_autoregressive_triton(w["latents"], *self.heads(x, "kv", 2), scale=1.0).flatten(-2)
        return x

    def prefill(self, x, room):
        w, B = self.w, x.shape[0]
        y, s1 = cf.short_convolution_prefill(x, w["conv"], w["bias"], "silu")
        x = x + y
        y, s2 = cf.state_space_scan_prefill(*self.split(x))
        x = x + y
        cache = {n: torch.zeros((B, room, self.H, self.D), device=DEV) for n in "kv"}
        lengths = torch.zeros((B,), dtype=torch.int32, device=DEV)
        y, cache = cf.softmax_attention_prefill(*self.heads(x, "qkv", 3), cache, lengths, softcap=10.0)
        lengths += x.shape[1]
        x = x + y.flatten(-2)
        y, s3 = cf.flare_autoregressive_prefill_triton(w["latents"], *self.heads(x, "kv", 2))
        return x + y.flatten(-2), [s1, s2, cache, lengths, s3]

    def decode(self, x, states):
        w = self.w
        s1, s2, cache, lengths, s3 = states
        x = x[:, None]
        x = x + cf.short_convolution_decode(x, w["conv"], w["bias"], "silu", s1)[0]
        x = x + cf.state_space_scan_decode(*self.split(x), state=s2)[0]
        x = x + cf.softmax_attention_decode(*self.heads(x, "qkv", 3), cache, lengths, softcap=10.0)[0].flatten(-2)
        lengths += 1
        return x + cf.flare_autoregressive_decode_triton(w["latents"], *self.heads(x, "kv", 2), state=s3)[0].flatten(-2)


def test_stack_prefill_and_decode_continue_each_other():
    """The same tokens whole, and as a prompt with single tokens behind it: fp32 sums in another order.

    What that may move an output by: a FLARE score s, rounded a few times at 2^-24 |s|, moves the
    weights by that part of themselves, and y by it times the values, twice (numerator and sum).
    These weights give scores of up to 290 and values of up to 46: with four roundings 2 * 4 *
    2^-24 * 290 * 46 = 6.4e-3, beside which the other layers' 1e-5 do not count.  (Half a step of
    fp32 on the inputs alone moves the outputs by 8e-4.)"""
    stack, x = Stack(), normal(gen(32), 2, 90, 128)
    near = functools.partial(torch.allclose, rtol=1e-5, atol=8 * E32 * 290 * 46)
    with torch.no_grad():
        want = stack.whole(x)
        y, states = stack.prefill(x[:, :77], 90)
        assert near(y, want[:, :77])
        for t in range(77, 90):
            y = stack.decode(x[:, t], states)
            assert near(y[:, 0], want[:, t]), t


def test_stack_of_packed_documents_trains_as_each_alone():
    stack, x = Stack(), normal(gen(33), 1, 150, 128)
    cuts = [0, 33, 100, 150]
    ids = torch.zeros((1, 150), dtype=torch.int32, device=DEV)
    for i in range(3):
        ids[:, cuts[i]:cuts[i + 1]] = i
    names = ("conv", "bias", "in", "qkv", "D")
    for n in names:
        stack.w[n].requires_grad_()
    dy = normal(gen(34), 1, 150, 128)
    a = x.clone().requires_grad_()
    y = stack.whole(a, ids)
    packed = torch.autograd.grad(y, [a] + [stack.w[n] for n in names], dy)
    total = None
    for i in range(3):
        s = slice(cuts[i], cuts[i + 1])
        one = x[:, s].clone().requires_grad_()
        yi = stack.whole(one, torch.zeros((1, cuts[i + 1] - cuts[i]), dtype=torch.int32, device=DEV))
        assert torch.allclose(yi, y[:, s], rtol=1e-4, atol=1e-4)
        gi = torch.autograd.grad(yi, [one] + [stack.w[n] for n in names], dy[:, s])
        assert torch.allclose(gi[0], packed[0][:, s], rtol=1e-3, atol=1e-3)
        total = list(gi[1:]) if total is None else [u + v for u, v in zip(total, gi[1:])]
    for n, u, v in zip(names, total, packed[1:]):
        assert torch.allclose(u, v, rtol=1e-3, atol=1e-3 * float(v.abs().max())), n


def test_a_cache_of_more_than_32_bits_of_elements():
    """2^31 + 2^25 keys' elements: all keys 0 but the last few, so that weights are 1 / n or known."""
    G, D = 16, 128
    S = (2 ** 31 + 2 ** 25) // (G * D)
    cache = {n: torch.zeros((1, S, G, D), dtype=BF16, device=DEV) for n in "kv"}
    n = S - 3
    cache["v"][0, n - 1] = 1.0
    q = torch.zeros((1, 1, G, D), dtype=BF16, device=DEV)
    q[..., 0] = 16.0
    cache["k"][0, n - 1, :, 0] = 16.0                       # a score of 256 / sqrt(128) = 22.6
    new = torch.zeros((1, 1, G, D), dtype=BF16, device=DEV)
    lengths = torch.tensor([n], device=DEV)
    y, _ = cf.softmax_attention_decode(q, new, new, cache, lengths)
    want = 1 / (1 + n * math.exp(-256 / math.sqrt(128)))
    assert torch.allclose(y.float(), torch.full_like(y.float(), want), rtol=2 ** -7)
    y2, _ = cf.softmax_attention_prefill(q.expand(1, 2, G, D), new.expand(1, 2, G, D), new.expand(1, 2, G, D) + 3, cache, lengths)
    assert torch.allclose(y2.float(), torch.full_like(y2.float(), want), rtol=2 ** -7)
    assert (cache["v"][0, n:n + 2] == 3.0).all() and not cache["v"][0, n + 2:].any()
