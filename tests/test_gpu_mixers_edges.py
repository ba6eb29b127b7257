"""The token mixers on the GPU where a formula meets its edges: infinite values that a cap or a mask
bounds, growth past fp32, gradients below a type's range, chunks of other lengths."""
import math
import random

import pytest
import torch

import causal_flare as cf
from causal_flare import _lib
from _mixers import U, attention, check, scan
import test_gpu_mixers as mixers
from test_gpu_mixers import (BF16, DEV, E32, F16, F32, close, close_attention, documents, gen, normal, same,
                             scan_inputs)

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan
ORDER = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")


# ---------------------------------------------------------------------------------------
# Softmax attention
# ---------------------------------------------------------------------------------------
def seen_sums(see, w, x):
    """sum_j w_ij x_jd over the pairs of `see` alone: what is not seen may be infinite."""
    return torch.where(see[..., None], w[..., None] * x[None], 0.0).sum(1)


def one_head(q, k, v, dy, see, cap, unit, slope=0.0):
    """{name: (value, tolerance)} of one head [N, D] with every sum over the seen pairs alone; the
    tolerances are those of `attention` in _mixers.py, a saturated score's own error being 0."""
    N, D = q.shape
    scale = D ** -0.5
    far = slope * (torch.arange(N)[:, None] - torch.arange(N)[None]).abs()
    some = see.any(1, keepdim=True)
    x = q @ k.t() * scale
    th = torch.tanh(x / cap) if cap else torch.zeros_like(x)
    s = torch.where(see, (cap * th if cap else x) - far, -INF)
    p = torch.where(some, torch.softmax(s, 1), 0.0)
    sums = lambda w, t: seen_sums(see, w, t)
    y, pv = sums(p, v), sums(p, v.abs())
    dp = dy @ v.t()
    delta = torch.where(some, (dy * y).sum(1, keepdim=True), 0.0)
    cut = 1 - th * th
    ds = p * (dp - delta) * cut * scale
    out = {"y": y, "dq": sums(ds, k), "dk": seen_sums(see.t(), ds.t(), q), "dv": seen_sums(see.t(), p.t(), dy)}
    size = (q.abs() @ k.abs().t() * scale).nan_to_num(0.0, 0.0, 0.0) + far
    es = E32 * (torch.where(see, size, 0.0).amax(1, keepdim=True) * (8 + D / 4) + 16 + 8 * (cap or 0.0))
    ey = (2 * unit + 2 * es + 64 * E32) * pv + unit * y.abs()
    edp = E32 * (16 + D) * (dy.abs() @ v.abs().t()) + (dy.abs() * ey).sum(1, keepdim=True)
    eds = (p * cut * edp + (2 * es + 64 * E32) * p * (dp - delta).abs() * (cut + 4) + unit * ds.abs() / scale
           + 2.0 ** -25 * (1 + (dp - delta).abs())) * scale
    tol = {"y": (unit + 2 * es + 64 * E32) * pv + 2.0 ** -25 * seen_sums(see, torch.ones_like(p), v.abs()),
           "dq": sums(eds + 64 * E32 * ds.abs(), k.abs()),
           "dk": seen_sums(see.t(), (eds + 64 * E32 * ds.abs()).t(), q.abs()),
           "dv": seen_sums(see.t(), ((unit + 2 * es + 64 * E32) * p + 2.0 ** -25).t(), dy.abs())}
    return {n: (out[n], tol[n]) for n in out}


def check_finite_part(got, ref, what, dtype):
    """The same entries are finite, and those are near."""
    value, tol = ref
    have, want = got.isfinite().cpu(), value.isfinite()
    assert torch.equal(have, want), (what, (have != want).nonzero()[:5].tolist())
    tol = tol.nan_to_num(0.0, 0.0, 0.0)
    check(torch.where(have.to(got.device), got.float(), 0.0).to(got.dtype), torch.where(want, value, 0.0),
          U[dtype] * (value.nan_to_num(0.0, 0.0, 0.0).abs() + tol) + tol, what, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("where", ["q", "k", "q and dy"])
@pytest.mark.parametrize("cap, D, docs, sloped", [
    (3.0, 64, True, False), (3.0, 128, False, True), (50.0, 48, True, False), (2.0, 32, False, False)])
def test_a_cap_bounds_infinite_scores(dtype, where, cap, D, docs, sloped):
    """An infinite element of a query or key makes scores of +-cap: weights, y and dv are finite, and only
    the gradients that multiply a score gradient of 0 by that element are none."""
    g = gen(D)
    N, at = 150, 70
    q, k, v, dy = (normal(g, 1, N, 2, D, dtype=dtype) for _ in range(4))
    (q if "q" in where else k)[0, at, 0, 5] = INF
    if "dy" in where:
        dy[0, at + 3, 0, 7] = -INF
    ids = torch.zeros((1, N), dtype=torch.int32, device=DEV)
    ids[:, 100:] = 1
    slopes = torch.tensor([0.25, 0.5], device=DEV) if sloped else None
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    y = cf.softmax_attention(*leaves, softcap=cap, document_ids=ids if docs else None, slopes=slopes)
    grads = torch.autograd.grad(y, leaves, dy)
    see = torch.ones((N, N), dtype=torch.bool).tril()
    if docs:
        see &= ids[0].cpu()[:, None] == ids[0].cpu()[None]
    for h in range(2):
        ref = one_head(*(t[0, :, h].double().cpu() for t in (q, k, v, dy)), see, cap, 0.0 if dtype is F32 else U[dtype],
                       float(slopes[h]) if sloped else 0.0)
        for n, got in zip(("y", "dq", "dk", "dv"), (y, *grads)):
            check_finite_part(got[0, :, h].detach(), ref[n], f"{n} of head {h}", dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [16, 32, 48, 80, 128])
@pytest.mark.parametrize("what", ["docs", "cap docs", "cap docs prefix slopes", "full docs slopes"])
def test_attention_of_every_width_with_documents(dtype, D, what):
    mixers.test_attention(dtype, 2, 150, 4, 2, D, what)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("N", [130, 1700])
def test_a_row_of_scores_that_are_all_minus_infinity_is_nan(dtype, N):
    """It sees keys, so it is no row of 0; rows and keys apart from it stay as they are.  1700 rows run in
    parts of the keys."""
    g = gen(N)
    H, D, at = 2, 64, 67
    q, k, v, dy = (normal(g, 1, N, H, D, dtype=dtype) for _ in range(4))
    k[0, :, 0, 0] = -1.0
    bad = q.clone()
    bad[0, at, 0, 0] = INF
    outs = []
    for x in (q, bad):
        leaves = [x.clone().requires_grad_(), k.clone().requires_grad_(), v.clone().requires_grad_()]
        y = cf.softmax_attention(*leaves)
        outs.append([y.detach(), *torch.autograd.grad(y, leaves, dy)])
    rest = [i for i in range(N) if i != at]
    assert outs[1][0][0, at, 0].isnan().all() and outs[1][1][0, at, 0].isnan().all()
    for i in (0, 1):
        assert torch.equal(outs[0][i][:, rest], outs[1][i][:, rest])
    for i in (2, 3):
        assert torch.equal(outs[0][i][:, at + 1:], outs[1][i][:, at + 1:])
        assert torch.equal(outs[0][i][:, :, 1], outs[1][i][:, :, 1])
        assert outs[1][i][0, :at + 1, 0].isnan().all()
    cache = {"k": k.clone(), "v": v.clone()}
    held = torch.tensor([at], device=DEV)
    new = [t[:, at:at + 4] for t in (bad, k, v)]
    y, _ = cf.softmax_attention_prefill(*new, cache, held, new_lengths=torch.tensor([2], device=DEV))
    assert y[0, 0, 0].isnan().all() and y[0, 1].isfinite().all() and not y[0, 2:].any()
    y, _ = cf.softmax_attention_decode(*(t[:, 0] for t in new), cache, held)
    assert y[0, 0, 0].isnan().all() and y[0, 0, 1].isfinite().all()


@pytest.mark.parametrize("cap, std", [(30.0, 1e-12), (30.4, 1e-14), (41.0, 1e-9), (50.0, 1e-12)])
def test_small_values_beside_scores_at_the_lower_end_of_a_cap(cap, std):
    """Rows whose scores are all -cap: their weights are of any size until the sum divides them.  y is off
    by the rounding of a weight and its own (bf16)."""
    g = gen(1)
    N, D = 200, 64
    q = torch.full((1, N, 1, D), 4.0, dtype=BF16, device=DEV)
    k = (torch.rand((1, N, 1, D), generator=g) * -100 - 100).to(BF16).to(DEV)
    v = normal(g, 1, N, 1, D, dtype=BF16, std=std)
    y = cf.softmax_attention(q, k, v, softcap=cap)
    p = torch.ones((N, N), dtype=torch.float64).tril()
    p /= p.sum(1, keepdim=True)
    v = v[0, :, 0].double().cpu()
    check(y[0, :, 0], p @ v, U[BF16] * (p @ v).abs() + 1.01 * U[BF16] * (p @ v.abs()), "y", BF16)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cap", [300.0, 1e4, 1e6, 1e8, 1e20])
@pytest.mark.parametrize("sloped", [False, True])
def test_large_caps_leave_small_scores_their_digits(dtype, cap, sloped):
    """A score far below the cap is nearly itself, so its error is that of a score without a cap
    (the tolerance of the call without one), however large the cap."""
    g = gen(41)
    N, H, D = 150, 2, 64
    q, k, v, dy = (normal(g, 1, N, H, D, dtype=dtype, std=s) for s in (2.0, 1.0, 1.0, 1.0))
    o = {"slopes": torch.tensor([0.125, 0.5], device=DEV)} if sloped else {}
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    y = cf.softmax_attention(*leaves, softcap=cap, **o)
    grads = torch.autograd.grad(y, leaves, dy)
    unit = 0.0 if dtype is F32 else U[dtype]
    tiny = 2.0 ** -25 if dtype is F16 else 2.0 ** -126
    ref, loose = (attention(q, k, v, softcap=c, dy=dy, unit=unit, tiny=tiny, **o) for c in (cap, None))
    for n, got in zip(("y", "dq", "dk", "dv"), (y, *grads)):
        close_attention(got, (ref[n][0], loose[n][1]), n, dtype)
    at = N - 1
    cache = {n: torch.cat((t[:, :at], torch.zeros_like(t)), 1) for n, t in (("k", k), ("v", v))}
    held = torch.tensor([at], device=DEV, dtype=torch.int32)
    step, _ = cf.softmax_attention_decode(q[:, at], k[:, at], v[:, at], cache, held, softcap=cap, **o)
    close_attention(step, (ref["y"][0][:, at:], loose["y"][1][:, at:]), "token", dtype)
    held -= 40
    y, _ = cf.softmax_attention_prefill(q[:, at - 40:], k[:, at - 40:], v[:, at - 40:], cache, held, softcap=cap, **o)
    close_attention(y, (ref["y"][0][:, at - 40:], loose["y"][1][:, at - 40:]), "prompt", dtype)


@pytest.mark.parametrize("std", [1e3, 1e-2, 1e-4, 1e-5])
@pytest.mark.parametrize("N, H, G, D, what", [(1025, 4, 2, 64, ""), (300, 2, 1, 128, "cap"), (700, 2, 2, 48, "docs"),
                                              (2100, 1, 1, 32, "")])
def test_small_and_large_gradients_of_fp16(std, N, H, G, D, what):
    """Score gradients of fp16 inputs keep their digits far below fp16's smallest numbers.  What rounding
    one may cost absolutely is half a step of 2^-24 where the largest that dy and v allow (2 |dy|_1 max|v|,
    a bound of |dP| + |delta|) lies at 2^14 or above: 2^-39 of that bound."""
    g = gen(N)
    q, k, v = (normal(g, 1, N, n, D, dtype=F16) for n in (H, G, G))
    dy = normal(g, 1, N, H, D, std=std).to(F16)
    o = {"softcap": 5.0} if what == "cap" else {}
    groups = [slice(0, N)]
    if what == "docs":
        # documents of very different gradients, and padding that holds large numbers
        ids = torch.zeros((1, N), dtype=torch.int32, device=DEV)
        ids[:, 200:], ids[:, 500:] = 1, -1
        groups, o["document_ids"] = [slice(0, 200), slice(200, 500)], ids
        dy[:, 200:500] *= 2.0 ** -6
        dy[:, 500:], v[:, 500:] = 6e4, 6e4
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(cf.softmax_attention(*leaves, **o), leaves, dy)
    real = slice(0, groups[-1].stop)
    bound = 2 * float(dy[:, real].double().abs().sum(-1).max()) * float(v[:, real].double().abs().max())
    for s in groups:
        part = [t[:, s] for t in (q, k, v)]
        ref = attention(*part, softcap=o.get("softcap"), dy=dy[:, s], unit=U[F16], tiny=2.0 ** -39 * bound)
        for n, got in zip(("dq", "dk"), grads):
            close_attention(got[:, s], ref[n], n, F16)
    if what == "docs":
        assert all(not t[:, 500:].any() for t in grads)


def test_fp16_training_steps_in_graphs():
    """The scales of fp16 score gradients are taken anew at every replay."""
    g = gen(51)
    q, k, v, dy = (normal(g, 2, 300, n, 64, dtype=F16) for n in (4, 2, 2, 4))
    ids = documents(g, 2, 300)

    def call():
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        y = cf.softmax_attention(*leaves, softcap=20.0, document_ids=ids)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        dy.copy_(normal(g, 2, 300, 4, 64, std=10.0 ** -i).to(F16))
        v.mul_(0.5)
        for x in out:
            x.fill_(1.0)
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert same(out, want), i


def test_decode_of_many_sequences_and_heads():
    """More rows of keys than a grid's second dimension takes: each as in a call of its own."""
    g = gen(9)
    B, H, G, D, S = 9000, 16, 8, 16, 3
    q, k, v = (normal(g, B, n, D, dtype=BF16) for n in (H, G, G))
    cache = {n: normal(g, B, S, G, D, dtype=BF16) for n in "kv"}
    held = torch.arange(B, device=DEV, dtype=torch.int32) % 5 - 1          # idle, 0, 1, 2 and full
    parts = []
    for s in (slice(0, 4500), slice(4500, B)):
        part = {n: t[s].clone() for n, t in cache.items()}
        parts.append([cf.softmax_attention_decode(q[s], k[s], v[s], part, held[s])[0], part["k"], part["v"]])
    y, _ = cf.softmax_attention_decode(q, k, v, cache, held)
    for got, want in zip((y, cache["k"], cache["v"]), zip(*parts)):
        assert torch.equal(got.nan_to_num(9.0), torch.cat(want).nan_to_num(9.0))
    assert y[4::5].isnan().all() and not y[0::5].any()


@pytest.mark.parametrize("seed", range(12))
def test_infinite_values_reach_what_the_formula_gives_them_to(seed):
    """Which entries of y and of the gradients are finite, with infinite values and NaNs anywhere."""
    for case in range(20):
        rng, g = random.Random(100 * seed + case), gen(100 * seed + case)
        dtype, D = rng.choice([F32, BF16, F16]), rng.choice([16, 32, 48, 64, 80, 96, 112, 128])
        N = rng.choice([3, 17, 40, 64, 65, 100, 129, 150, 200, 260, 700])
        t = {n: normal(g, 1, N, 1, D, dtype=dtype) for n in "qkvd"}
        o, see = {}, torch.ones((N, N), dtype=torch.bool)
        if rng.random() < 0.8:
            see = see.tril()
            if rng.random() < 0.3:
                o["prefix_lengths"] = torch.tensor([rng.randrange(N + 1)], device=DEV)
                see |= torch.arange(N)[None] < int(o["prefix_lengths"])
        else:
            o["causal"] = False
        if rng.random() < 0.5:
            o["document_ids"] = documents(g, 1, N)
            ids = o["document_ids"][0].cpu()
            see &= (ids[:, None] == ids[None]) & (ids[:, None] >= 0)
        cap = rng.choice([None, None, 3.0, 20.0, 40.0, 400.0])
        if cap:
            o["softcap"] = cap
        slope = rng.choice([0.0, 0.25, -0.01])
        if slope:
            o["slopes"] = torch.tensor([slope], device=DEV)
        holes = [(rng.choice("qkvd"), rng.randrange(N), rng.randrange(D), rng.choice([INF, -INF, NAN]))
                 for _ in range(rng.randrange(4))]
        for n, i, d, x in holes:
            t[n][0, i, 0, d] = x
        leaves = [t[n].clone().requires_grad_() for n in "qkv"]
        y = cf.softmax_attention(*leaves, **o)
        grads = torch.autograd.grad(y, leaves, t["d"])
        ref = one_head(*(t[n][0, :, 0].double().cpu() for n in "qkvd"), see, cap, 0.0, slope)
        for n, got in zip(("y", "dq", "dk", "dv"), (y, *grads)):
            have, want = got[0, :, 0].isfinite().cpu(), ref[n][0].isfinite()
            off = (have != want).nonzero()[:3].tolist()
            assert not off, (n, dtype, N, D, list(o), cap, slope, holes, off)


def test_lengths_that_are_no_tensor_are_refused():
    qkv, cache = [normal(gen(0), 2, 1, 4, 32) for _ in range(3)], {n: normal(gen(1), 2, 9, 4, 32) for n in "kv"}
    for call in (cf.softmax_attention_prefill, cf.softmax_attention_decode):
        with pytest.raises(ValueError, match="expects a tensor in lengths"):
            call(*qkv, cache, None)


@pytest.mark.parametrize("N", [2048, 2081, 2600])
def test_attention_of_a_round_of_workgroups(N):
    """Sizes at which rows of 16 heads take two parts, and above them: against 64 bits on the GPU.  A
    score is a product over D (8 + D / 4 roundings of its terms' sizes), an exponential and the sums some
    64 more, as in `attention` of _mixers.py."""
    g = gen(N)
    H, D = 16, 32
    q, k, v = (normal(g, 1, N, H, D) for _ in range(3))
    y = cf.softmax_attention(q, k, v)
    see = torch.ones((N, N), dtype=torch.bool, device=DEV).tril()
    for h in (0, 7, 15):
        a, b, c = (t[0, :, h].double() for t in (q, k, v))
        p = torch.softmax(torch.where(see, (a @ b.t()) * D ** -0.5, -INF), 1)
        size = torch.where(see, (a.abs() @ b.abs().t()) * D ** -0.5, 0.0).amax(1, keepdim=True)
        tol = E32 * (2 * (size * (8 + D / 4) + 16) + 64) * (p @ c.abs())
        check(y[0, :, h], (p @ c).cpu(), (tol + E32 * (p @ c).abs()).cpu(), f"y of head {h}")


@pytest.mark.parametrize("N", [300, 1500])
def test_fp16_gradients_where_few_keys_hold_large_values(N):
    """Rows that divide their weight between a key of large values and one of small ones far behind it,
    which of 1500 rows other workgroups take: dy . y is as large as the former."""
    g = gen(N)
    D, far = 64, N - 100
    q, k, v, dy = (torch.zeros((1, N, 1, D), dtype=F16, device=DEV) for _ in range(4))
    q[..., :8], k[0, 10, 0, :8], k[0, far, 0, :8] = 4.0, 8.0, 8.0          # scores of 32 and of 0
    v[:] = normal(g, 1, N, 1, D, dtype=F16)
    v[0, 10] = 1000.0
    dy[:] = normal(g, 1, N, 1, D).abs().to(F16)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(cf.softmax_attention(*leaves), leaves, dy)
    bound = 2 * float(dy.double().abs().sum(-1).max()) * float(v.double().abs().max())
    ref = attention(q, k, v, dy=dy, unit=U[F16], tiny=2.0 ** -39 * bound)
    # (dk of key 10 is past fp16's largest number: 100 rows of dS = 1/4 1000 |dy|_1 scale, times q = 4)
    for n, got in zip(("dq", "dk"), grads):
        close_attention(got, ref[n], n, F16)


# ---------------------------------------------------------------------------------------
# State space scan
# ---------------------------------------------------------------------------------------
class WithChunk:
    """The library with chunks of a given length for the scan."""

    def __init__(self, lib, chunk):
        self._lib, self.flare_scan_chunk = lib, lambda *sizes: chunk

    def __getattr__(self, name):
        return getattr(self._lib, name)


@pytest.fixture
def chunks(monkeypatch):
    lib = _lib.lib()
    return lambda n: monkeypatch.setattr(_lib, "lib", lambda: WithChunk(lib, n))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("chunk", [32, 128])
@pytest.mark.parametrize("where", ["dy", "x", "z"])
@pytest.mark.parametrize("C, S", [(48, 16), (70, 8), (20, 40)])
@pytest.mark.parametrize("poison", [INF, NAN])
def test_scan_keeps_documents_apart_whatever_one_holds(dtype, chunk, where, C, S, poison, chunks):
    """A document's infinite values and gradients stay its own: in it, before it and behind it, at
    borders within a piece of four tokens, within a stretch and where a chunk ends."""
    chunks(chunk)
    g = gen(C)
    N = 200
    t = scan_inputs(g, 1, N, C, S, 1, dtype)
    dy = normal(g, 1, N, C, dtype=dtype)
    ids = torch.zeros((1, N), dtype=torch.int32, device=DEV)
    for i, cut in enumerate((29, 46, 64, 131, 160)):
        ids[:, cut:] = i + 1
    outs = []
    for bad in (False, True):
        s, d = {n: x.clone() for n, x in t.items()}, dy.clone()
        if bad:
            for row in (40, 130):                                 # documents 1 and 3
                (d if where == "dy" else s[where])[0, row, C - 1] = poison
        leaves = [s[n].requires_grad_() for n in ORDER]
        y = cf.state_space_scan(*leaves, dt_softplus=True, document_ids=ids)
        grads = torch.autograd.grad(y, leaves, d)
        outs.append([y.detach()] + [grads[ORDER.index(n)] for n in ("x", "dt", "B", "C", "z")])
    apart = ((ids[0] != 1) & (ids[0] != 3)).cpu()
    for name, a, b in zip(("y", "dx", "ddt", "dB", "dC", "dz"), *outs):
        assert torch.equal(a[:, apart], b[:, apart]), name
    assert not outs[1][1 if where == "dy" else 0].isfinite().all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("chunk", [32, 128])
def test_scan_of_zero_states_and_gradients_under_any_growth(dtype, chunk, chunks):
    """States grow by 2^9 a token, 2^288 and more over a chunk: one of 0 stays 0 as it does token by
    token, and so does the gradient that enters from behind."""
    chunks(chunk)
    g = gen(3)
    N, C, S = 400, 20, 16
    z = torch.zeros((1, N, C), dtype=dtype, device=DEV)
    t = {"x": z.clone(), "dt": z + 1, "A": torch.full((C, S), 9 * math.log(2.0), device=DEV),
         "B": normal(g, 1, N, 1, S, dtype=dtype), "C": normal(g, 1, N, 1, S, dtype=dtype), "D": normal(g, C),
         "z": normal(g, 1, N, C, dtype=dtype), "dt_bias": None}
    dy = z.clone()
    t["x"][:, -6:], dy[:, :6] = normal(g, 1, 6, C, dtype=dtype), normal(g, 1, 6, C, dtype=dtype)
    names = [n for n in ORDER if t[n] is not None]
    leaves = {n: t[n].clone().requires_grad_() for n in names}
    y = cf.state_space_scan(*[leaves.get(n) for n in ORDER])
    grads = torch.autograd.grad(y, [leaves[n] for n in names], dy)
    ref = scan(**t, dy=dy)
    assert y.isfinite().all() and all(x.isfinite().all() for x in grads)
    close(y, ref["y"], "y", dtype, ref["k"])
    for n, got in zip(names, grads):
        close(got, ref["d" + n], "d" + n, F32 if n in "AD" else dtype, 2 * ref["k"] + C)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("chunk, B, N, C, S, G, docs, more", [
    (128, 2, 300, 70, 16, 1, True, True), (128, 1, 257, 48, 4, 1, False, False), (96, 1, 200, 130, 16, 2, False, True),
    (64, 2, 131, 20, 33, 1, True, True), (128, 1, 260, 24, 64, 1, False, True), (128, 1, 250, 32, 24, 2, True, True),
    (120, 1, 250, 32, 40, 1, True, True)])
def test_scan_in_longer_chunks(chunk, dtype, B, N, C, S, G, docs, more, chunks):
    """The chunks of large calls on small ones: several kept stretches a chunk, forward chunks of more than
    8 tokens."""
    chunks(chunk)
    mixers.test_scan(dtype, B, N, C, S, G, docs, more)


@pytest.mark.parametrize("dtype, B, N, C, S, G", [
    (F16, 4, 1, 16, 16, 1), (F16, 5, 33, 70, 16, 2), (F16, 4, 90, 64, 20, 1)])
def test_scan_prefill_and_decode_of_fp16(dtype, B, N, C, S, G):
    mixers.test_scan_prefill_and_decode(dtype, B, N, C, S, G)


@pytest.mark.parametrize("chunk, dtype, B, N, C, S, G", [
    (13, F32, 3, 260, 40, 8, 1), (128, BF16, 3, 260, 40, 8, 1), (128, F16, 4, 300, 64, 20, 1),
    (64, F32, 3, 65, 16, 64, 1),
    (1 << 32, BF16, 3, 65, 16, 16, 1), ((1 << 63) - 1, F16, 3, 65, 16, 16, 1)])
def test_scan_prefill_in_other_chunks(chunk, dtype, B, N, C, S, G, chunks):
    chunks(chunk)
    mixers.test_scan_prefill_and_decode(dtype, B, N, C, S, G)
