"""Rotary positions against their plain 64-bit form."""
import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import _mixers as M
import _quantized as Q
import causal_flare as cf

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def rng(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, dtype=torch.float64).to(dtype)


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def near(got, x, frequencies, at, interleaved, what, inverse=False):
    ref, mag = Q.rotary(x, frequencies, at, interleaved, inverse)
    # sine and cosine: 2e-9 from their series, 2^-33 of a turn and three roundings; then two products and a sum.
    # (The plain form's angles lose the position's digits: 2^-53 of it, times a frequency below 1.)
    tol = mag * (7 * 2.0 ** -24 + 4e-9) + M.U[got.dtype] * ref.abs() + mag * 2.0 ** -51 * at.abs().max()
    M.check(got, ref, tol, what, got.dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H, G, D, R", [(4, 2, 64, 64), (16, 4, 128, 128), (3, 1, 128, 64), (2, 2, 80, 32), (2, 1, 48, 24), (1, 1, 32, 6),
                                        (5, 1, 36, 2), (2, 2, 33, 32), (1, 1, 256, 256), (7, 3, 96, 40), (1, 1, 2, 2), (40, 8, 64, 64)])
def test_turns_and_gradients(dtype, interleaved, H, G, D, R):
    dt, g = TYPES[dtype], rng(D + R)
    f = cf.rotary_frequencies(R)
    for B, N in ((1, 1), (2, 37), (3, 130)):
        q, k = normal(g, B, N, H, D, dtype=dt).cuda().requires_grad_(), normal(g, B, N, G, D, dtype=dt).cuda().requires_grad_()
        at = torch.arange(N).expand(B, N)
        for how in ({}, {"lengths": torch.randint(0, 9000, (B,), generator=g)}, {"positions": torch.randint(-70, 2 ** 17, (B, N), generator=g)}):
            if "lengths" in how:
                at = how["lengths"][:, None] + torch.arange(N)
            if "positions" in how:
                at = how["positions"]
            out = cf.rotary_positions(q, k, f, interleaved=interleaved, **{n: t.cuda() for n, t in how.items()})
            dy = [normal(g, *t.shape, dtype=dt).cuda() for t in out]
            grads = torch.autograd.grad(out, (q, k), dy)
            for y, x, dx, d, n in zip(out, (q, k), grads, dy, "qk"):
                assert y.dtype is dt and y.is_contiguous()
                near(y, x, f, at, interleaved, n)
                near(dx, d, f, at, interleaved, "d" + n, inverse=True)


def test_far_positions_and_any_frequency():
    g = rng(2)
    # of 2^31 tokens, forwards and back, by lengths and by positions; frequencies of more than a turn, negative ones and 0
    f = torch.tensor([1.0, 0.3, 1e-4, 0.0, -0.7, 6.5, 100.25, 3.0], dtype=torch.float64)
    x = normal(g, 1, 5, 2, 16).cuda()
    at = torch.tensor([[2 ** 31 - 1, -2 ** 31, 2 ** 30 + 12345, -1, 0]], dtype=torch.int64)
    y = cf.rotary_positions(x, None, f, positions=at.cuda())
    # turns in whole numbers: a frequency's turns a token to 2^-64, a position exactly
    from fractions import Fraction
    two_pi = Fraction(884279719003555, 140737488355328) + Fraction(2.449293598294706e-16)        # 2 pi to 106 bits
    angle = torch.empty(5, 8, dtype=torch.float64)
    for t in range(5):
        for i in range(8):
            turns = Fraction(float(f[i])) / two_pi * int(at[0, t])
            angle[t, i] = float((turns - round(turns)) * two_pi)
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = x[0].double().cpu()[..., :8], x[0].double().cpu()[..., 8:]
    ref = torch.cat((a * c - b * s, a * s + b * c), -1)[None]
    # 2^31 positions times 2^-64 turns and the rounding of turns to 64 bits (long double) on the host
    M.check(y, ref, (a.abs() + b.abs()).repeat(1, 1, 2)[None] * (8 * 2.0 ** -24 + 1e-8) + 2.0 ** -24 * ref.abs(), "y")
    z = cf.rotary_positions(x[:, :1], None, f, lengths=ints(2 ** 31 - 1))
    assert torch.equal(z, y[:, :1])
    # lengths[b] + t does not wrap
    far = cf.rotary_positions(x, None, f[:1], lengths=ints(2 ** 31 - 3))
    ref, mag = Q.rotary(x, f[:1], torch.arange(5)[None] + (2 ** 31 - 3))
    M.check(far, ref, mag * (8 * 2.0 ** -24 + 4e-9 + 2.0 ** 31 * 2.0 ** -53) + 2.0 ** -24 * ref.abs(), "y")


def test_scaled_frequencies():
    f = cf.rotary_frequencies(64, base=500000.0)
    assert f.dtype is torch.float64 and f.device.type == "cpu" and f.shape == (32,)
    assert torch.allclose(f, 500000.0 ** (-torch.arange(32, dtype=torch.float64) / 32), rtol=1e-14)
    assert torch.equal(cf.rotary_frequencies(64, factor=4.0), cf.rotary_frequencies(64) / 4)
    parts = cf.rotary_frequencies(64, factor=8.0, original_length=4096, low_turns=1.0, high_turns=4.0)
    turns = 4096 * cf.rotary_frequencies(64) / 6.283185307179586
    assert torch.equal(parts[turns >= 4], cf.rotary_frequencies(64)[turns >= 4])
    assert torch.allclose(parts[turns <= 1], cf.rotary_frequencies(64)[turns <= 1] / 8, rtol=1e-14)
    assert ((parts[1:] <= parts[:-1])).all()


def test_strides_types_and_missing_parts():
    g = rng(4)
    f = cf.rotary_frequencies(64)
    fused = normal(g, 2, 9, 12, 64, dtype=torch.bfloat16).cuda()
    q, k = fused[:, :, :8], fused[:, :, 8:]
    a, b = cf.rotary_positions(q, k, f), cf.rotary_positions(q.contiguous(), k.contiguous(), f)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # heads before tokens, dimensions that are not adjacent, rows that are not aligned, broadcast heads
    moved = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    apart = q.transpose(2, 3).contiguous().transpose(2, 3)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape).copy_(q)
    for t in (moved, apart, odd):
        assert torch.equal(cf.rotary_positions(t, None, f), a[0])
    one = q[:, :, :1].expand(-1, -1, 8, -1)
    assert torch.equal(cf.rotary_positions(one, k, f)[0], cf.rotary_positions(one.contiguous(), k, f)[0])
    # gradients of a broadcast head add up, and of one tensor alone
    leaf = normal(g, 2, 9, 1, 64).cuda().requires_grad_()
    dy = normal(g, 2, 9, 8, 64).cuda()
    dx, = torch.autograd.grad(cf.rotary_positions(leaf.expand(-1, -1, 8, -1), k.float(), f)[0], leaf, dy)
    ref = Q.rotary(dy, f, torch.arange(9).expand(2, 9), inverse=True)[0].sum(2, keepdim=True)
    M.check(dx, ref, 16 * 2.0 ** -24 * Q.rotary(dy, f, torch.arange(9).expand(2, 9), inverse=True)[1].sum(2, keepdim=True), "dx")
    kk = normal(g, 2, 9, 4, 64).cuda().requires_grad_()
    out = cf.rotary_positions(q.float(), kk, f)
    assert not out[0].grad_fn is None and torch.autograd.grad(out[1].sum(), kk)[0].shape == kk.shape
    # one of two outputs used, and a gradient that is an expanded scalar
    both = [normal(g, 2, 9, h, 64).cuda().requires_grad_() for h in (8, 4)]
    y = cf.rotary_positions(*both, f)
    dq, dk = torch.autograd.grad(y[0].sum(), both)
    assert (dk == 0).all() and torch.isfinite(dq).all()
    # two types: each comes back as it went in
    y = cf.rotary_positions(q, kk.detach(), f)
    assert y[0].dtype is torch.bfloat16 and y[1].dtype is torch.float32
    near(y[0], q, f, torch.arange(9).expand(2, 9), False, "q")
    near(y[1], kk, f, torch.arange(9).expand(2, 9), False, "k")
    wide = cf.rotary_positions(q.double(), None, f)
    assert wide.dtype is torch.float64
    # single tokens without their dimension, nothing at all
    t = cf.rotary_positions(q[:, 3], k[:, 3], f, lengths=ints(3, 3))
    assert torch.equal(t[0], a[0][:, 3]) and torch.equal(t[1], a[1][:, 3])
    e = cf.rotary_positions(q[:, :0], k[:, :0], f)
    assert e[0].shape == (2, 0, 8, 64) and e[1].shape == (2, 0, 4, 64)
    assert cf.rotary_positions(q[:0], None, f, lengths=ints()).shape == (0, 9, 8, 64)


def test_gradients_of_two_types_and_changed_arguments():
    g = rng(14)
    f = cf.rotary_frequencies(32)
    at = torch.arange(9).expand(2, 9)
    q, k = normal(g, 2, 9, 4, 48, dtype=torch.bfloat16).cuda().requires_grad_(), normal(g, 2, 9, 2, 48).cuda().requires_grad_()
    y = cf.rotary_positions(q, k, f)
    dy = [normal(g, *t.shape, dtype=t.dtype).cuda() for t in y]
    for dx, d, x in zip(torch.autograd.grad(y, (q, k), dy), dy, (q, k)):
        assert dx.dtype is x.dtype
        near(dx, d, f, at, False, "gradient", inverse=True)
    # queries alone, gradients that lie apart
    y = cf.rotary_positions(q, None, f)
    dy = normal(g, 2, 9, 48, 4, dtype=torch.bfloat16).cuda().transpose(2, 3)
    dx, = torch.autograd.grad(y, q, dy)
    near(dx, dy, f, at, False, "gradient", inverse=True)
    # what the gradients need may not change before they are taken
    for change in ("frequencies", "positions"):
        mine, where = f.clone(), torch.arange(9, dtype=torch.int32, device="cuda").expand(2, 9).contiguous()
        y = cf.rotary_positions(k, k, mine, positions=where)
        (mine if change == "frequencies" else where).add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y[0].sum(), k)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx, = torch.autograd.grad(cf.rotary_positions(k, k, f)[0].square().sum(), k, create_graph=True)
        dx.sum().backward()


def test_nan_stays_in_its_pair():
    f = cf.rotary_frequencies(16)
    for dt in TYPES.values():
        x = torch.ones(1, 2, 1, 24, dtype=dt, device="cuda")
        x[0, 1, 0, 3], x[0, 1, 0, 20] = float("nan"), float("inf")
        y = cf.rotary_positions(x, None, f)
        odd = ~torch.isfinite(y[0, 1, 0])
        assert odd.nonzero().flatten().tolist() == [3, 11, 20] and torch.isfinite(y[0, 0]).all()
        y = cf.rotary_positions(x, None, f, interleaved=True)
        assert (~torch.isfinite(y[0, 1, 0])).nonzero().flatten().tolist() == [2, 3, 20]


def test_captured_training_step():
    g = rng(5)
    f = cf.rotary_frequencies(128, factor=4.0)
    q, k = (normal(g, 2, 50, h, 128, dtype=torch.bfloat16).cuda().requires_grad_() for h in (8, 2))
    dq, dk = (normal(g, 2, 50, h, 128, dtype=torch.bfloat16).cuda() for h in (8, 2))
    at = torch.arange(50, device="cuda", dtype=torch.int32).expand(2, 50).contiguous()

    def step():
        y = cf.rotary_positions(q, k, f, positions=at)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, (q, k), (dq, dk)))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            for t in (q, k, dq, dk):
                t.copy_(normal(g, *t.shape, dtype=torch.bfloat16))
            at += 1000 * i
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_positions_cache_and_attention_together():
    """Prompts and tokens of a layer: turned queries and keys, keys and values held in 8 or 4 bits."""
    g = rng(6)
    B, H, G, D, S = 2, 8, 2, 64, 400
    f = cf.rotary_frequencies(48, base=50000.0, factor=2.0, original_length=256)
    lengths = [0, 150]
    tokens = 90
    for bits in (4, 8):
        cache = cf.quantized_cache(B, S, G, D, bits)
        old = [normal(g, B, 150, G, D, dtype=torch.bfloat16).cuda() for _ in range(2)]
        cf.quantized_cache_write(cache, *old, ints(0, 0), new_lengths=ints(*lengths))
        q, k, v = (normal(g, B, tokens + 3, h, D, dtype=torch.bfloat16).cuda() for h in (H, G, G))
        lens = ints(*lengths)
        got = []
        for now in (slice(0, tokens), *(slice(i, i + 1) for i in range(tokens, tokens + 3))):
            qq, kk = cf.rotary_positions(q[:, now], k[:, now], f, lengths=lens)
            call = cf.softmax_attention_prefill if now.start == 0 else cf.softmax_attention_decode
            got.append(call(qq, kk, v[:, now], cache, lens)[0])
            lens += now.stop - now.start
        y = torch.cat(got, 1)
        for b in range(B):
            n = lengths[b] + tokens + 3
            at = torch.arange(lengths[b], n)[None]
            # queries and keys as the calls rounded them: to within a unit of the plain form's
            turned = cf.rotary_positions(q[b:b + 1], k[b:b + 1], f, lengths=ints(lengths[b]))
            near(turned[0], q[b:b + 1], f, at, False, "q")
            kk, vv = (Q.held(cache[x][b:b + 1, :n], cache[x + "_scale"][b:b + 1, :n]) for x in ("k", "v"))
            assert torch.equal(kk[:, lengths[b]:], Q.rounded(turned[1].cpu(), bits)[0])
            assert torch.equal(vv[:, lengths[b]:], Q.rounded(v[b:b + 1].cpu(), bits)[0])
            ref, tol = M.attention(turned[0], kk, vv, offset=[lengths[b]], unit=M.U[torch.bfloat16], tiny=2.0 ** -126)["y"]
            M.check(y[b:b + 1], ref, tol + M.U[torch.bfloat16] * ref.abs(), "y", torch.bfloat16)


@pytest.mark.parametrize("shape", [(2, 7), (2,)])
def test_tangents_are_refused(shape):
    g = rng(20)
    f = cf.rotary_frequencies(32)
    q, k = normal(g, *shape, 4, 32).cuda(), normal(g, *shape, 2, 32).cuda()
    lens = ints(3, 50)
    plain = cf.rotary_positions(q, k, f, lengths=lens)
    with forward_ad.dual_level():
        for turned in ((forward_ad.make_dual(q, torch.ones_like(q)), k), (q, forward_ad.make_dual(k, torch.ones_like(k))),
                       (forward_ad.make_dual(q, torch.ones_like(q)), None)):
            with pytest.raises(NotImplementedError, match="jvp"):
                cf.rotary_positions(*turned, f, lengths=lens)
        with pytest.raises(NotImplementedError, match="jvp"):
            cf.rotary_positions(q, k, forward_ad.make_dual(f, torch.ones_like(f)), lengths=lens)
        inside = cf.rotary_positions(q, k, f, lengths=lens)
    assert all(torch.equal(a, b) for a, b in zip(plain, inside))


def test_angles_are_rounded_to_the_nearest():
    """Angles near quarter turns, where a sine or cosine is as far off as its angle."""
    from fractions import Fraction
    two_pi = Fraction(884279719003555, 140737488355328) + Fraction(2.449293598294706e-16)        # 2 pi to 106 bits
    g = rng(22)
    at = torch.randint(1, 2 ** 17, (40,), generator=g)
    worst = 0.0
    for i in range(len(at)):
        p = int(at[i])
        # turns a token by which p tokens make a whole number of quarter turns, but for 2^-13 of a turn at most
        quarters = torch.randint(0, p, (64,), generator=g).double() + torch.randn(64, generator=g).double().clamp(-3, 3) * 2.0 ** -13
        f = quarters / 4 / p * (2 * math.pi)
        x = torch.zeros(1, 1, 1, 128)
        x[..., :64] = 1.0
        y = cf.rotary_positions(x.cuda(), None, f, positions=torch.tensor([[p]], device="cuda"))[0, 0, 0].double().cpu()
        for j in range(64):
            turns = Fraction(float(f[j])) / two_pi * p
            quarter = round(4 * turns)
            rest = float((turns - Fraction(quarter, 4)) * two_pi)        # |rest| < 2^-8
            # that of cosine and sine which is small
            got, sign = (y[64 + j], 1 if quarter % 4 == 0 else -1) if quarter % 2 == 0 else (y[j], 1 if quarter % 4 == 3 else -1)
            # half a step of 2^-32 turns, the frequency's of 2^-64 (and as much again in 64-bit turns of a radian) p times, and
            # three roundings of a number of 2^-8
            tol = 2 * math.pi * (2.0 ** -33 + 3 * 2.0 ** -64 * p) + 4 * 2.0 ** -24 * abs(rest)
            worst = max(worst, abs(float(got) - sign * math.sin(rest)) / tol)
    assert worst <= 1.0, worst
