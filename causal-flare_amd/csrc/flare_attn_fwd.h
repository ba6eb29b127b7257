// flare_attn_fwd.h -- softmax attention, forward (training and prompts that continue a cache).
//
// A workgroup of four waves owns 64 QT queries of one head, 16 QT a wave, with Q as the B
// operand in registers; K and V come through LDS in tiles of KT keys, two of each, the next
// one's loads in flight while one is computed.  The running maximum moves only when a score
// passes it by 2^8, so that most tiles rescale nothing.  Weights are rounded to the inputs' type
// for the product with V (their sum is taken before that, in fp32).  Where there are few rows the
// keys are split over `splits` workgroups, whose shares attn_rows joins.
//
// Bound: at two waves a SIMD (the registers hold Q, 32 x 64 scores and 32 x D sums a wave) the
// products and the exponentials of a wave alternate and overlap only with the other wave's.  bf16,
// causal, products at a large matrix product's rate for comparison: 16384 rows, 16 heads of 128 over
// 4, 1243 us, 0.88 PFLOP/s of 1.34; 4 x 4096 rows, 16 heads of 64, capped scores (three
// transcendental instructions a pair) 260 us, 0.53.  32 queries a wave against 16: 275 and 285 us.
#pragma once

#include "flare_attn.h"

namespace flare {
namespace attn {

// With weights of 2^(s - cap) a row's largest is at least 2^(-2 cap): bf16 holds that, with all that
// counts beside it, and fp16 does not.  Up to here (log2 units; caps of 30.5) it is 2^-88 or more, and its
// products with values of 2^-49 keep 12 digits above fp32's smallest number.  (fp32 inputs would lose
// digits: s - cap rounds to fewer than s has.)
constexpr float kCapFixedMost = 44.0f;
constexpr float kSlack = 8.0f;       // log2 of the largest weight before the reference moves

template <typename E, int DP, int KT>
struct ForwardLds {
    static constexpr int KP = row_pitch<E, DP>(), VP = column_pitch<E, DP>();
    static constexpr size_t k_bytes = sizeof(E) * KT * KP, v_bytes = sizeof(E) * KT * VP;
    static constexpr size_t bytes = 2 * (k_bytes + v_bytes + KT * sizeof(int)) + sizeof(int);
};

template <typename E, int DP, int QT, int KT, int CAP>
__global__ __launch_bounds__(256, 2) void attn_forward_kernel(AttnArgs p) {
    typedef typename Elem<E>::S S;
    typedef typename Elem<E>::Frag Frag;
    using Lds = ForwardLds<E, DP, KT>;
    constexpr int QB = 64 * QT, DK = DP / 32, DT = DP / 16, NK = KT / 16, KP = Lds::KP, VP = Lds::VP;
    extern __shared__ __align__(16) char smem[];
    S* kl = (S*)smem;
    S* vl = (S*)(smem + 2 * Lds::k_bytes);
    int* idl = (int*)(smem + 2 * (Lds::k_bytes + Lds::v_bytes));
    int* oddl = idl + 2 * KT;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, c = lane & 15;

    // heads that share keys, and then the tiles of one head, are 8 workgroups or a multiple of
    // that apart where there are 8 key heads: one XCD and its L2.  The longest rows come first.
    const int R = (int)(p.H / p.G), nq = ((int)p.N + QB - 1) / QB;
    int id = blockIdx.x;
    const int kvh = id % (int)p.G;
    id /= (int)p.G;
    const int parts = (int)p.splits, part = id % parts;            // of the keys
    id /= parts;
    const QueryBlock at(p, id, R, nq);
    const int64_t b = at.b;
    const int h = kvh * R + at.rep, q0 = at.tile * QB;

    int off = 0, qlen = (int)p.N, kvlen = (int)p.M;
    bool refused = false;
    if (p.lengths) {
        off = p.lengths[b];
        qlen = (int)(p.fresh ? clamp_to(p.fresh[b], p.N) : p.N);
        if (off < 0) off = qlen = 0;
        refused = (int64_t)off + qlen > p.M;
        if (refused) off = qlen = 0;
        kvlen = off + qlen;
    }
    const int prefix = p.prefix ? (int)clamp_to(p.prefix[b], p.M) : 0;
    int kv_end = 0;
    if (q0 < qlen) {
        kv_end = kvlen;
        if (p.causal) kv_end = min(kvlen, max(off + min(q0 + QB, qlen), prefix));
    }
    int k_begin = 0;
    if (parts > 1) {
        const int tiles = (kv_end + KT - 1) / KT;
        k_begin = (int)((int64_t)tiles * part / parts) * KT;
        kv_end = min(kv_end, (int)((int64_t)tiles * (part + 1) / parts) * KT);
    }
    IdRange mine{0, 0, true};
    if (p.ids) mine = id_block(p, b, q0, QB);

    const int w0 = q0 + wave * 16 * QT;                // this wave's first query
    Frag qf[QT][DK];
    int pos[QT], lim[QT];                              // of this lane's queries: position, and the keys below
    int qid[QT];                                       // which it sees those of its document
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int i = w0 + 16 * t + c;
        const bool live = i < qlen;
        pos[t] = i + off;
        lim[t] = !live ? 0 : p.causal ? min(kvlen, max(pos[t] + 1, prefix)) : kvlen;
        qid[t] = kNoQuery;
        if (p.ids && live) {
            const int d = p.ids[b * p.N + i];
            qid[t] = d < 0 ? kNoQuery : d;
        }
        const S* row = (const S*)p.q.p + b * p.q.sb + (live ? i : 0) * p.q.sn + h * p.q.sh;
#pragma unroll
        for (int kk = 0; kk < DK; ++kk) {
            const int d = 32 * kk + 8 * g;
            qf[t][kk] = Frag{};
            if (live && d < p.D) qf[t][kk] = frag_rows<E>(row + d);
            if (p.scale < 0.0f) qf[t][kk] = -qf[t][kk];          // scores then scale by |scale|
        }
    }
    const S* kbase = (const S*)p.k.p + b * p.k.sb + kvh * p.k.sh;
    const S* vbase = (const S*)p.v.p + b * p.v.sb + kvh * p.v.sh;
    const float scale2 = fabsf(p.scale) * kLog2e, slope2 = p.slopes ? p.slopes[h] * kLog2e : 0.0f;
    const float cap2 = p.cap * kLog2e, to_tanh = CAP ? fabsf(p.scale) / p.cap : 0.0f, into_cap = 2.0f * kLog2e * to_tanh;

    f32x4 acc[QT][DT];
    float top[QT], sum[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        top[t] = CAP == kCapFixed ? cap2 : kNegInf;
        sum[t] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[t][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    auto covers = [&](int k0, int first, int last) {       // every query sees every key
        if (k0 + KT > kvlen || last >= qlen) return false;
        if (p.causal && k0 + KT - 1 > first + off && k0 + KT > prefix) return false;
        return !p.ids || mine.same(id_range(p, b, k0 / kIdTile));
    };
    Stage<E, KT, DP, KP, 256> ks;
    Stage<E, KT, DP, VP, 256> vs;
    ks.begin(p.k.sn, p.D, tid);
    vs.begin(p.v.sn, p.D, tid);
    int next_id = -1;
    auto fetch = [&](int k0) {
        ks.load(kbase + k0 * p.k.sn, kvlen - k0, p.k.sn, p.D);
        vs.load(vbase + k0 * p.v.sn, kvlen - k0, p.v.sn, p.D);
        if (p.ids && tid < KT) next_id = max(k0 + tid < (int)p.N ? p.ids[b * p.N + k0 + tid] : kNoKey, kNoKey);
    };
    auto place = [&](int k0, int buf) {
        // A weight of 0 times an infinite value is NaN: tiles that some query does not see whole
        // leave such values to the end.
        if (!covers(k0, q0, q0 + QB - 1) && vs.odd()) {
            vs.clean();
            *oddl = 1;
        }
        ks.store(kl + buf * KT * KP, tid);
        vs.store(vl + buf * KT * VP, tid);
        if (p.ids && tid < KT) idl[buf * KT + tid] = next_id;
    };

    TileWalk<KT> walk(p, b, kv_end, mine);
    int k0 = walk.next(k_begin);
    int buf = 0;
    if (tid == 0) *oddl = 0;
    __syncthreads();
    if (k0 < kv_end) {
        fetch(k0);
        place(k0, 0);
    }
    __syncthreads();
    while (k0 < kv_end) {
        const int k1 = walk.next(k0 + KT);
        if (k1 < kv_end) fetch(k1);
        const bool hidden = w0 >= qlen || (p.causal && k0 > w0 + 16 * QT - 1 + off && k0 >= prefix);
        if (!hidden) {
            const S* kt = kl + buf * KT * KP;
            const S* vt = vl + buf * KT * VP;
            f32x4 s[QT][NK];
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
                for (int n = 0; n < NK; ++n) s[t][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int n = 0; n < NK; ++n) {
#pragma unroll
                for (int kk = 0; kk < DK; ++kk) {
                    const Frag a = frag_rows<E>(kt + (16 * n + c) * KP + 32 * kk + 8 * g);
#pragma unroll
                    for (int t = 0; t < QT; ++t) s[t][n] = mma(a, qf[t][kk], s[t][n]);
                }
            }
            const bool whole = covers(k0, w0, w0 + 16 * QT - 1);
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                // Scores become log2 weights: those that the cap bounds relative to it (kCapFixed),
                // others absolute, and plain ones stay as they are until their exponential.
                const bool plain = CAP == kNoCap && whole && !p.slopes;
                if (CAP != kNoCap) {
#pragma unroll
                    for (int n = 0; n < NK; ++n) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if constexpr (CAP == kCapFine) {
                                s[t][n][i] = cap2 * fine_tanh(s[t][n][i] * to_tanh).t;
                                continue;
                            }
                            // cap tanh(x / cap) = cap - 2 cap / (e^(2 x / cap) + 1)
                            const float r = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(s[t][n][i] * into_cap));
                            s[t][n][i] = CAP == kCapFixed ? -2.0f * cap2 * r : cap2 - 2.0f * cap2 * r;
                        }
                    }
                } else if (!plain) {
#pragma unroll
                    for (int n = 0; n < NK; ++n) s[t][n] *= scale2;
                }
                if (p.slopes) {
                    const float base = (float)(pos[t] - k0 - 4 * g);
#pragma unroll
                    for (int n = 0; n < NK; ++n) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[t][n][i] -= slope2 * fabsf(base - (float)(16 * n + i));
                    }
                }
                if (!whole) {
                    const int left = lim[t] - k0 - 4 * g;
#pragma unroll
                    for (int n = 0; n < NK; ++n) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[t][n][i] = 16 * n + i < left ? s[t][n][i] : kNegInf;
                        if (p.ids) {
                            const int4 d = *reinterpret_cast<const int4*>(idl + buf * KT + 16 * n + 4 * g);
                            s[t][n][0] = d.x == qid[t] ? s[t][n][0] : kNegInf;
                            s[t][n][1] = d.y == qid[t] ? s[t][n][1] : kNegInf;
                            s[t][n][2] = d.z == qid[t] ? s[t][n][2] : kNegInf;
                            s[t][n][3] = d.w == qid[t] ? s[t][n][3] : kNegInf;
                        }
                    }
                }
                float ref = 0.0f;
                if (CAP != kCapFixed) {
                    // not the inline assembly of max3_raw: the compiler leaves no wait states between a
                    // product and assembly that reads it
                    float m = kNegInf;
#pragma unroll
                    for (int n = 0; n < NK; ++n) {
                        m = fmaxf(fmaxf(s[t][n][0], s[t][n][1]), m);
                        m = fmaxf(fmaxf(s[t][n][2], s[t][n][3]), m);
                    }
                    m = column_max(m);
                    if (plain) m *= scale2;
                    if (__any(m > top[t] + kSlack)) {
                        const float to = fmaxf(m, top[t]);
                        const float f = top[t] == to ? 1.0f : __builtin_amdgcn_exp2f(top[t] - to);
                        top[t] = to;
                        sum[t] *= f;
#pragma unroll
                        for (int d = 0; d < DT; ++d) acc[t][d] *= f;
                    }
                    ref = top[t] == kNegInf ? 0.0f : top[t];
                }
                if (plain) {
#pragma unroll
                    for (int n = 0; n < NK; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[t][n][i] = __builtin_amdgcn_exp2f(s[t][n][i] * scale2 - ref);
                } else {
#pragma unroll
                    for (int n = 0; n < NK; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            s[t][n][i] = __builtin_amdgcn_exp2f(CAP == kCapFixed ? s[t][n][i] : s[t][n][i] - ref);
                }
#pragma unroll
                for (int n = 0; n < NK; ++n) sum[t] += (s[t][n][0] + s[t][n][1]) + (s[t][n][2] + s[t][n][3]);
            }
            Frag w[QT][NK / 2];
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
                for (int n = 0; n < NK / 2; ++n) w[t][n] = frag_tiles(s[t][2 * n], s[t][2 * n + 1], S{});
#pragma unroll
            for (int n = 0; n < NK / 2; ++n) {
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const Frag a = frag_columns<E>(vt + 32 * n * VP + 16 * d, VP, g, c);
#pragma unroll
                    for (int t = 0; t < QT; ++t) acc[t][d] = mma(a, w[t][n], acc[t][d]);
                }
            }
        }
        if (k1 < kv_end) place(k1, buf ^ 1);
        __syncthreads();
        buf ^= 1;
        k0 = k1;
    }

    if (*oddl) {
        // the infinite values and NaNs that a query does see, from memory
        TileWalk<KT> again(p, b, kv_end, mine);
        for (k0 = again.next(k_begin); k0 < kv_end; k0 = again.next(k0 + KT)) {
            if (covers(k0, q0, q0 + QB - 1)) continue;
            for (int j = k0; j < min(k0 + KT, kvlen); ++j) {
#pragma unroll
                for (int t = 0; t < QT; ++t) {
                    if (j >= lim[t] || (p.ids && max(p.ids[b * p.N + j], kNoKey) != qid[t])) continue;
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (16 * d >= p.D) continue;
                            const float v = (float)vbase[j * p.v.sn + 16 * d + 4 * g + e];
                            if (!(fabsf(v) < -kNegInf)) acc[t][d][e] += v;
                        }
                    }
                }
            }
        }
    }

#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int i = w0 + 16 * t + c;
        const float total = column_sum(sum[t]);
        // Every query but padding and those behind the length sees itself.  (A sum of 0 does not tell: the
        // scores of one that sees keys may all be -inf, and its y is NaN.)
        const bool sees = lim[t] > 0 && (!p.ids || qid[t] != kNoQuery);
        const float inv = sees ? 1.0f / total : 0.0f;
        if (i >= p.N) continue;
        if (parts > 1) {
            float* to = p.parts + (((b * p.H + h) * p.N + i) * parts + part) * (p.D + 4);
#pragma unroll
            for (int d = 0; d < DT; ++d)
                if (16 * d < p.D) *reinterpret_cast<f32x4*>(to + 16 * d + 4 * g) = acc[t][d];
            if (g == 0) {
                to[p.D] = top[t];
                to[p.D + 1] = total;
            }
            continue;
        }
        if (p.lse && g == 0)
            p.lse[(b * p.H + h) * p.N + i] = sees ? top[t] + __builtin_amdgcn_logf(total) : -kNegInf;
        const int64_t row = ((b * p.N + i) * p.H + h) * p.D;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            if (16 * d < p.D) {
                f32x4 o = acc[t][d] * inv;
                if (refused) o = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
                put_y<S>(p, row + 16 * d + 4 * g, o);
            }
        }
    }
}

// What the parts of each row leave, joined: 32 lanes a row, four dimensions a lane.
template <typename E>
__global__ __launch_bounds__(256) void attn_rows_kernel(AttnArgs p) {
    typedef typename Elem<E>::S S;
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);             // (b, h, i)
    const int d = (threadIdx.x & 31) * 4;
    if (row >= p.B * p.H * p.N || d >= p.D) return;
    const int64_t i = row % p.N, h = row / p.N % p.H, b = row / p.N / p.H;
    const Joined j = join_parts<1, 4>(p.parts + row * p.splits * (p.D + 4), 0, (int)p.splits, p.D, d);
    bool sees = !p.ids || p.ids[b * p.N + i] >= 0, refused = false;       // as in attn_forward
    if (p.lengths) {
        const int64_t off = p.lengths[b], n = p.fresh ? clamp_to(p.fresh[b], p.N) : p.N;
        sees = off >= 0 && i < n;
        refused = off >= 0 && off + n > p.M;
    }
    f32x4 v = sees ? j.v * (1.0f / j.total) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (refused) v = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
    put_y<S>(p, ((b * p.N + i) * p.H + h) * p.D + d, v);
    if (p.lse && d == 0) p.lse[row] = sees ? j.top + __builtin_amdgcn_logf(j.total) : -kNegInf;
}

template <typename E, int DP, int CAP>
static int forward_cap(const AttnArgs& p, hipStream_t stream) {
    constexpr int QT = q_tiles(sizeof(E)), KT = sizeof(E) == 2 ? 64 : 32;
    constexpr size_t bytes = ForwardLds<E, DP, KT>::bytes;
    auto kernel = attn_forward_kernel<E, DP, QT, KT, CAP>;
    if (bytes > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != hipSuccess) {
            set_error("attn_forward: %s", hipGetErrorString(e));
            return FLARE_ERR_LAUNCH;
        }
    }
    const int64_t blocks = ceil_div(p.N, 64 * QT) * p.H * p.B * p.splits;
    kernel<<<dim3((unsigned)blocks), 256, bytes, stream>>>(p);
    const int rc = check_launch("attn_forward");
    if (rc != FLARE_OK || p.splits == 1) return rc;
    attn_rows_kernel<E><<<dim3((unsigned)ceil_div(p.B * p.H * p.N, 8)), 256, 0, stream>>>(p);
    return check_launch("attn_rows");
}
template <typename E, int DP>
static int forward_dp(const AttnArgs& p, hipStream_t stream) {
    if (p.cap == 0.0f) return forward_cap<E, DP, kNoCap>(p, stream);
    if constexpr (__is_same(E, __hip_bfloat16))
        if (!p.slopes && p.cap * kLog2e <= kCapFixedMost) return forward_cap<E, DP, kCapFixed>(p, stream);
    if constexpr (sizeof(E) == 2)
        if (p.cap <= kCoarseCapMost) return forward_cap<E, DP, kCap>(p, stream);
    return forward_cap<E, DP, kCapFine>(p, stream);
}
template <typename E>
int forward_e(const AttnArgs& p, hipStream_t stream) {
    return p.D <= 32   ? forward_dp<E, 32>(p, stream)
           : p.D <= 64 ? forward_dp<E, 64>(p, stream)
           : p.D <= 96 ? forward_dp<E, 96>(p, stream)
                       : forward_dp<E, 128>(p, stream);
}

}  // namespace attn
}  // namespace flare
