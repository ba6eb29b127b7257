// flare_attn_bwd.h -- gradients of softmax attention.
//
//   delta_i = dy_i . y_i;  dP_ij = dy_i . v_j;  dS_ij = P_ij (dP_ij - delta_i) (1 - tanh^2) scale
//   dq_i = sum_j dS_ij k_j;  dk_j = sum_i dS_ij q_i;  dv_j = sum_i P_ij dy_i
//
// The weights come again from the scores and the forward's log-sum-exp.  Two kernels, so that
// every sum has one owner and one order: attn_dq owns queries and walks over keys, attn_dkv owns
// keys and walks over the queries of every head that shares them.  That costs seven products for
// the five of a joint kernel, whose dq would be added up by atomics.  Where there are few rows or
// keys the sums are split over workgroups, and attn_parts adds them up in order.
//
// Score gradients of 16-bit inputs go into their products in two parts (the value rounded to the type,
// and the rest): their rounding left dq and dk 2.5e-3 off the 64-bit ones (norms), where they are
// 1.9e-3 with both, for 8% of the step.
//
// Tiles of 64 rows (32 in fp32), taken 32 at a time: a tile of 32 rows in LDS, with a barrier for
// each, took 20% longer for dk and dv and 16% for dq (16384 rows in six documents, 16 heads of 128 over
// 4, bf16).  Of 16384 causal rows of one document dq takes 1990 us: 3 + 1 products at 1.1 PFLOP/s; dk and
// dv 3120 us, 4 + 1 products at 0.88 (a large matrix product: 1.34); with capped scores (4 x 4096 rows, 16
// heads of 64) 444 and 577 us, vector instructions.
//
// What a wave owns, us: 32 queries against 16 (D = 64, dq) 476, 526; 32 keys against 16 at D = 64
// (dk and dv) 604, 633; at D = 128 32 keys leave room for one wave a SIMD: 3405, 2439.
#pragma once

#include "flare_attn.h"

namespace flare {
namespace attn {

// Score gradients of fp16 inputs go into their products times a power of 2: with a small dy or long rows
// they lie below fp16's smallest numbers otherwise, the second part too (4096 keys, dy of 1e-4: dq 8%
// off).  |dS_ij| <= |dy_i . v_j| + |dy_i . y_i| <= 2 |dy_i|_1 max|v| comes to between 2^14 and 2^15 so: row by
// row in dq, in dk for all rows that see a workgroup's keys.  attn_ranges, which that takes, is 5 us for
// 512 rows of 8 heads of 64, 7 for 16384 of 16 heads of 128 over 4.
template <typename E> constexpr bool kScaled = __is_same(E, __half);

// delta, from y before its rounding (y and what it was rounded by): an error of delta adds to all of
// a row's dS with one sign.  bf16 dq and dk were 2.7e-3 to 3.0e-3 off the 64-bit ones (norms) with
// delta from the rounded y.  `lanes` (a power of 2) for each row of a head, 16 bytes of it a lane.
template <typename E>
__global__ __launch_bounds__(256) void attn_delta_kernel(AttnArgs p, int lanes, float* delta, float* norms) {
    typedef typename Elem<E>::S S;
    constexpr int PER = 16 / sizeof(E);
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, row = id / lanes;         // (b, i, h)
    if (row >= p.B * p.N * p.H) return;                    // whole rows
    const int col = (int)(id % lanes) * PER;
    float s = 0.0f, norm = 0.0f;
    if (col < p.D) {
        typedef S V __attribute__((ext_vector_type(PER)));
        const V y = *reinterpret_cast<const V*>((const S*)p.y + row * p.D + col);
        const V dy = *reinterpret_cast<const V*>((const S*)p.dy + row * p.D + col);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            s += (float)y[i] * (float)dy[i];
            if (kScaled<E>) norm += fabsf((float)dy[i]);
        }
        if (p.y_rest) {
            const V rest = *reinterpret_cast<const V*>((const S*)p.y_rest + row * p.D + col);
#pragma unroll
            for (int i = 0; i < PER; ++i) s += (float)rest[i] * (float)dy[i];
        }
    }
    for (int o = lanes / 2; o > 0; o >>= 1) {
        s += __shfl_xor(s, o, 64);
        if (kScaled<E>) norm += __shfl_xor(norm, o, 64);
    }
    const int64_t h = row % p.H, i = row / p.H % p.N, b = row / p.H / p.N;
    if (col) return;
    delta[(b * p.H + h) * p.N + i] = s;
    if (kScaled<E>) norms[(b * p.H + h) * p.N + i] = norm;
}

// The largest of each 64 tokens' |dy|_1 and |v|: padding and what is infinite or NaN do not count.
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    return x;
}
template <typename E>
__global__ __launch_bounds__(1024) void attn_ranges_kernel(AttnArgs p, float* ranges) {
    typedef typename Elem<E>::S S;
    __shared__ float left[16][2];
    const int64_t b = blockIdx.y, first = (int64_t)blockIdx.x * kIdTile;
    const int n = (int)min((int64_t)kIdTile, p.N - first), D8 = (int)p.D / 8, GD8 = (int)p.G * D8;
    const int32_t* ids = p.ids ? p.ids + b * p.N + first : nullptr;
    float norm = 0.0f, most = 0.0f;
    for (int e = threadIdx.x; e < (int)p.H * kIdTile; e += 1024) {
        const int i = e % kIdTile;
        if (i >= n || (ids && ids[i] < 0)) continue;
        const float x = p.norms[(b * p.H + e / kIdTile) * p.N + first + i];
        if (x < -kNegInf) norm = fmaxf(norm, x);
    }
#pragma unroll 4
    for (int e = threadIdx.x; e < n * GD8; e += 1024) {
        const int i = e / GD8, g = e % GD8 / D8;
        if (ids && ids[i] < 0) continue;
        const auto v = frag_rows<E>((const S*)p.v.p + b * p.v.sb + (first + i) * p.v.sn + g * p.v.sh + e % D8 * 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = fabsf((float)v[j]);
            if (x < -kNegInf) most = fmaxf(most, x);
        }
    }
    norm = wave_max(norm), most = wave_max(most);
    if ((threadIdx.x & 63) == 0) {
        left[threadIdx.x >> 6][0] = norm;
        left[threadIdx.x >> 6][1] = most;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < 16; ++w) x = fmaxf(x, left[w][threadIdx.x]);
        ranges[(b * gridDim.x + blockIdx.x) * 2 + threadIdx.x] = x;
    }
}
// Over the tiles of tokens first .. last-1 that `mine` meets; the same in all lanes of the wave.
__device__ __forceinline__ float largest(const AttnArgs& p, int64_t b, int which, int first, int last, IdRange mine) {
    const int tiles = id_tiles(p.N);
    float most = 0.0f;
    for (int t = first / kIdTile + (threadIdx.x & 63); t * kIdTile < last; t += 64)
        if (!p.ids || id_range(p, b, t).meets(mine)) most = fmaxf(most, p.ranges[(b * tiles + t) * 2 + which]);
    return wave_max(most);
}
// The power of 2 that brings `bound` to between 2^14 and 2^15.
__device__ __forceinline__ float scale_to(float bound) {
    if (!(bound > 0.0f && bound < -kNegInf)) return 1.0f;
    return __builtin_ldexpf(1.0f, 15 - __builtin_amdgcn_frexp_expf(bound));
}

// An infinite value or NaN in a row of K, Q or dY counts for the pairs that see that row, and a weight
// of 0 times it is NaN for the others.  So tiles that not every pair sees and that hold one take
// their products from operands without such values; what they add to the pairs that do see them
// comes by element from memory in the end: in dq and dk NaN, as the score gradient beside an
// infinite score is 0 or NaN (under a cap with finite weights), and in dv the value itself.
__device__ __forceinline__ bool is_odd(float x) { return !(fabsf(x) < -kNegInf); }

// An operand's infinite values and NaNs set to 0.
template <typename F>
__device__ __forceinline__ F finite(F f) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (is_odd((float)f[i])) f[i] = 0.0f;
    return f;
}

// The weights of the dv product are normalised ones, which in a long row lie below fp16's
// smallest normal number (2^-14): there they come 2^10 times as large.
template <typename E> constexpr float weight_shift() { return __is_same(E, __half) ? 10.0f : 0.0f; }

template <typename E, int DP>
struct BackwardLds {
    static constexpr int T = sizeof(E) == 2 ? 64 : 32;                 // rows of a tile, taken 32 at a time
    static constexpr int P = column_pitch<E, DP>();                    // read both ways
    static constexpr size_t tile = sizeof(E) * T * P;
    static constexpr size_t bytes = 4 * tile + 2 * (3 * T + 4) * sizeof(float);
};

template <typename E, int DP, int QT, int CAP>
__global__ __launch_bounds__(256, 2) void attn_dq_kernel(AttnArgs p) {
    typedef typename Elem<E>::S S;
    typedef typename Elem<E>::Frag Frag;
    using Lds = BackwardLds<E, DP>;
    constexpr int KT = Lds::T, QB = 64 * QT, DK = DP / 32, DT = DP / 16, P = Lds::P;
    extern __shared__ __align__(16) char smem[];
    S* kl = (S*)smem;                                   // [2][KT][P]
    S* vl = (S*)(smem + 2 * Lds::tile);
    int* idl = (int*)(smem + 4 * Lds::tile);            // [2][KT]
    int* oddl = idl + 2 * KT;                           // [2][4]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, c = lane & 15;
    const int N = (int)p.N, R = (int)(p.H / p.G), nq = (N + QB - 1) / QB;
    int id = blockIdx.x;
    const int kvh = id % (int)p.G;
    id /= (int)p.G;
    const int parts = (int)p.dq_splits, part_id = id % parts;      // of the keys
    id /= parts;
    const QueryBlock at(p, id, R, nq);
    const int64_t b = at.b;
    const int h = kvh * R + at.rep, q0 = at.tile * QB;

    const int prefix = p.prefix ? (int)clamp_to(p.prefix[b], p.N) : 0;
    int k_begin = 0, kv_end = p.causal ? max(min(q0 + QB, N), prefix) : N;
    const int seen_end = kv_end;                        // of all parts: y is of all that a row sees
    if (parts > 1) {
        const int tiles = (kv_end + KT - 1) / KT;
        k_begin = (int)((int64_t)tiles * part_id / parts) * KT;
        kv_end = min(kv_end, (int)((int64_t)tiles * (part_id + 1) / parts) * KT);
    }
    IdRange mine{0, 0, true};
    if (p.ids) mine = id_block(p, b, q0, QB);
    const int w0 = q0 + wave * 16 * QT;
    Frag qf[QT][DK], gf[QT][DK];
    int pos[QT], lim[QT], qid[QT];                     // as in attn_forward
    float lse[QT], delta[QT], factor[QT];
    const float most_v = kScaled<E> ? largest(p, b, 1, 0, seen_end, mine) : 0.0f;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int i = w0 + 16 * t + c;
        const bool live = i < N;
        pos[t] = i;
        lim[t] = !live ? 0 : p.causal ? max(i + 1, prefix) : N;
        qid[t] = kNoQuery;
        if (p.ids && live) {
            const int d = p.ids[b * p.N + i];
            qid[t] = d < 0 ? kNoQuery : d;
        }
        lse[t] = live ? p.lse[(b * p.H + h) * p.N + i] : -kNegInf;
        delta[t] = live ? p.delta[(b * p.H + h) * p.N + i] : 0.0f;
        factor[t] = 1.0f;
        if (kScaled<E>) {
            factor[t] = scale_to(live ? 2.0f * most_v * p.norms[(b * p.H + h) * p.N + i] : 0.0f);
            delta[t] *= factor[t];
        }
        const S* q = (const S*)p.q.p + b * p.q.sb + (live ? i : 0) * p.q.sn + h * p.q.sh;
        const S* dy = (const S*)p.dy + ((b * p.N + (live ? i : 0)) * p.H + h) * p.D;
#pragma unroll
        for (int kk = 0; kk < DK; ++kk) {
            const int d = 32 * kk + 8 * g;
            qf[t][kk] = gf[t][kk] = Frag{};
            if (live && d < p.D) {
                qf[t][kk] = frag_rows<E>(q + d);
                gf[t][kk] = frag_rows<E>(dy + d);
            }
        }
    }
    const S* kbase = (const S*)p.k.p + b * p.k.sb + kvh * p.k.sh;
    const S* vbase = (const S*)p.v.p + b * p.v.sb + kvh * p.v.sh;
    const float scale2 = p.scale * kLog2e, slope2 = p.slopes ? p.slopes[h] * kLog2e : 0.0f;
    const float cap2 = p.cap * kLog2e, to_tanh = CAP ? p.scale / p.cap : 0.0f, into_cap = 2.0f * kLog2e * to_tanh;

    const float out_scale = CAP ? 4.0f * p.scale : p.scale;
    f32x4 acc[QT][DT];
    float cap_lse[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        cap_lse[t] = cap2 - lse[t];
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[t][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    auto covers = [&](int k0, int rows, int first, int last) {
        if (k0 + rows > N || last >= N) return false;
        if (p.causal && k0 + rows - 1 > first && k0 + rows > prefix) return false;
        return !p.ids || mine.same(id_range(p, b, k0 / kIdTile));
    };
    Stage<E, KT, DP, P, 256> ks, vs;
    ks.begin(p.k.sn, p.D, tid);
    vs.begin(p.v.sn, p.D, tid);
    int next_id = -1;
    auto fetch = [&](int k0) {
        ks.load(kbase + k0 * p.k.sn, N - k0, p.k.sn, p.D);
        vs.load(vbase + k0 * p.v.sn, N - k0, p.v.sn, p.D);
        if (p.ids && tid < KT) next_id = max(k0 + tid < N ? p.ids[b * p.N + k0 + tid] : kNoKey, kNoKey);
    };
    auto place = [&](int k0, int buf) {
        ks.store(kl + buf * KT * P, tid);
        vs.store(vl + buf * KT * P, tid);
        if (p.ids && tid < KT) idl[buf * KT + tid] = next_id;
        const bool odd = !covers(k0, KT, q0, q0 + QB - 1) && __any(ks.odd());
        if (lane == 0) oddl[buf * 4 + wave] = odd;
    };
    TileWalk<KT> walk(p, b, kv_end, mine);
    int tile = walk.next(k_begin);
    int buf = 0, any_odd = 0;
    if (tile < kv_end) {
        fetch(tile);
        place(tile, 0);
    }
    __syncthreads();
    while (tile < kv_end) {
        const int k1 = walk.next(tile + KT);
        if (k1 < kv_end) fetch(k1);
        const int4 odds = *reinterpret_cast<const int4*>(oddl + buf * 4);
        const int odd = __builtin_amdgcn_readfirstlane(odds.x | odds.y | odds.z | odds.w);
        any_odd |= odd;
#pragma unroll 1
        for (int part = 0; part < KT; part += 32) {
            const int k0 = tile + part;
            const bool hidden = w0 >= N || k0 >= N || (p.causal && k0 > w0 + 16 * QT - 1 && k0 >= prefix);
            if (hidden) continue;
            const S* kt = kl + (buf * KT + part) * P;
            const S* vt = vl + (buf * KT + part) * P;
            f32x4 s[QT][2], dp[QT][2];
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
                for (int n = 0; n < 2; ++n) s[t][n] = dp[t][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int n = 0; n < 2; ++n) {
#pragma unroll
                for (int kk = 0; kk < DK; ++kk) {
                    const Frag a = frag_rows<E>(kt + (16 * n + c) * P + 32 * kk + 8 * g);
                    const Frag v = frag_rows<E>(vt + (16 * n + c) * P + 32 * kk + 8 * g);
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        s[t][n] = mma(a, qf[t][kk], s[t][n]);
                        dp[t][n] = mma(v, gf[t][kk], dp[t][n]);
                    }
                }
            }
            const bool whole = covers(k0, 32, w0, w0 + 16 * QT - 1);
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                const float base = (float)(pos[t] - k0 - 4 * g);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float x = s[t][n][i], slope = 1.0f;        // a quarter of 1 - tanh^2
                        if (CAP == kCapFine) {
                            const Tanh u = fine_tanh(x * to_tanh);
                            x = cap2 * u.t - lse[t];
                            slope = u.slope;
                        } else if (CAP) {
                            // cap tanh(x / cap) = cap (1 - 2 r), 1 - tanh^2 = 4 r (1 - r)
                            const float r = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * into_cap));
                            x = cap_lse[t] - 2.0f * cap2 * r;
                            slope = r - r * r;
                        } else {
                            x = x * scale2 - lse[t];
                        }
                        if (p.slopes) x -= slope2 * fabsf(base - (float)(16 * n + i));
                        const float w = __builtin_amdgcn_exp2f(x);
                        float ds = w * (kScaled<E> ? dp[t][n][i] * factor[t] - delta[t] : dp[t][n][i] - delta[t]);
                        if (CAP) ds *= slope;                  // and 4 in the end
                        s[t][n][i] = ds;
                    }
                }
                if (!whole) {
                    const int left = lim[t] - k0 - 4 * g;
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[t][n][i] = 16 * n + i < left ? s[t][n][i] : 0.0f;
                        if (p.ids) {
                            const int4 d = *reinterpret_cast<const int4*>(idl + buf * KT + part + 16 * n + 4 * g);
                            s[t][n][0] = d.x == qid[t] ? s[t][n][0] : 0.0f;
                            s[t][n][1] = d.y == qid[t] ? s[t][n][1] : 0.0f;
                            s[t][n][2] = d.z == qid[t] ? s[t][n][2] : 0.0f;
                            s[t][n][3] = d.w == qid[t] ? s[t][n][3] : 0.0f;
                        }
                    }
                }
            }
            Frag w[QT], rest[QT];
#pragma unroll
            for (int t = 0; t < QT; ++t) w[t] = split_tiles(s[t][0], s[t][1], rest[t], S{});
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                Frag a = frag_columns<E>(kt + 16 * d, P, g, c);
                if (odd) a = finite(a);
#pragma unroll
                for (int t = 0; t < QT; ++t) {
                    acc[t][d] = mma(a, w[t], acc[t][d]);
                    if (sizeof(E) == 2) acc[t][d] = mma(a, rest[t], acc[t][d]);
                }
            }
        }
        if (k1 < kv_end) place(k1, buf ^ 1);
        __syncthreads();
        buf ^= 1;
        tile = k1;
    }
    if (any_odd) {
        TileWalk<KT> again(p, b, kv_end, mine);
        for (tile = again.next(k_begin); tile < kv_end; tile = again.next(tile + KT)) {
            if (covers(tile, KT, q0, q0 + QB - 1)) continue;
            for (int j = tile; j < min(tile + KT, N); ++j) {
#pragma unroll
                for (int t = 0; t < QT; ++t) {
                    if (j >= lim[t] || (p.ids && max(p.ids[b * p.N + j], kNoKey) != qid[t])) continue;
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        const S* k = kbase + j * p.k.sn + 16 * d + 4 * g;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (16 * d < p.D && is_odd((float)k[e])) acc[t][d][e] = __builtin_nanf("");
                    }
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int i = w0 + 16 * t + c;
        if (i >= N) continue;
        const int64_t row = ((b * p.N + i) * p.H + h) * p.D;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            if (16 * d < p.D) {
                typedef S S4 __attribute__((ext_vector_type(4)));
                const int64_t at = row + 16 * d + 4 * g;
                const f32x4 v = acc[t][d] * (out_scale / factor[t]);
                if (parts > 1) *reinterpret_cast<f32x4*>(p.dq_parts + part_id * (p.B * p.N * p.H * p.D) + at) = v;
                else *reinterpret_cast<S4*>((S*)p.dq + at) = __builtin_convertvector(v, S4);
            }
        }
    }
}

template <typename E, int DP, int KQ, int CAP>
__global__ __launch_bounds__(256, 2) void attn_dkv_kernel(AttnArgs p) {
    typedef typename Elem<E>::S S;
    typedef typename Elem<E>::Frag Frag;
    using Lds = BackwardLds<E, DP>;
    constexpr float kShift = weight_shift<E>(), kUnshift = kShift == 0.0f ? 1.0f : 0x1p-10f;
    constexpr int QR = Lds::T, KB = 64 * KQ, DK = DP / 32, DT = DP / 16, P = Lds::P;
    extern __shared__ __align__(16) char smem[];
    S* ql = (S*)smem;                                   // [2][QR][P]
    S* gl = (S*)(smem + 2 * Lds::tile);
    float* lsel = (float*)(smem + 4 * Lds::tile);       // [2][QR]
    float* dell = lsel + 2 * QR;
    int* idl = (int*)(dell + 2 * QR);
    int* oddl = idl + 2 * QR;                           // [2][4]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, c = lane & 15;
    const int N = (int)p.N, R = (int)(p.H / p.G), parts = (int)p.splits, row_parts = (int)p.row_splits;
    int id = blockIdx.x;
    const int kvh = id % (int)p.G;
    id /= (int)p.G;
    // this workgroup's part of the queries: some of the heads that share these keys, some of the
    // rows; by length alone the keys most queries see come first
    int64_t b;
    int part, kb;
    if (p.key_order) {
        const int tiles = (N + KB - 1) / KB, o = p.key_order[id / parts];
        part = id % parts, b = o / tiles, kb = o % tiles * KB;
    } else {
        b = id % (int)p.B, part = id / (int)p.B % parts, kb = id / (int)p.B / parts * KB;
    }
    const int rep0 = part / row_parts * R / (parts / row_parts);
    const int rep1 = (part / row_parts + 1) * R / (parts / row_parts);

    const int prefix = p.prefix ? (int)clamp_to(p.prefix[b], p.N) : 0;
    int q_begin = p.causal && kb >= prefix ? kb : 0, q_end = N;
    if (row_parts > 1) {
        const int k = part % row_parts, tiles = (N - q_begin + QR - 1) / QR, from = q_begin;
        q_begin = from + (int)((int64_t)tiles * k / row_parts) * QR;
        q_end = min(N, from + (int)((int64_t)tiles * (k + 1) / row_parts) * QR);
    }
    IdRange mine{0, 0, true};
    if (p.ids) mine = id_block(p, b, kb, KB);
    const int w0 = kb + wave * 16 * KQ;                 // this wave's first key
    Frag kf[KQ][DK], vf[KQ][DK];
    int kid[KQ], from[KQ];                              // of this lane's keys: document, and the first row to see it
#pragma unroll
    for (int t = 0; t < KQ; ++t) {
        const int j = w0 + 16 * t + c;
        const bool live = j < N;
        from[t] = !live ? INT32_MAX : p.causal && j >= prefix ? j : 0;
        kid[t] = !live ? kNoKey : p.ids ? max(p.ids[b * p.N + j], kNoKey) : 0;
        const S* k = (const S*)p.k.p + b * p.k.sb + (live ? j : 0) * p.k.sn + kvh * p.k.sh;
        const S* v = (const S*)p.v.p + b * p.v.sb + (live ? j : 0) * p.v.sn + kvh * p.v.sh;
#pragma unroll
        for (int kk = 0; kk < DK; ++kk) {
            const int d = 32 * kk + 8 * g;
            kf[t][kk] = vf[t][kk] = Frag{};
            if (live && d < p.D) {
                kf[t][kk] = frag_rows<E>(k + d);
                vf[t][kk] = frag_rows<E>(v + d);
            }
        }
    }
    const float scale2 = p.scale * kLog2e;
    const float cap2 = p.cap * kLog2e, to_tanh = CAP ? p.scale / p.cap : 0.0f, into_cap = 2.0f * kLog2e * to_tanh;
    float factor = 1.0f;
    if (kScaled<E>) {
        factor = scale_to(2.0f * largest(p, b, 0, q_begin, q_end, mine) * largest(p, b, 1, 0, N, mine));
        factor = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, factor)));
    }
    const float to_ds = kUnshift * factor;              // of dP and delta beside a shifted weight
    f32x4 dk[KQ][DT], dv[KQ][DT];
#pragma unroll
    for (int t = 0; t < KQ; ++t)
#pragma unroll
        for (int d = 0; d < DT; ++d) dk[t][d] = dv[t][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    auto covers = [&](int q0, int rows, int first, int last) {
        if (q0 + rows > N || last >= N) return false;
        if (p.causal && last > q0 && last >= prefix) return false;
        return !p.ids || mine.same(id_range(p, b, q0 / kIdTile));
    };
    Stage<E, QR, DP, P, 256> qs, gs;
    qs.begin(p.q.sn, p.D, tid);
    gs.begin(p.H * p.D, p.D, tid);
    float next_lse = 0.0f, next_delta = 0.0f;
    int next_id = -1;
    auto fetch = [&](int h, int q0) {
        qs.load((const S*)p.q.p + b * p.q.sb + h * p.q.sh + q0 * p.q.sn, N - q0, p.q.sn, p.D);
        gs.load((const S*)p.dy + ((b * p.N + q0) * p.H + h) * p.D, N - q0, p.H * p.D, p.D);
        if (tid < QR) {
            const bool live = q0 + tid < N;
            const int64_t at = (b * p.H + h) * p.N + q0 + tid;
            next_lse = live ? p.lse[at] - kShift - (CAP == kCap ? cap2 : 0.0f) : -kNegInf;
            next_delta = live ? p.delta[at] * to_ds : 0.0f;
            next_id = !live ? kNoQuery : p.ids ? p.ids[b * p.N + q0 + tid] : 0;
            next_id = next_id < 0 ? kNoQuery : next_id;
        }
    };
    auto place = [&](int q0, int buf) {
        const bool odd = !covers(q0, QR, kb, kb + KB - 1) && __any(qs.odd() || gs.odd());
        if (lane == 0) oddl[buf * 4 + wave] = odd;
        qs.store(ql + buf * QR * P, tid);
        gs.store(gl + buf * QR * P, tid);
        if (tid < QR) {
            lsel[buf * QR + tid] = next_lse;
            dell[buf * QR + tid] = next_delta;
            idl[buf * QR + tid] = next_id;
        }
    };
    int buf = 0, any_odd = 0;
    for (int rep = rep0; rep < rep1; ++rep) {
        const int h = kvh * R + rep;
        const float slope2 = p.slopes ? p.slopes[h] * kLog2e : 0.0f;
        TileWalk<QR> walk(p, b, q_end, mine);
        int tile = walk.next(q_begin);
        if (tile < q_end) {
            fetch(h, tile);
            place(tile, buf);
        }
        __syncthreads();
        while (tile < q_end) {
            const int q1 = walk.next(tile + QR);
            if (q1 < q_end) fetch(h, q1);
            const int4 odds = *reinterpret_cast<const int4*>(oddl + buf * 4);
            const int odd = __builtin_amdgcn_readfirstlane(odds.x | odds.y | odds.z | odds.w);
            any_odd |= odd;
#pragma unroll 1
            for (int from_row = 0; from_row < QR; from_row += 32) {
                const int q0 = tile + from_row;
                const bool hidden = w0 >= N || q0 >= N || (p.causal && w0 > q0 + 31 && w0 >= prefix);
                if (hidden) continue;
                const S* qt = ql + (buf * QR + from_row) * P;
                const S* gt = gl + (buf * QR + from_row) * P;
                f32x4 s[KQ][2], dp[KQ][2];
#pragma unroll
                for (int t = 0; t < KQ; ++t)
#pragma unroll
                    for (int n = 0; n < 2; ++n) s[t][n] = dp[t][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int n = 0; n < 2; ++n) {
#pragma unroll
                    for (int kk = 0; kk < DK; ++kk) {
                        const Frag a = frag_rows<E>(qt + (16 * n + c) * P + 32 * kk + 8 * g);
                        const Frag o = frag_rows<E>(gt + (16 * n + c) * P + 32 * kk + 8 * g);
#pragma unroll
                        for (int t = 0; t < KQ; ++t) {
                            s[t][n] = mma(a, kf[t][kk], s[t][n]);
                            dp[t][n] = mma(o, vf[t][kk], dp[t][n]);
                        }
                    }
                }
                const bool whole = covers(q0, 32, w0, w0 + 16 * KQ - 1);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const f32x4 lse = *reinterpret_cast<const f32x4*>(lsel + buf * QR + from_row + 16 * n + 4 * g);
                    const f32x4 delta = *reinterpret_cast<const f32x4*>(dell + buf * QR + from_row + 16 * n + 4 * g);
#pragma unroll
                    for (int t = 0; t < KQ; ++t) {
                        const float base = (float)(q0 + 4 * g - (w0 + 16 * t + c));
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float x = s[t][n][i], slope = 1.0f;
                            if (CAP == kCapFine) {
                                const Tanh u = fine_tanh(x * to_tanh);
                                x = cap2 * u.t - lse[i];
                                slope = u.slope;
                            } else if (CAP) {
                                const float r = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * into_cap));
                                x = -2.0f * cap2 * r - lse[i];          // the log-sum-exp less the cap
                                slope = r - r * r;
                            } else {
                                x = x * scale2 - lse[i];
                            }
                            if (p.slopes) x -= slope2 * fabsf(base + (float)(16 * n + i));
                            const float w = __builtin_amdgcn_exp2f(x);
                            float ds = w * (dp[t][n][i] * to_ds - delta[i]);
                            if (CAP) ds *= slope;
                            s[t][n][i] = w;
                            dp[t][n][i] = ds;
                        }
                        if (!whole) {
                            const int late = from[t] - q0 - 4 * g - 16 * n;
                            const int4 d = *reinterpret_cast<const int4*>(idl + buf * QR + from_row + 16 * n + 4 * g);
                            const int row_id[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                // no branch (&&): in one the compiler left some unseen pairs their weights
                                const bool see = (i >= late) & (row_id[i] == kid[t]);
                                s[t][n][i] = see ? s[t][n][i] : 0.0f;
                                dp[t][n][i] = see ? dp[t][n][i] : 0.0f;
                            }
                        }
                    }
                }
                Frag w[KQ], ds[KQ], rest[KQ];
#pragma unroll
                for (int t = 0; t < KQ; ++t) {
                    w[t] = frag_tiles(s[t][0], s[t][1], S{});
                    ds[t] = split_tiles(dp[t][0], dp[t][1], rest[t], S{});
                }
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    Frag a = frag_columns<E>(qt + 16 * d, P, g, c);
                    Frag o = frag_columns<E>(gt + 16 * d, P, g, c);
                    if (odd) {
                        a = finite(a);
                        o = finite(o);
                    }
#pragma unroll
                    for (int t = 0; t < KQ; ++t) {
                        dk[t][d] = mma(a, ds[t], dk[t][d]);
                        if (sizeof(E) == 2) dk[t][d] = mma(a, rest[t], dk[t][d]);
                        dv[t][d] = mma(o, w[t], dv[t][d]);
                    }
                }
            }
            if (q1 < q_end) place(q1, buf ^ 1);
            __syncthreads();
            buf ^= 1;
            tile = q1;
        }
    }
    for (int rep = rep0; rep < (any_odd ? rep1 : rep0); ++rep) {
        TileWalk<QR> again(p, b, q_end, mine);
        for (int tile = again.next(q_begin); tile < q_end; tile = again.next(tile + QR)) {
            if (covers(tile, QR, kb, kb + KB - 1)) continue;
            for (int i = tile; i < min(tile + QR, N); ++i) {
                const int row_id = p.ids ? p.ids[b * p.N + i] : 0;
                const S* q = (const S*)p.q.p + b * p.q.sb + (kvh * R + rep) * p.q.sh + i * p.q.sn + 4 * g;
                const S* dy = (const S*)p.dy + ((b * p.N + i) * p.H + kvh * R + rep) * p.D + 4 * g;
#pragma unroll
                for (int t = 0; t < KQ; ++t) {
                    if (i < from[t] || row_id < 0 || row_id != kid[t]) continue;
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (16 * d >= p.D) continue;
                            const float o = (float)dy[16 * d + e];
                            if (is_odd((float)q[16 * d + e])) dk[t][d][e] = __builtin_nanf("");
                            if (is_odd(o)) dv[t][d][e] += o;
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < KQ; ++t) {
        const int j = w0 + 16 * t + c;
        if (j >= N) continue;
        const int64_t row = ((b * p.N + j) * p.G + kvh) * p.D, all = p.B * p.N * p.G * p.D;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            if (16 * d < p.D) {
                typedef S S4 __attribute__((ext_vector_type(4)));
                const f32x4 k4 = dk[t][d] * ((CAP ? 4.0f * p.scale : p.scale) / factor), v4 = dv[t][d] * kUnshift;
                const int64_t at = row + 16 * d + 4 * g;
                if (p.splits > 1) {
                    *reinterpret_cast<f32x4*>(p.parts + part * 2 * all + at) = k4;
                    *reinterpret_cast<f32x4*>(p.parts + (part * 2 + 1) * all + at) = v4;
                } else {
                    *reinterpret_cast<S4*>((S*)p.dk + at) = __builtin_convertvector(k4, S4);
                    *reinterpret_cast<S4*>((S*)p.dv + at) = __builtin_convertvector(v4, S4);
                }
            }
        }
    }
}

// The parts' sums, in order: of dq (blockIdx.y 0), dk and dv, those that were split.
template <typename E>
__global__ __launch_bounds__(256) void attn_parts_kernel(AttnArgs p) {
    typedef typename Elem<E>::S S;
    typedef S S4 __attribute__((ext_vector_type(4)));
    constexpr int U = 4;
    const int what = blockIdx.y;
    const int64_t all = p.B * p.N * p.D * (what ? p.G : p.H), at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    const int splits = (int)(what ? p.splits : p.dq_splits);
    if (at >= all || splits == 1) return;
    const int64_t stride = what ? 2 * all : all;
    const float* from = (what ? p.parts + (what - 1) * all : p.dq_parts) + at;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < splits; s0 += U) {
        f32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const f32x4*>(from + min(s0 + u, splits - 1) * stride);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + u < splits) sum += v[u];
    }
    S* to = (S*)(what == 0 ? p.dq : what == 1 ? p.dk : p.dv) + at;
    *reinterpret_cast<S4*>(to) = __builtin_convertvector(sum, S4);
}

template <typename K>
static int allow_lds(K kernel, size_t bytes, const char* what) {
    if (bytes <= 65536) return FLARE_OK;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == hipSuccess) return FLARE_OK;
    set_error("%s: %s", what, hipGetErrorString(e));
    return FLARE_ERR_LAUNCH;
}

template <typename E, int DP, int CAP>
static int backward_cap(const AttnArgs& p, hipStream_t stream) {
    constexpr int QT = q_tiles(sizeof(E));
    constexpr size_t bytes = BackwardLds<E, DP>::bytes;
    auto dq = attn_dq_kernel<E, DP, QT, CAP>;
    constexpr int KQ = kv_tiles(sizeof(E), DP);
    auto dkv = attn_dkv_kernel<E, DP, KQ, CAP>;
    int rc = allow_lds(dq, bytes, "attn_dq");
    if (rc == FLARE_OK) rc = allow_lds(dkv, bytes, "attn_dkv");
    if (rc != FLARE_OK) return rc;
    const int64_t blocks = ceil_div(p.N, 64 * QT) * p.B;
    dq<<<dim3((unsigned)(blocks * p.H * p.dq_splits)), 256, bytes, stream>>>(p);
    if ((rc = check_launch("attn_dq")) != FLARE_OK) return rc;
    dkv<<<dim3((unsigned)(ceil_div(p.N, 64 * KQ) * p.B * p.G * p.splits)), 256, bytes, stream>>>(p);
    if ((rc = check_launch("attn_dkv")) != FLARE_OK || (p.splits == 1 && p.dq_splits == 1)) return rc;
    const int64_t most = p.B * p.N * p.D * (p.dq_splits > 1 ? p.H : p.G);
    attn_parts_kernel<E><<<dim3((unsigned)ceil_div(most, 1024), p.splits > 1 ? 3 : 1), 256, 0, stream>>>(p);
    return check_launch("attn_parts");
}
template <typename E, int DP>
static int backward_dp(const AttnArgs& p, hipStream_t stream) {
    if (p.cap == 0.0f) return backward_cap<E, DP, kNoCap>(p, stream);
    if constexpr (sizeof(E) == 2)
        if (p.cap <= kCoarseCapMost) return backward_cap<E, DP, kCap>(p, stream);
    return backward_cap<E, DP, kCapFine>(p, stream);
}
template <typename E>
int backward_e(const AttnArgs& p, float* delta, float* norms, float* ranges, hipStream_t stream) {
    int lanes = 2;
    while (lanes * (int)(16 / sizeof(E)) < p.D) lanes *= 2;
    const int64_t threads = p.B * p.N * p.H * lanes;
    attn_delta_kernel<E><<<dim3((unsigned)ceil_div(threads, 256)), 256, 0, stream>>>(p, lanes, delta, norms);
    int rc = check_launch("attn_delta");
    if (rc != FLARE_OK) return rc;
    if constexpr (kScaled<E>) {
        attn_ranges_kernel<E><<<dim3((unsigned)ceil_div(p.N, kIdTile), (unsigned)p.B), 1024, 0, stream>>>(p, ranges);
        if ((rc = check_launch("attn_ranges")) != FLARE_OK) return rc;
    }
    return p.D <= 32   ? backward_dp<E, 32>(p, stream)
           : p.D <= 64 ? backward_dp<E, 64>(p, stream)
           : p.D <= 96 ? backward_dp<E, 96>(p, stream)
                       : backward_dp<E, 128>(p, stream);
}

}  // namespace attn
}  // namespace flare
