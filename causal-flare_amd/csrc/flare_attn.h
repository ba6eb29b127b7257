// flare_attn.h -- exact softmax attention: what its kernels share.
//
//   x_ij = scale q_i . k_j, or cap tanh(scale q_i . k_j / cap);  s_ij = x_ij - slope |i - j|
//   p_ij = exp(s_ij) / sum_j exp(s_ij) over the keys j that i sees;   y_i = sum_j p_ij v_j
//
// Query i sees key j if j <= i or j < prefix (or all, without `causal`), if the two have the
// same document id and it is not negative, and if neither lies behind its sequence's end.  A
// query that sees nothing has y = 0.  Positions count from the front of the cache where there
// is one.  Scores are kept in log2 units.
//
// Products.  With lane = (g, c), g = lane / 16, c = lane % 16, the 16x16 MFMA takes row c of A
// and column c of B with contraction indices 8g .. 8g+7 (of 32), and leaves rows 4g .. 4g+3 of
// column c.  So S^T = K Q^T leaves a lane 4 keys of each 16 of one query, and two such tiles are
// the B operand of a product over keys, if its A operand takes the keys in the same order: 4g+i
// of the first 16 and 4g+i of the second.  Transposed LDS reads give just that from rows of V.
// Scores, weights and outputs thus never change lanes.  fp32 operands go through eight 16x16x4
// products, which take the same registers.
#pragma once

#include "flare_mix.h"

namespace flare {
namespace attn {

using mfma::bf16;
using mfma::bf16x8;
using mfma::f16;
using mfma::f16x8;
using mfma::f32x4;
using mix::ceil_div;
using mix::kLn2;
using mix::kLog2e;
using mix::known_dtype;

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32;
typedef u32 u32x2 __attribute__((ext_vector_type(2)));
typedef u32 u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int64_t kMostStride = 1 << 22;      // between rows, so that a tile's offsets fit 31 bits
constexpr int kIdTile = 64;          // tokens of one entry of the id statistics

struct Rows {                        // a [B, n, heads, D] tensor: element strides
    const void* p;
    int64_t sb, sn, sh;
};

// Rows on 16-byte boundaries.
inline bool aligned(const Rows& r, int dtype) {
    const int64_t per = dtype == FLARE_F32 ? 4 : 8;
    return ((uintptr_t)r.p & 15) == 0 && r.sb % per == 0 && r.sn % per == 0 && r.sh % per == 0 && r.sn >= 0 &&
           r.sn < kMostStride;
}

struct AttnArgs {
    Rows q, k, v;
    void* y;                         // [B, N, H, D]
    void* y_rest;                    // [B, N, H, D] or NULL: what y was rounded by, for the backward's dy . y
    float* lse;                      // [B, H, N], log2 units; +inf for a row that sees nothing
    const float* slopes;             // [H]
    const int32_t *ids, *prefix;     // [B, N], [B]
    const int32_t* id_stats;         // [B, tiles, 3]: smallest and largest id of 64 tokens, whether they have just one
    const int32_t *order, *key_order;    // blocks of queries and of keys, the costliest first (or NULL)
    const int32_t *lengths, *fresh;  // [B]: tokens in the cache before these, and how many of these are real
    int64_t B, N, M, H, G, D;        // M: rows of k and v
    float scale, cap;
    int causal;
    // backward
    const void* dy;                  // [B, N, H, D]
    const float* delta;              // [B, H, N]: dy . y
    const float* norms;              // [B, H, N]: sum of |dy| (fp16)
    const float* ranges;             // [B, tiles, 2]: of 64 tokens the largest norm and |v| (fp16)
    void *dq, *dk, *dv;
    int64_t row_splits;              // of `splits`: parts of the rows, times parts of the heads; over a cache of 8 or 4
                                     // bits: key heads of the same tokens that a workgroup's waves take side by side
    float* dq_parts;                 // what `dq_splits` workgroups leave of each row of dq
    int64_t dq_splits;
    // single tokens
    const void *k_new, *v_new;       // [B, G, D]
    int64_t kn_sb, kn_sg, vn_sb, vn_sg;
    int64_t kn_sn, vn_sn;            // of their tokens, where there may be more than one
    float* parts;                    // what `splits` workgroups leave of each sum
    int64_t splits;
    // a cache of 8 or 4 bits: the codes are k.p and v.p
    uint8_t *k_scale, *v_scale;      // [B, M, G, blocks of 32 dimensions]
};

// How a kernel takes scores: as they are; capped, with tanh to an absolute error (kCap), and against the
// cap itself in place of a running maximum where nothing is added (kCapFixed, forward); or with a tanh that
// keeps the digits of small scores too (kCapFine).
enum { kNoCap = 0, kCap = 1, kCapFixed = 2, kCapFine = 3 };
// tanh as 1 - 2 / (e^2x + 1) leaves a score some 1.3e-7 of the cap off, however small it is: up to this cap
// 2^-15, a sixteenth of what fp16's rounding of a weight is off by.  Beyond it, and for fp32 inputs,
// kCapFine.  us of 4 x 4096 rows, 16 heads of 64, fp16, with caps of 200 and of 300: forward 286, 401; dq
// 442, 535; dk and dv 554, 738.  (Single tokens always: 185 us with either.)
constexpr float kCoarseCapMost = 256.0f;
// Caps that keep scale / cap and cap log2(e) far from fp32's ends.
constexpr float kLeastCap = 0x1p-100f, kMostCap = 0x1p100f;

// Tiles of 16 queries a wave of the forward's and the query gradients' kernels owns (fp32 operands take
// twice the registers).
constexpr int q_tiles(int size) { return size == 2 ? 2 : 1; }
// Tiles of 16 keys a wave of the key gradients' kernel owns: as many as leave two waves a SIMD.
constexpr int kv_tiles(int size, int DP) { return size == 2 && DP <= 64 ? 2 : 1; }

// Four dimensions of a row of y at element `at`, and what they are rounded by.
template <typename S>
__device__ __forceinline__ void put_y(const AttnArgs& p, int64_t at, f32x4 o) {
    typedef S S4 __attribute__((ext_vector_type(4)));
    const S4 y = __builtin_convertvector(o, S4);
    *reinterpret_cast<S4*>((S*)p.y + at) = y;
    if (p.y_rest) {
        const f32x4 rest = o - __builtin_convertvector(y, f32x4);
        *reinterpret_cast<S4*>((S*)p.y_rest + at) = __builtin_convertvector(rest, S4);
    }
}

// Ids as the kernels compare them: padding's negative ones are those of no key and of no query.
constexpr int kNoKey = -1, kNoQuery = -2;

__device__ __forceinline__ int64_t clamp_to(int64_t n, int64_t most) { return n < 0 ? 0 : (n > most ? most : n); }

template <typename E> struct Elem;
template <> struct Elem<__hip_bfloat16> {
    typedef bf16 S;
    typedef bf16x8 Frag;
};
template <> struct Elem<__half> {
    typedef f16 S;
    typedef f16x8 Frag;
};
template <> struct Elem<float> {
    typedef float S;
    typedef f32x8 Frag;
};

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(f32x8 a, f32x8 b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
}

// Eight elements as an operand; p is 16-byte aligned.
template <typename E>
__device__ __forceinline__ typename Elem<E>::Frag frag_rows(const typename Elem<E>::S* p) {
    typedef typename Elem<E>::Frag F;
    if constexpr (sizeof(E) == 4) {
        const f32x4* q = reinterpret_cast<const f32x4*>(p);
        return __builtin_shufflevector(q[0], q[1], 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
        return *reinterpret_cast<const F*>(p);
    }
}
// The two tiles of weights of one query (or key) as an operand over 32 keys (queries).
__device__ __forceinline__ bf16x8 frag_tiles(f32x4 a, f32x4 b, bf16) {
    typedef bf16 v4 __attribute__((ext_vector_type(4)));
    return __builtin_shufflevector(__builtin_convertvector(a, v4), __builtin_convertvector(b, v4), 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ f16x8 frag_tiles(f32x4 a, f32x4 b, f16) {
    typedef f16 v4 __attribute__((ext_vector_type(4)));
    return __builtin_shufflevector(__builtin_convertvector(a, v4), __builtin_convertvector(b, v4), 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ f32x8 frag_tiles(f32x4 a, f32x4 b, float) {
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
// The same, and what that rounds the values by as an operand of its own.
__device__ __forceinline__ bf16x8 split_tiles(f32x4 a, f32x4 b, bf16x8& rest, bf16 type) {
    // the upper half of each value; the rest is exact in fp32
    auto pack = [](f32x4 v) {
        typedef bf16 v4 __attribute__((ext_vector_type(4)));
        const u32x4 u = __builtin_bit_cast(u32x4, v);
        const u32x2 hi = {__builtin_amdgcn_perm(u[1], u[0], 0x07060302u), __builtin_amdgcn_perm(u[3], u[2], 0x07060302u)};
        return __builtin_bit_cast(v4, hi);
    };
    auto left = [](f32x4 v) {
        return v - __builtin_bit_cast(f32x4, __builtin_bit_cast(u32x4, v) & 0xffff0000u);
    };
    rest = frag_tiles(left(a), left(b), type);
    return __builtin_shufflevector(pack(a), pack(b), 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ f16x8 split_tiles(f32x4 a, f32x4 b, f16x8& rest, f16 type) {
    typedef f16 v4 __attribute__((ext_vector_type(4)));
    const v4 ha = __builtin_convertvector(a, v4), hb = __builtin_convertvector(b, v4);
    rest = frag_tiles(a - __builtin_convertvector(ha, f32x4), b - __builtin_convertvector(hb, f32x4), type);
    return __builtin_shufflevector(ha, hb, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ f32x8 split_tiles(f32x4 a, f32x4 b, f32x8&, float type) { return frag_tiles(a, b, type); }
// Rows 4g+i and 16+4g+i of column c of a tile in LDS (rows `pitch` apart): the operand that
// goes with frag_tiles.
template <typename E>
__device__ __forceinline__ typename Elem<E>::Frag frag_columns(const typename Elem<E>::S* tile, int pitch, int g, int c) {
    if constexpr (sizeof(E) == 2) {
        const short* p = (const short*)tile + (4 * g + (c >> 2)) * pitch + 4 * (c & 3);
        const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p));
        const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 16 * pitch)));
        return __builtin_bit_cast(typename Elem<E>::Frag, __builtin_shufflevector(a, b, 0, 1, 2, 3));
    } else {
        f32x8 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            r[i] = tile[(4 * g + i) * pitch + c];
            r[4 + i] = tile[(16 + 4 * g + i) * pitch + c];
        }
        return r;
    }
}

// Over the four lanes of one column (g = 0 .. 3).
__device__ __forceinline__ float column_max(float x) {
    const mix::Halves a = mix::swap32(x, x);
    x = fmaxf(a.first, a.second);
    const mix::Halves b = mix::swap16(x, x);
    return fmaxf(b.first, b.second);
}
__device__ __forceinline__ float column_sum(float x) {
    const mix::Halves a = mix::swap32(x, x);
    x = a.first + a.second;
    const mix::Halves b = mix::swap16(x, x);
    return b.first + b.second;
}

// tanh(x) with a relative error of some 2^-23 for small x too, and (1 - tanh^2) / 4.  Below
// 0.7 the continued fraction x / (1 + x^2 / (3 + x^2 / (5 + x^2 / (7 + x^2 / 9)))), 2e-9 off there.
struct Tanh {
    float t, slope;
};
__device__ __forceinline__ Tanh fine_tanh(float x) {
    const float r = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * (2.0f * kLog2e)));
    const float q = x * x, d = 945.0f + q * (420.0f + 15.0f * q);
    float inv = __builtin_amdgcn_rcpf(d);
    inv = inv * (2.0f - d * inv);
    const float t = x * (945.0f + q * (105.0f + q)) * inv;
    const bool small = fabsf(x) < 0.7f;
    return Tanh{small ? t : 1.0f - 2.0f * r, small ? 0.25f - 0.25f * t * t : r - r * r};
}

// ROWS rows of DP elements from memory to LDS through registers, 16 bytes a thread at a time:
// rows that are none and columns behind D become 0.  The loads go through a buffer descriptor of
// the tile's rows, so a lane's part of the address is one number for all tiles.
template <typename E, int ROWS, int DP, int PITCH, int NT>
struct Stage {
    typedef typename Elem<E>::S S;
    static constexpr int PER = 16 / sizeof(E), CPR = DP / PER, N = (ROWS * CPR + NT - 1) / NT;
    static constexpr bool EVEN = NT % CPR == 0;         // a round of the threads is whole rows
    static constexpr int M = EVEN ? 1 : N;
    u32x4 r[N];
    u32 at[M], step, to[M];
    __device__ __forceinline__ void begin(int64_t stride, int64_t D, int tid) {
        step = EVEN ? (u32)(NT / CPR) * (u32)stride * sizeof(E) : 0;
#pragma unroll
        for (int i = 0; i < M; ++i) {
            const int e = i * NT + tid, row = e / CPR, col = e % CPR * PER;
            at[i] = e < ROWS * CPR && col < D ? (u32)(row * (u32)stride + col) * (u32)sizeof(E) : 0x80000000u;
            to[i] = row * PITCH + col;
        }
    }
    // `first`: row 0 of the tile; the `rows` of it that are there
    __device__ __forceinline__ void load(const S* first, int rows, int64_t stride, int64_t D) {
        const int n = min(rows, ROWS);
        const int bytes = n > 0 ? ((n - 1) * (int)stride + (int)D) * (int)sizeof(E) : 0;
        const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<S*>(first), 0, bytes, 0x00020000);
#pragma unroll
        for (int i = 0; i < N; ++i)
            r[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                 rsrc, EVEN ? at[0] + i * step : at[i % M], 0, 0));
    }
    __device__ __forceinline__ void store(S* lds, int tid) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (ROWS * CPR % NT == 0 || i * NT + tid < ROWS * CPR)
                *reinterpret_cast<u32x4*>(lds + (EVEN ? to[0] + i * (NT / CPR) * PITCH : to[i % M])) = r[i];
        }
    }
    // whether one of these elements is infinite or NaN
    __device__ __forceinline__ bool odd() const {
        bool any = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (sizeof(E) == 4) any |= (r[i][j] & 0x7f800000u) == 0x7f800000u;
                else {
                    constexpr u32 m = __is_same(E, __half) ? 0x7c00u : 0x7f80u;
                    any |= (r[i][j] & m) == m || (r[i][j] >> 16 & m) == m;
                }
            }
        }
        return any;
    }
    // ... and those set to 0
    __device__ __forceinline__ void clean() {
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (sizeof(E) == 4) {
                    if ((r[i][j] & 0x7f800000u) == 0x7f800000u) r[i][j] = 0;
                } else {
                    constexpr u32 m = __is_same(E, __half) ? 0x7c00u : 0x7f80u;
                    if ((r[i][j] & m) == m) r[i][j] &= 0xffff0000u;
                    if ((r[i][j] >> 16 & m) == m) r[i][j] &= 0xffffu;
                }
            }
        }
    }
};

// Pitches (elements) that spread the rows over the banks: a 16-byte read of 16 rows, and a
// transposed read of four rows of 32 bytes in each 16 lanes.
template <typename E, int DP> constexpr int row_pitch() { return DP + (sizeof(E) == 2 ? 8 : 4); }
template <typename E, int DP> constexpr int column_pitch() { return DP + (sizeof(E) == 2 ? 16 : 4); }

// What the tokens of a block of queries (or keys) may meet, by document ids.
struct IdRange {
    int lo, hi;                      // of the ids that are not negative; lo > hi if there is none
    bool pure;                       // one id alone, none negative
    __device__ __forceinline__ bool meets(const IdRange& o) const { return lo <= o.hi && o.lo <= hi; }
    __device__ __forceinline__ bool same(const IdRange& o) const { return pure && o.pure && lo == o.lo; }
};
__device__ __forceinline__ int id_tiles(int64_t N) { return ((int)N + kIdTile - 1) / kIdTile; }
__device__ __forceinline__ IdRange id_range(const AttnArgs& p, int64_t b, int tile) {
    const int32_t* s = p.id_stats + (b * id_tiles(p.N) + tile) * 3;
    return IdRange{s[0], s[1], s[2] != 0};
}
// Tokens first .. first+n-1 (first a multiple of 64, or all within one tile).
__device__ __forceinline__ IdRange id_block(const AttnArgs& p, int64_t b, int first, int n) {
    IdRange r = id_range(p, b, first / kIdTile);
    for (int t = first / kIdTile + 1; t * kIdTile < min(first + n, (int)p.N); ++t) {
        const IdRange o = id_range(p, b, t);
        r.pure = r.same(o);
        r.lo = min(r.lo, o.lo);
        r.hi = max(r.hi, o.hi);
    }
    return r;
}

// Which queries a workgroup takes: `id` without its key head.  In the order given, or, by length
// alone, the last rows first.
struct QueryBlock {
    int64_t b;
    int rep, tile;
    __device__ __forceinline__ QueryBlock(const AttnArgs& p, int id, int R, int tiles) {
        if (p.order) {
            const int o = p.order[id / R];
            rep = id % R, b = o / tiles, tile = o % tiles;
        } else {
            const int B = (int)p.B;
            b = id % B, rep = id / B % R, tile = tiles - 1 - id / B / R;
        }
    }
};

// The tiles of STEP tokens in [begin, end) whose ids meet `mine`, in order; all of them without
// ids.  64 tiles are looked at in one go, so every lane of the wave has to take part.
template <int STEP>
struct TileWalk {
    const AttnArgs& p;
    int64_t b;
    int end;
    IdRange mine;
    int window;                      // the 64 tiles of ids that `mask` tells of begin here
    uint64_t mask;
    __device__ __forceinline__ TileWalk(const AttnArgs& p, int64_t b, int end, IdRange mine)
        : p(p), b(b), end(end), mine(mine), window(-64), mask(0) {}
    __device__ __forceinline__ int next(int k) {       // k: a multiple of STEP
        if (!p.ids) return k;
        while (k < end) {
            const int t = k / kIdTile;
            if (t >= window + 64) {
                window = t;
                const int at = t + (threadIdx.x & 63);
                mask = __ballot(at < id_tiles(p.N) && id_range(p, b, at).meets(mine));
            }
            const uint64_t left = mask >> (t - window);
            if (left & 1) return k;
            k = (left ? t + __builtin_ctzll(left) : window + 64) * kIdTile;
        }
        return k;
    }
};

// What `splits` workgroups left of a row, joined: D floats each, and behind them the reference and the
// sum, `stride` apart.  Parts `from`, from + STEP, .. of the dimensions d .. d+3; U of them are under way at
// a time, as one after the other their latency is all that a row costs.
struct Joined {
    float top, total;
    f32x4 v;
    __device__ __forceinline__ void add(float t, float sum, f32x4 o) {
        const float to = fmaxf(top, t);
        const float mine = top == to ? 1.0f : __builtin_amdgcn_exp2f(top - to);
        const float its = t == to ? 1.0f : __builtin_amdgcn_exp2f(t - to);
        top = to;
        total = total * mine + sum * its;
        v = v * mine + o * its;
    }
};
template <int STEP, int U>
__device__ __forceinline__ Joined join_parts(const float* part, int from, int splits, int64_t D, int d) {
    const int64_t stride = D + 4;
    Joined j{kNegInf, 0.0f, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
    for (int s0 = from; s0 < splits; s0 += U * STEP) {
        f32x4 o[U], end[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float* q = part + min(s0 + u * STEP, splits - 1) * stride;
            o[u] = *reinterpret_cast<const f32x4*>(q + d);
            end[u] = *reinterpret_cast<const f32x4*>(q + D);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + u * STEP < splits) j.add(end[u][0], end[u][1], o[u]);
    }
    return j;
}

}  // namespace attn
}  // namespace flare
