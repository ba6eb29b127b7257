// flare_rotary.hip -- rotary positions of queries and keys, and their gradients.
//
// Pair i of a head, (a, b), is turned by the angle position * frequency_i:
//   (a cos - b sin, a sin + b cos)
// and a gradient by the same angle the other way.  The pairs are (x_i, x_{i + R/2}), or (x_2i, x_2i+1)
// interleaved; dimensions from R on stay as they are.
//
// An angle matters to a whole turn only, so a frequency is taken as turns a token in 64 bits behind
// the point, the nearest: its product with a whole position, without the turns before the point, is exact
// however far the position, and is rounded to the nearest 2^-32 of a turn (0.7e-9 off).  Sine and cosine of
// what is left after the nearest quarter turn are their series to x^9 and x^10, below 2e-9 off at an
// eighth of a turn.
//
// Bytes bound all but small calls, 36 us for 168 MB (4.7 TB/s; a copy goes at 4.9); one token for 64 sequences takes 4,
// a launch and a chain of loads.
#include "flare_mix.h"

#include <math.h>

namespace flare {
namespace rotary {

using mix::ceil_div;

constexpr int kMostPairs = 128;
constexpr long double kTurns = 0x1p64L / 6.283185307179586476925286766559L;       // of a radian, in 2^-64 turns

struct Head {                        // a [B, N, heads, D] tensor: element strides
    const void* p;
    int64_t sb, sn, sh;
    void* out;                       // [B, N, heads, D]
};

struct Args {
    Head q, k;                       // k: no heads if NULL
    int64_t B, N;
    int H, G, D, R;
    const int32_t *positions, *lengths;      // [B, N], [B]
    int interleaved, inverse;
    int units, parts;                // of a token: vectors (pairs of vectors) of a head, threads that share the heads
    uint64_t turns[kMostPairs];      // a token, 64 bits behind the point
};

struct Turn {
    float c, s;
};
__device__ __forceinline__ Turn turn_of(int64_t position, uint64_t turns) {
    const uint32_t at = (uint32_t)(((uint64_t)position * turns + 0x80000000u) >> 32);
    const uint32_t quarter = (at + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(at - (quarter << 30)) * 1.46291807926715968105e-9f;      // 2 pi / 2^32
    const float q = x * x;
    float s = 1.0f / 362880.0f;
    s = s * q - 1.0f / 5040.0f;
    s = s * q + 1.0f / 120.0f;
    s = s * q - 1.0f / 6.0f;
    s = x + x * (q * s);
    float c = -1.0f / 3628800.0f;
    c = c * q + 1.0f / 40320.0f;
    c = c * q - 1.0f / 720.0f;
    c = c * q + 1.0f / 24.0f;
    c = c * q - 0.5f;
    c = 1.0f + q * c;
    const bool swap = quarter & 1;
    Turn t{swap ? s : c, swap ? c : s};
    if ((quarter + 1) & 2) t.c = -t.c;
    if (quarter & 2) t.s = -t.s;
    return t;
}

template <typename T, int V>
struct alignas(V * sizeof(T)) Vec {
    T v[V];
};

// Heads a thread turns, where there is work for more threads than the card takes at once: four vectors of loads
// under way.  us of 4 x 4096 tokens, 16 and 4 heads of 128, bf16: pairs of halves with 2, 4 and 8 heads 36, 41, 45;
// adjacent pairs with 2, 4 and 8 39, 31, 32 (a copy of these 168 MB takes 34, and repeated calls find part of their inputs
// in the last-level cache).  Stores that pass by that cache take 33, and what reads the result then takes that much
// longer.
constexpr int heads_of(bool interleaved) { return interleaved ? 4 : 2; }

// V: elements of a vector; 1: element by element, whatever the strides.
// A thread turns the same pairs of heads part, part + parts, ..: the angles are computed once for them.
template <typename T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(Args p) {
    constexpr int kBatch = heads_of(INTERLEAVED), PAIRS = INTERLEAVED && V > 1 ? V / 2 : V, VECS = INTERLEAVED && V > 1 ? 1 : 2;
    typedef Vec<T, V> W;
    const int per = p.units * p.parts, tokens = 256 / per;
    const int within = threadIdx.x % per, unit = within % p.units, part = within / p.units;
    const int64_t token = (int64_t)blockIdx.x * tokens + threadIdx.x / per;
    if ((int)threadIdx.x >= tokens * per || token >= p.B * p.N) return;
    const int64_t b = token / p.N, t = token % p.N;
    const int heads = p.H + p.G, turned = p.R / 2 / PAIRS;
    // of this thread's two vectors
    const bool turns = unit < turned;
    int first, second;
    if (!turns) first = second = p.R + (unit - turned) * V;
    else if (INTERLEAVED) first = unit * 2 * PAIRS, second = first + (V == 1 ? 1 : 0);
    else first = unit * V, second = first + p.R / 2;

    auto row = [&](int h) {
        return h < p.H ? (const T*)p.q.p + b * p.q.sb + t * p.q.sn + h * p.q.sh
                       : (const T*)p.k.p + b * p.k.sb + t * p.k.sn + (h - p.H) * p.k.sh;
    };
    auto to = [&](int h) {
        return h < p.H ? (T*)p.q.out + (token * p.H + h) * p.D : (T*)p.k.out + (token * p.G + (h - p.H)) * p.D;
    };
    Turn angle[PAIRS];
    if (turns) {
        const int64_t at = p.positions ? (int64_t)p.positions[token] : p.lengths ? (int64_t)p.lengths[b] + t : t;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            angle[i] = turn_of(at, p.turns[unit * PAIRS + i]);
            if (p.inverse) angle[i].s = -angle[i].s;
        }
    }
    for (int h0 = part; h0 < heads; h0 += kBatch * p.parts) {
        W a[kBatch], c[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const T* from = row(min(h0 + i * p.parts, heads - 1));
            a[i] = *reinterpret_cast<const W*>(from + first);
            if (VECS == 2 && turns) c[i] = *reinterpret_cast<const W*>(from + second);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int h = h0 + i * p.parts;
            if (h >= heads) break;
            T* out = to(h);
            if (!turns) {
                *reinterpret_cast<W*>(out + first) = a[i];
                continue;
            }
#pragma unroll
            for (int e = 0; e < PAIRS; ++e) {
                T& u = VECS == 1 ? a[i].v[2 * e] : a[i].v[e];
                T& w = VECS == 1 ? a[i].v[2 * e + 1] : c[i].v[e];
                const float x = to_f32(u), y = to_f32(w);
                u = from_f32<T>(x * angle[e].c - y * angle[e].s);
                w = from_f32<T>(x * angle[e].s + y * angle[e].c);
            }
            *reinterpret_cast<W*>(out + first) = a[i];
            if (VECS == 2) *reinterpret_cast<W*>(out + second) = c[i];
        }
    }
}

template <typename T, int V>
static int launch(Args p, hipStream_t stream) {
    const int heads = p.H + p.G;
    const int pairs = p.interleaved && V > 1 ? V / 2 : V;
    p.units = p.R / 2 / pairs + (p.D - p.R) / V;
    // a head a thread where that leaves no more than the card takes at once
    const int64_t all = p.B * p.N * heads * p.units;
    const int each = heads_of(p.interleaved), want = all <= 256 * 1024 ? heads : (heads + each - 1) / each;
    p.parts = 256 / p.units < want ? 256 / p.units : want;
    const int64_t blocks = ceil_div(p.B * p.N, 256 / (p.units * p.parts));
    if (blocks > mix::kMostBlocks) {
        set_error("flare_rotary: too large");
        return FLARE_ERR_INVALID;
    }
    if (p.interleaved) rotary_kernel<T, V, true><<<dim3((unsigned)blocks), 256, 0, stream>>>(p);
    else rotary_kernel<T, V, false><<<dim3((unsigned)blocks), 256, 0, stream>>>(p);
    return check_launch("rotary");
}

// Vectors of V elements: where rows begin on their boundary and neither a pair's halves nor the
// dimensions that stay cut one.
static bool vectors(const Args& p, int V, int size) {
    const int64_t bytes = (int64_t)V * size;
    const int run = p.interleaved ? p.R : p.R / 2;
    if (run % V || p.D % V) return false;
    for (const Head* h : {&p.q, &p.k}) {
        if (!h->p) continue;
        if ((uintptr_t)h->p % bytes || (uintptr_t)h->out % bytes || h->sb % V || h->sn % V || h->sh % V) return false;
    }
    return true;
}

template <typename T>
static int launch_type(const Args& p, hipStream_t stream) {
    constexpr int size = sizeof(T);
    if (vectors(p, 16 / size, size)) return launch<T, 16 / size>(p, stream);
    if (vectors(p, 8 / size, size)) return launch<T, 8 / size>(p, stream);
    return launch<T, 1>(p, stream);
}

}  // namespace rotary
}  // namespace flare

using namespace flare;
using namespace flare::rotary;

extern "C" int flare_rotary(const void* q, const void* k, const int64_t* strides, int dtype, int64_t B, int64_t N,
                            int64_t H, int64_t G, int64_t D, int64_t R, const double* frequencies,
                            const int32_t* positions, const int32_t* lengths, int interleaved, int inverse, void* q_out,
                            void* k_out, void* stream) {
    FLARE_REQUIRE(q && strides && frequencies && q_out && (!k || k_out), "flare_rotary: null pointer");
    FLARE_REQUIRE(mix::known_dtype(dtype), "flare_rotary: unknown dtype %d", dtype);
    FLARE_REQUIRE(B >= 1 && N >= 1 && H >= 1 && (!k || G >= 1), "flare_rotary: sizes must be positive");
    FLARE_REQUIRE(R >= 2 && R % 2 == 0 && R <= D && D <= 2 * kMostPairs,
                  "flare_rotary: %lld of %lld dimensions; an even number, up to all of 256", (long long)R, (long long)D);
    FLARE_REQUIRE(!(positions && lengths), "flare_rotary: positions exclude lengths");
    FLARE_REQUIRE(B <= (1 << 24) && N <= (1 << 30) && H <= 65535 && G <= 65535, "flare_rotary: too large");
    Args p = {};
    p.q = {q, strides[0], strides[1], strides[2], q_out};
    p.k = {k, strides[3], strides[4], strides[5], k_out};
    p.B = B, p.N = N, p.H = (int)H, p.G = k ? (int)G : 0, p.D = (int)D, p.R = (int)R;
    p.positions = positions, p.lengths = lengths, p.interleaved = interleaved, p.inverse = inverse;
    for (int i = 0; i < R / 2; ++i) {
        const long double f = frequencies[i];
        if (f >= 0.0L && f < 6.0L) {
            p.turns[i] = (uint64_t)(f * kTurns + 0.5L);     // below 0.96 2^64; roundl would add 0.6 us to a call of 64 pairs
            continue;
        }
        FLARE_REQUIRE(isfinite(frequencies[i]), "flare_rotary: frequency %d is not finite", i);
        const long double turns = f * (kTurns * 0x1p-64L), part = turns - floorl(turns);     // in [0, 1]: 1 only by rounding
        p.turns[i] = part < 1.0L ? (uint64_t)roundl(ldexpl(part, 64)) : 0;      // at most 2^64 - 1, which 64 bits hold
    }
    return FLARE_BY_DTYPE(dtype, launch_type, (p, (hipStream_t)stream));
}
