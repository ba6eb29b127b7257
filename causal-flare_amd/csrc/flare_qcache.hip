// flare_qcache.hip -- writing prompts to a cache of 8 or 4 bits, and reading it back.
//
// Bytes bound both.  A quad of lanes owns a block of 32 values, eight a lane: their largest magnitude takes two
// exchanges within the quad.  A thread takes a key and its value, so that what it computes of addresses counts for
// both and two loads are under way.  us, keys and values in threads of their own and together, bf16: 4 x 4096 tokens, 16
// heads of 128, written in 4 bits 43, 38 (4.5 TB/s; a copy goes at 4.9), in 8 bits 45, 43; read 30, 28 and 39, 36 (the
// codes in part from the last-level cache); 16 x 8192 tokens, 4 heads of 80, 4 bits, written 56, 51, read 47, 36.
#include "flare_internal.h"
#include "flare_qcache.h"

namespace flare {
namespace qcache {

using attn::ceil_div;
using attn::clamp_to;
using attn::Rows;

struct Cache {
    uint8_t *k, *v, *k_scale, *v_scale;
};

// blockIdx.y: a sequence; x: quads of its rows, each of a key and of its value.
template <typename T, int BITS>
__global__ __launch_bounds__(256) void qcache_write_kernel(Rows k, Rows v, const int32_t* lengths, const int32_t* fresh,
                                                           unsigned N, int64_t M, unsigned G, unsigned D, Cache to) {
    const unsigned NB = (D + kBlock - 1) / kBlock, b = blockIdx.y;
    const unsigned id = blockIdx.x * 256 + threadIdx.x, quad = id >> 2, block = quad % NB, g = quad / NB % G;
    const unsigned t = quad / NB / G, d = block * kBlock + (id & 3) * 8;
    const int64_t off = lengths[b], n = fresh ? clamp_to(fresh[b], N) : N;
    if (off < 0 || off + n > M || t >= n) return;                       // a quad at a time
    float x[2][8] = {};
    if (d < D) {
        load8((const T*)k.p + b * k.sb + t * k.sn + g * k.sh + d, x[0]);
        load8((const T*)v.p + b * v.sb + t * v.sn + g * v.sh + d, x[1]);
    }
    const int64_t row = ((int64_t)b * M + off + t) * G + g;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const u32 byte = scale_of<BITS>(quad_max(top_of(x[i])), __is_same(T, __half));
        if (d < D) *reinterpret_cast<Codes<BITS>*>((i ? to.v : to.k) + row * (D * BITS / 8) + d * BITS / 8) = encode<BITS>(x[i], byte);
        if ((id & 3) == 0) (i ? to.v_scale : to.k_scale)[row * NB + block] = (uint8_t)byte;
    }
}

// Rows first[b] .. first[b] + N - 1 of each sequence; 0 outside of it.  Eight values of a key and of its value a
// thread.  With `lengths` those that a sequence of so many tokens and `fresh` (or all N_new) new ones holds, and no others.
template <typename T, int BITS>
__global__ __launch_bounds__(256) void qcache_read_kernel(Cache from, const int32_t* first, unsigned N, int64_t M, unsigned G,
                                                          unsigned D, const int32_t* lengths, const int32_t* fresh,
                                                          int64_t N_new, T* k, T* v) {
    const unsigned per = D / 8, NB = (D + kBlock - 1) / kBlock, b = blockIdx.y;
    const unsigned id = blockIdx.x * 256 + threadIdx.x, d = id % per * 8, g = id / per % G, t = id / per / G;
    if (t >= N) return;
    if (lengths) {
        const int64_t off = lengths[b], n = fresh ? clamp_to(fresh[b], N_new) : N_new;
        if (off < 0 || t >= off + n) return;
    }
    const int64_t at = (first ? (int64_t)first[b] : 0) + t;
    f32x8 x[2] = {};
    if (at >= 0 && at < M) {
        const int64_t row = ((int64_t)b * M + at) * G + g, codes = row * (D * BITS / 8) + d * BITS / 8, scale = row * NB + d / kBlock;
        const Codes<BITS> c = *reinterpret_cast<const Codes<BITS>*>(from.k + codes);
        const Codes<BITS> w = *reinterpret_cast<const Codes<BITS>*>(from.v + codes);
        x[0] = decode<BITS>(c.w, scale_value(from.k_scale[scale]), float{});
        x[1] = decode<BITS>(w.w, scale_value(from.v_scale[scale]), float{});
    }
    const int64_t to = (((int64_t)b * N + t) * G + g) * D + d;
    constexpr int PER = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < 8; i += PER) {
            float o[PER];
#pragma unroll
            for (int e = 0; e < PER; ++e) o[e] = x[j][i + e];
            mix::store_row<T, PER>((j ? v : k) + to + i, o);
        }
    }
}

template <typename T>
static int write_type(const Rows& k, const Rows& v, int bits, const int32_t* lengths, const int32_t* fresh, int64_t B,
                      int64_t N, int64_t M, int64_t G, int64_t D, const Cache& to, hipStream_t stream) {
    const dim3 grid((unsigned)ceil_div(N * G * row_scales(D) * 4, 256), (unsigned)B);
    const auto kernel = bits == 8 ? qcache_write_kernel<T, 8> : qcache_write_kernel<T, 4>;
    kernel<<<grid, 256, 0, stream>>>(k, v, lengths, fresh, (unsigned)N, M, (unsigned)G, (unsigned)D, to);
    return check_launch("qcache_write");
}
template <typename T>
static int read_type(const Cache& from, int bits, const int32_t* first, int64_t B, int64_t N, int64_t M, int64_t G, int64_t D,
                     const int32_t* lengths, const int32_t* fresh, int64_t N_new, void* k, void* v, hipStream_t stream) {
    const dim3 grid((unsigned)ceil_div(N * G * D / 8, 256), (unsigned)B);
    const auto kernel = bits == 8 ? qcache_read_kernel<T, 8> : qcache_read_kernel<T, 4>;
    kernel<<<grid, 256, 0, stream>>>(from, first, (unsigned)N, M, (unsigned)G, (unsigned)D, lengths, fresh, N_new,
                                      (T*)k, (T*)v);
    return check_launch("qcache_read");
}

int qcache_expand(const attn::AttnArgs& p, int dtype, int bits, void* k, void* v, hipStream_t stream) {
    const Cache from = {(uint8_t*)p.k.p, (uint8_t*)p.v.p, p.k_scale, p.v_scale};
    return FLARE_BY_DTYPE(dtype, read_type, (from, bits, nullptr, p.B, p.M, p.M, p.G, p.D, p.lengths, p.fresh, p.N, k, v, stream));
}

}  // namespace qcache
}  // namespace flare

using namespace flare;
using namespace flare::qcache;

#define QCACHE_REQUIRE_SIZES(name)                                                                                     \
    FLARE_REQUIRE(attn::known_dtype(dtype), name ": unknown dtype %d", dtype);                                         \
    FLARE_REQUIRE(bits == 4 || bits == 8, name ": %d bits; 4 or 8", bits);                                             \
    FLARE_REQUIRE(B >= 1 && N >= 1 && M >= 1 && G >= 1, name ": sizes must be positive");                              \
    FLARE_REQUIRE(D >= 16 && D <= 128 && D % 16 == 0, name ": head dimension %lld is not a multiple of 16 up to 128",  \
                  (long long)D);                                                                                       \
    FLARE_REQUIRE(B <= 65535 && N <= (1 << 30) && M <= (1 << 30) && G <= 65535 && N * G <= (1 << 27), name ": too large")

extern "C" int flare_qcache_write(const void* k, const void* v, const int64_t* strides, int dtype, int bits, int64_t B,
                                  int64_t N, int64_t M, int64_t G, int64_t D, const int32_t* lengths,
                                  const int32_t* new_lengths, void* k_cache, void* k_scale, void* v_cache, void* v_scale,
                                  void* stream) {
    FLARE_REQUIRE(k && v && strides && lengths && k_cache && k_scale && v_cache && v_scale,
                  "flare_qcache_write: null pointer");
    QCACHE_REQUIRE_SIZES("flare_qcache_write");
    const Rows kr = {k, strides[0], strides[1], strides[2]}, vr = {v, strides[3], strides[4], strides[5]};
    FLARE_REQUIRE(attn::aligned(kr, dtype) && attn::aligned(vr, dtype) && (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0,
                  "flare_qcache_write: rows must be 16-byte aligned and less than 2^22 elements apart");
    const Cache to = {(uint8_t*)k_cache, (uint8_t*)v_cache, (uint8_t*)k_scale, (uint8_t*)v_scale};
    return FLARE_BY_DTYPE(dtype, write_type, (kr, vr, bits, lengths, new_lengths, B, N, M, G, D, to, (hipStream_t)stream));
}

extern "C" int flare_qcache_read(const void* k_cache, const void* k_scale, const void* v_cache, const void* v_scale, int dtype,
                                 int bits, int64_t B, int64_t N, int64_t M, int64_t G, int64_t D, const int32_t* first,
                                 void* k, void* v, void* stream) {
    FLARE_REQUIRE(k && v && k_cache && k_scale && v_cache && v_scale, "flare_qcache_read: null pointer");
    QCACHE_REQUIRE_SIZES("flare_qcache_read");
    FLARE_REQUIRE((((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)k | (uintptr_t)v) & 15) == 0,
                  "flare_qcache_read: tensors must be 16-byte aligned");
    const Cache from = {(uint8_t*)k_cache, (uint8_t*)v_cache, (uint8_t*)k_scale, (uint8_t*)v_scale};
    return FLARE_BY_DTYPE(dtype, read_type, (from, bits, first, B, N, M, G, D, nullptr, nullptr, 0, k, v, (hipStream_t)stream));
}
