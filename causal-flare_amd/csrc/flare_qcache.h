// flare_qcache.h -- a cache of keys and values held in 8 or 4 bits: its codes, and what they stand for.
//
// A row of D values (a token's key or value of one head) is cut into blocks of 32, the last of which may
// have 16.  A block has a scale of its own, 2^e, held as the byte e + 127, and its values are x = code 2^e
// with codes of 8 bits (e4m3, up to 448) or 4 bits (e2m1: 0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign; the value
// of the lower index in the lower half of a byte).  e is the least for which the block's largest value
// rounds to no more than the largest code: max |x| <= 464 2^e or 7 2^e.  Values are rounded to the nearest,
// ties to the even code; what is left beyond the largest code becomes it.  A block that holds an infinite
// value or a NaN has the scale byte 255, and all of it reads back as NaN.
//
// So a value that a cache holds is exact in bf16 (4 significant bits), and in fp16 where it was written
// from that: the least and the largest e are kept within what the writer's type has.  gfx950 converts two
// values with their scale in one instruction, at the rate of a product.  Off by, of normally distributed
// values (root of the mean square): 2.7% with 8 bits and 11.2% with 4 (11.5% if the largest value may not
// pass the largest code, or may reach the next power of 2).
#pragma once

#include "flare_attn.h"

namespace flare {
namespace qcache {

using attn::f32x8;
using attn::u32;
using attn::u32x2;
using attn::u32x4;
using mfma::bf16;
using mfma::bf16x8;
using mfma::f16;
using mfma::f16x8;

constexpr int kBlock = 32;
constexpr u32 kNoValue = 255;        // the scale of a block that is NaN

// most: the largest code; room: the mantissa of the largest value at a scale of 1, and power its
// exponent; lo, hi: exponents of scales, of values written from fp16 (narrow) and from wider types.
template <int BITS> struct Form;
template <> struct Form<8> {
    static constexpr float most = 448.0f;
    static constexpr u32 room = 0x680000;                 // 464 = 1.8125 2^8
    static constexpr int power = 8, lo = -117, hi = 119, narrow_lo = -15, narrow_hi = 7;
};
template <> struct Form<4> {
    static constexpr float most = 6.0f;
    static constexpr u32 room = 0x600000;                 // 7 = 1.75 2^2
    static constexpr int power = 2, lo = -125, hi = 125, narrow_lo = -23, narrow_hi = 13;
};

// The scale's byte of a block whose largest magnitude is `top`.
template <int BITS>
__device__ __forceinline__ u32 scale_of(float top, bool narrow) {
    typedef Form<BITS> F;
    const u32 bits = __builtin_bit_cast(u32, top);
    const int e = (int)((bits + (0x7fffffu - F::room)) >> 23) - 127 - F::power;      // one more behind `room`
    const int lo = narrow ? F::narrow_lo : F::lo, hi = narrow ? F::narrow_hi : F::hi;
    return bits >= 0x7f800000u ? kNoValue : (u32)(min(max(e, lo), hi) + 127);
}
__device__ __forceinline__ float scale_value(u32 byte) { return __builtin_bit_cast(float, byte << 23); }    // 255: infinite

// The largest magnitude of eight values; infinite for a NaN too.
__device__ __forceinline__ float top_of(const float (&v)[8]) {
    float m = 0.0f;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        m = fmaxf(m, fabsf(v[i]));
        odd |= v[i] != v[i];
    }
    return odd ? -kNegInf : m;
}

// Eight codes of eight values, the first in the lowest bits.
template <int BITS>
struct Codes {
    u32 w[BITS / 4];
};
template <int BITS>
__device__ __forceinline__ Codes<BITS> encode(const float (&v)[8], u32 byte) {
    Codes<BITS> r = {};
    if (byte == kNoValue) return r;
    const float scale = scale_value(byte), most = Form<BITS>::most * scale;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __builtin_amdgcn_fmed3f(v[i], -most, most);
    if constexpr (BITS == 4) {
        u32 w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
        r.w[0] = w;
    } else {
        typedef short s16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            s16x2 w = {0, 0};
            w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[4 * i], x[4 * i + 1], scale, false);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[4 * i + 2], x[4 * i + 3], scale, true);
            r.w[i] = __builtin_bit_cast(u32, w);
        }
    }
    return r;
}

// What eight codes stand for, as an operand (`type` says which).
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef f16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <int BITS>
__device__ __forceinline__ bf16x8 decode(const u32* w, float scale, bf16) {
    bf16x2 a, b, c, d;
    if constexpr (BITS == 4) {
        a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], scale, 0);
        b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], scale, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], scale, 2);
        d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], scale, 3);
    } else {
        a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], scale, false);
        b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], scale, true);
        c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], scale, false);
        d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], scale, true);
    }
    const u32x4 r = {__builtin_bit_cast(u32, a), __builtin_bit_cast(u32, b), __builtin_bit_cast(u32, c),
                     __builtin_bit_cast(u32, d)};
    return __builtin_bit_cast(bf16x8, r);
}
template <int BITS>
__device__ __forceinline__ f16x8 decode(const u32* w, float scale, f16) {
    f16x2 a, b, c, d;
    if constexpr (BITS == 4) {
        a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], scale, 0);
        b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], scale, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], scale, 2);
        d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], scale, 3);
    } else {
        a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[0], scale, false);
        b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[0], scale, true);
        c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[1], scale, false);
        d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[1], scale, true);
    }
    const u32x4 r = {__builtin_bit_cast(u32, a), __builtin_bit_cast(u32, b), __builtin_bit_cast(u32, c),
                     __builtin_bit_cast(u32, d)};
    return __builtin_bit_cast(f16x8, r);
}
// (through bf16, in which they are exact: the conversions to pairs of floats take three times as long)
template <int BITS>
__device__ __forceinline__ f32x8 decode(const u32* w, float scale, float) {
    const u32x4 h = __builtin_bit_cast(u32x4, decode<BITS>(w, scale, bf16{}));
    f32x8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[2 * i] = __builtin_bit_cast(float, h[i] << 16);
        r[2 * i + 1] = __builtin_bit_cast(float, h[i] & 0xffff0000u);
    }
    return r;
}

// Over the four lanes of a quad.
__device__ __forceinline__ float quad_max(float x) {
    const int a = __builtin_bit_cast(int, x);
    x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(a, 0xB1, 0xf, 0xf, true)));
    const int b = __builtin_bit_cast(int, x);
    return fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(b, 0x4E, 0xf, 0xf, true)));
}

// Eight elements of a row (on a 16-byte boundary) as floats.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    mix::load_row<T, 16 / sizeof(T)>(p, reinterpret_cast<float (&)[16 / sizeof(T)]>(v[0]));
    if constexpr (sizeof(T) == 4) mix::load_row<T, 4>(p + 4, reinterpret_cast<float (&)[4]>(v[4]));
}

// What the cache of `p` holds of each sequence, its new tokens included, as k and v [B, M, G, D] of `dtype`; rows
// behind that are left as they are.
int qcache_expand(const attn::AttnArgs& p, int dtype, int bits, void* k, void* v, hipStream_t stream);

__host__ __device__ __forceinline__ int64_t row_codes(int64_t D, int bits) { return D * bits / 8; }
__host__ __device__ __forceinline__ int64_t row_scales(int64_t D) { return (D + kBlock - 1) / kBlock; }

}  // namespace qcache
}  // namespace flare
