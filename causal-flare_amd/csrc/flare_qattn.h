// flare_qattn.h -- softmax attention of one or a few new tokens a sequence over a cache of 8 or 4 bits.
//
// The cache's bytes bound it, and behind them the instructions that turn codes into operands.  A wave takes
// TK keys at a time, their codes loaded while those before are computed.  K's codes go straight into the A
// operand of S^T = K Q^T: of each 16 keys lane (g, c) holds key c's dimensions 8 DK g .. 8 DK (g + 1) - 1,
// DK = dimensions / 32, whose DK eights are the contraction indices 8g .. 8g+7 of DK products, and Q is laid
// out the same.  V's codes become 16-bit values in a stretch of LDS of the wave's own, to be read transposed.
// There the columns stand by eights: the first eight of every block of 32, then the second, and so on, so that
// the lanes' writes lie side by side.  The columns of S^T are rows (token, head) of the heads that share the
// keys, the heads of one token next to each other; a wave owns RT tiles of 16.
//
// What the cache holds is exact in bf16, and in fp16 where it was written from that.  fp16 queries see values of
// wider types rounded, infinite beyond fp16's range.  Such values stand before the call's own tokens, where every row
// sees them: the weights of 0 of keys that a row may not see meet values that are finite, or of blocks that are NaN.
// Weights of 16-bit queries are rounded to their type for the product with V, as the matrix instructions take them (sums of
// weights, maxima and what is joined are fp32): y is 1.9e-3 to 2.1e-3 off in bf16, where rounding y alone leaves 1.7e-3.
// fp32 queries and weights enter as three bf16 parts, 24 bits: three products for each of the others', and registers
// for two waves a SIMD, 90 us for 64 sequences of 8192 tokens where bf16 queries take 61 (4 key heads of 128, 4 bits, 16
// heads, 285 MB).
//
// The keys of a sequence are split over `splits` workgroups of four waves by its true length; qattn_join adds
// up what they leave.  A workgroup's waves are shares of one head's keys, or heads that lie side by side.  Up to 16 new
// keys and values a sequence are quantised by the workgroups whose share they are in, each put into the cache by one of
// them; qcache_write puts more there first.
//
// 64 sequences of up to 8192 tokens, 4 key heads of 128, 4 bits, 250 MB: 59 us and 6 for the joining, 66 a call (a copy
// of these bytes takes 51).  The same loads without the rest take 63 a call, so that 46% of the vector issue slots and
// 12% of the matrix pipe's cycles lie behind them, and two tiles under way at a time gained nothing (66, 65).  In 8 bits,
// 484 MB, 102.  Rows of 64 bytes lie four to a token: heads of the same tokens on different XCDs took 85 for the loads.
// Buffer loads whose size the compiler held in a vector register took a loop each, 10 us of the 66.
#pragma once

#include "flare_qcache.h"

namespace flare {
namespace attn {

using qcache::Codes;
using qcache::kBlock;
using qcache::kNoValue;

constexpr float kRowsSlack = 8.0f;   // log2 of the largest weight before the reference moves

// The type that codes are turned into, and the parts of a query or weight.
template <typename E> struct Held {
    typedef E Type;
    static constexpr int parts = 1;
};
template <> struct Held<float> {
    typedef __hip_bfloat16 Type;
    static constexpr int parts = 3;
};

template <int DP>
struct RowsLds {
    static constexpr int P = DP + 16;                                              // elements, as column_pitch
    static constexpr size_t v_bytes = 2 * 32 * P;                                  // of a wave
    static constexpr size_t o_bytes = sizeof(float) * 16 * (DP + 2);               // of a wave, after the loop
    static constexpr size_t bytes = 4 * (v_bytes > o_bytes ? v_bytes : o_bytes);
    // and behind that codes and scales of `tokens` new keys and values of each of `heads` heads
    static constexpr size_t row_words(int bits) { return 4 * bits + 4; }
    static size_t all(int64_t heads, int64_t tokens, int bits) { return bytes + heads * 2 * tokens * row_words(bits) * 4; }
};

// x as three parts of 8 bits that add up to it; an infinite value or a NaN is the first alone.
__device__ __forceinline__ void three_parts(float x, bf16& a, bf16& b, bf16& c) {
    const u32 u = __builtin_bit_cast(u32, x);
    const bool odd = (u & 0x7f800000u) == 0x7f800000u;
    const float hi = __builtin_bit_cast(float, u & 0xffff0000u), rest = x - hi;
    const float mid = __builtin_bit_cast(float, __builtin_bit_cast(u32, rest) & 0xffff0000u);
    a = odd ? (bf16)x : (bf16)hi;
    b = odd ? (bf16)0.0f : (bf16)mid;
    c = odd ? (bf16)0.0f : (bf16)(rest - mid);
}

// W dwords from `offset` bytes of a buffer, 0 where that lies behind its end.
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer_of(const uint8_t* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, bytes, 0x00020000);
}
template <int W>
__device__ __forceinline__ void load_words(Buffer from, u32 offset, u32* to) {
    if constexpr (W >= 4) {
        const u32x4 r = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, offset, 0, 0));
#pragma unroll
        for (int i = 0; i < 4; ++i) to[i] = r[i];
        if constexpr (W > 4) load_words<W - 4>(from, offset + 16, to + 4);
    } else if constexpr (W == 3) {
        typedef u32 u32x3 __attribute__((ext_vector_type(3)));
        const u32x3 r = __builtin_bit_cast(u32x3, __builtin_amdgcn_raw_buffer_load_b96(from, offset, 0, 0));
        to[0] = r[0], to[1] = r[1], to[2] = r[2];
    } else if constexpr (W == 2) {
        const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(from, offset, 0, 0));
        to[0] = r[0], to[1] = r[1];
    } else {
        to[0] = __builtin_bit_cast(u32, __builtin_amdgcn_raw_buffer_load_b32(from, offset, 0, 0));
    }
}
constexpr u32 kNowhere = 0x80000000u;        // an offset behind every buffer's end

// Waves a SIMD: as many as the registers of a tile of scores, its codes and the sums leave.
constexpr int rows_waves(int size, int bits, int tiles) { return tiles == 2 || size == 4 ? 2 : bits == 4 ? 4 : 3; }

template <typename E, int BITS, int DP, int CAP, int RT>
__global__ __launch_bounds__(256, rows_waves(sizeof(E), BITS, RT)) void qattn_rows_kernel(AttnArgs p) {
    typedef typename Elem<E>::S S;
    typedef typename Held<E>::Type HE;                 // what the products take
    typedef typename Elem<HE>::S HS;
    typedef typename Elem<HE>::Frag Frag;
    using Lds = RowsLds<DP>;
    constexpr int PARTS = Held<E>::parts;
    constexpr int DK = DP / 32, DT = DP / 16, NB = DP / kBlock, P = Lds::P;
    constexpr int TK = 32, NM = TK / 16, W8 = BITS / 4;                                  // W8: words of eight codes
    constexpr int NSC = DK == 3 ? 3 : 1;               // blocks that a lane's dimensions of K may lie in
    constexpr int NV = (TK * NB + 63) / 64;            // blocks of V a lane takes
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, c = lane & 15;
    const unsigned D = (unsigned)p.D, G = (unsigned)p.G, H = (unsigned)p.H, N = (unsigned)p.N, splits = (unsigned)p.splits;
    const unsigned R = H / G, rows = R * N, groups = (rows + 16 * RT - 1) / (16 * RT);
    // of the workgroup's waves, and of this one
    const unsigned heads = (unsigned)p.row_splits, shares = 4 / heads, head = wave % heads, part = wave / heads, sets = G / heads;
    // workgroups of the same tokens are 8 apart: one XCD, as their rows share lines of its L2
    const unsigned kvh0 = blockIdx.x / 8 % sets * heads, kvh = kvh0 + head, unit = blockIdx.x / (8 * sets) * 8 + blockIdx.x % 8;
    const unsigned split = unit % splits, group = unit / splits % groups, b = unit / (splits * groups);
    if (b >= (unsigned)p.B) return;
    const bool fused = p.k_new != nullptr;             // the new keys and values are not in the cache yet
    const int off = p.lengths[b], fresh = p.fresh ? min(max(p.fresh[b], 0), (int)N) : (int)N;
    S* y = (S*)p.y + (int64_t)b * N * H * D;
    if (off < 0 || (int64_t)off + fresh > p.M) {
        // an idle sequence, or a full cache
        if (splits == 1) {
            for (unsigned i = lane + 64 * part; i < 16 * RT * D; i += 64 * shares) {
                const unsigned r = group * 16 * RT + i / D;
                if (r < rows) y[((int64_t)(r / R) * H + kvh * R + r % R) * D + i % D] = (S)(off < 0 ? 0.0f : __builtin_nanf(""));
            }
        }
        return;
    }
    const int n = off + fresh, prefix = p.prefix ? min(max(p.prefix[b], 0), n) : 0;
    // the tokens whose rows these are, and the keys that the last of them sees
    const int token0 = (int)(group * 16 * RT / R), token1 = min((int)min((group * 16 * RT + 16 * RT - 1) / R, N), fresh - 1);
    const int seen = token0 < fresh ? min(n, max(off + token1 + 1, prefix)) : 0;
    const int step = (int)shares * TK;
    const unsigned share = ((unsigned)seen + splits - 1) / splits;
    const int per = (int)((share + step - 1) / step * step);
    const int first = (int)min((int64_t)split * per, (int64_t)seen), last = (int)min((int64_t)first + per, (int64_t)seen);
    const int held = fused ? min(last, off) : last;            // what of it memory holds
    const unsigned codes = D * BITS / 8, scales = (D + kBlock - 1) / kBlock;
    const unsigned stride = G * codes, scale_stride = G * scales;
    const int64_t row0 = (int64_t)b * p.M * G + kvh;
    const uint8_t* kc = (const uint8_t*)p.k.p + row0 * codes;
    const uint8_t* vc = (const uint8_t*)p.v.p + row0 * codes;
    const uint8_t* ksc = p.k_scale + row0 * scales;
    const uint8_t* vsc = p.v_scale + row0 * scales;

    // the new keys and values of this share: a quad of lanes a block.  A token goes into the cache from the group that its
    // last row is in, as that sees it.
    constexpr unsigned RW = Lds::row_words(BITS);
    u32* fresh_rows = (u32*)(smem + Lds::bytes);
    auto fresh_row = [&](unsigned head, unsigned value, unsigned token) {
        return fresh_rows + ((head * 2 + value) * N + token) * RW;       // codes, and the scales of four blocks
    };
    if (fused && last > max(first, off)) {
        const unsigned begin = max(first, off) - off, count = last - max(first, off);
        for (unsigned i = tid; i < heads * count * 8 * NB; i += 256) {
            const unsigned block = i / 4 % NB, value = i / (4 * NB) % 2, t = begin + i / (8 * NB) % count;
            const unsigned at = i / (8 * NB) / count, d = block * kBlock + (i & 3) * 8;
            const S* from = value ? (const S*)p.v_new + b * p.vn_sb + t * p.vn_sn + (kvh0 + at) * p.vn_sg
                                  : (const S*)p.k_new + b * p.kn_sb + t * p.kn_sn + (kvh0 + at) * p.kn_sg;
            float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
            if (d < D) qcache::load8(reinterpret_cast<const E*>(from) + d, x);
            const u32 byte = qcache::scale_of<BITS>(qcache::quad_max(qcache::top_of(x)), __is_same(E, __half));
            const Codes<BITS> w = qcache::encode<BITS>(x, byte);
            u32* to = fresh_row(at, value, t);
#pragma unroll
            for (int j = 0; j < W8; ++j) to[d / 8 * W8 + j] = w.w[j];
            if ((i & 3) == 0) to[4 * BITS + block] = byte;
            if ((t * R + R - 1) / (16 * RT) == group && d < D) {
                const int64_t row = ((int64_t)b * p.M + off + t) * G + kvh0 + at;
                *reinterpret_cast<Codes<BITS>*>((uint8_t*)(value ? p.v.p : p.k.p) + row * codes + d * BITS / 8) = w;
                if ((i & 3) == 0) (value ? p.v_scale : p.k_scale)[row * scales + block] = (uint8_t)byte;
            }
        }
        __syncthreads();
    }

    HS* vt = (HS*)(smem + wave * Lds::v_bytes);
    const bool full = D == DP;
    u32 kw[NM][DK * W8], kb[NM][NSC];                  // codes and scales of the tile that is next
    u32 vw[NV][BITS], vb[NV];
    // key and block of V of this lane's unit i: keys 0, 2, 1, 3 follow each other, as rows two apart
    // lie half the banks apart
    auto unit_key = [&](int i) {
        const int t = (i * 64 + lane) / NB;
        return (t & ~3) | (t & 1) << 1 | (t >> 1 & 1);
    };
    auto unit_block = [&](int i) { return (i * 64 + lane) % NB; };
    auto unit_there = [&](int i) { return TK * NB % 64 == 0 || i * 64 + lane < TK * NB; };
    // a lane's offsets within a tile
    u32 k_at[DK], ks_at[NSC], v_at[NV], vs_at[NV];
#pragma unroll
    for (int kk = 0; kk < DK; ++kk) {
        const unsigned d = 8 * (DK * g + kk);
        k_at[kk] = d < D ? c * stride + d * BITS / 8 : kNowhere;
    }
#pragma unroll
    for (int i = 0; i < NSC; ++i) {
        const unsigned block = 8 * (DK * g + i) / kBlock;
        ks_at[i] = block < scales ? c * scale_stride + block : kNowhere;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const unsigned block = unit_block(i);
        const bool there = unit_there(i) && block < scales;
        v_at[i] = there ? unit_key(i) * stride + block * (4 * BITS) : kNowhere;
        vs_at[i] = there ? unit_key(i) * scale_stride + block : kNowhere;
    }
    // a last block of V may have half the values
    bool half[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) half[i] = (unsigned)(unit_block(i) + 1) * kBlock > D;
    auto fetch = [&](int k0) {
        // (as scalars: a buffer whose size the compiler holds in a vector register costs a loop a load)
        const int there = __builtin_amdgcn_readfirstlane(min(max(held - k0, 0), TK));
        const int64_t at = k0;
        const int bytes = there ? (there - 1) * (int)stride + (int)codes : 0;
        const int sbytes = there ? (there - 1) * (int)scale_stride + (int)scales : 0;
        const Buffer kr = buffer_of(kc + at * stride, bytes), vr = buffer_of(vc + at * stride, bytes);
        const Buffer kr_s = buffer_of(ksc + at * scale_stride, sbytes), vr_s = buffer_of(vsc + at * scale_stride, sbytes);
#pragma unroll
        for (int m = 0; m < NM; ++m) {
            if (full) {
                load_words<DK * W8>(kr, k_at[0] + 16 * m * stride, kw[m]);
            } else {
#pragma unroll
                for (int kk = 0; kk < DK; ++kk) load_words<W8>(kr, k_at[kk] + 16 * m * stride, &kw[m][kk * W8]);
            }
#pragma unroll
            for (int i = 0; i < NSC; ++i)
                kb[m][i] = (u32)(uint8_t)__builtin_amdgcn_raw_buffer_load_b8(kr_s, ks_at[i] + 16 * m * scale_stride, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (full) {
                load_words<BITS>(vr, v_at[i], vw[i]);
            } else {
                load_words<BITS / 2>(vr, v_at[i], vw[i]);
                load_words<BITS / 2>(vr, half[i] ? kNowhere : v_at[i] + 2 * BITS, vw[i] + BITS / 2);
            }
            vb[i] = (u32)(uint8_t)__builtin_amdgcn_raw_buffer_load_b8(vr_s, vs_at[i], 0, 0);
        }
    };
    // the new tokens' codes, for the lanes that take their place
    auto insert = [&](int k0) {
#pragma unroll
        for (int m = 0; m < NM; ++m) {
            const int j = k0 + 16 * m + c;
            if (j < off || j >= last) continue;
            const u32* from = fresh_row(head, 0, j - off);
#pragma unroll
            for (int i = 0; i < DK * W8; ++i) kw[m][i] = from[DK * W8 * g + i];
#pragma unroll
            for (int i = 0; i < NSC; ++i) kb[m][i] = from[4 * BITS + 8 * (DK * g + i) / kBlock];
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = k0 + unit_key(i);
            if (!unit_there(i) || j < off || j >= last) continue;
            const u32* from = fresh_row(head, 1, j - off);
#pragma unroll
            for (int w = 0; w < BITS; ++w) vw[i][w] = from[unit_block(i) * BITS + w];
            vb[i] = from[4 * BITS + unit_block(i)];
        }
    };
    const int begin = first + (int)part * TK;
    if (begin < last) fetch(begin);

    Frag qf[RT][PARTS][DK];
    float slope2[RT];
    int lim[RT], pos[RT];                              // of this lane's rows: the keys it sees are below, and its place
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const unsigned r = group * 16 * RT + 16 * t + c, token = r / R, h = kvh * R + r % R;
        const bool live = r < rows && (int)token < fresh;
        pos[t] = off + (int)token;
        lim[t] = live ? min(n, max(pos[t] + 1, prefix)) : 0;
        slope2[t] = p.slopes && live ? p.slopes[h] * kLog2e : 0.0f;
#pragma unroll
        for (int kk = 0; kk < DK; ++kk) {
            const unsigned d = 8 * (DK * g + kk);
#pragma unroll
            for (int i = 0; i < PARTS; ++i) qf[t][i][kk] = Frag{};
            if (!live || d >= D) continue;
            const S* from = (const S*)p.q.p + b * p.q.sb + token * p.q.sn + h * p.q.sh + d;
            if constexpr (PARTS == 1) {
                qf[t][0][kk] = frag_rows<E>(from);
            } else {
                const f32x8 x = frag_rows<E>(from);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    bf16 u, v, w;
                    three_parts(x[e], u, v, w);
                    qf[t][0][kk][e] = u, qf[t][PARTS / 2][kk][e] = v, qf[t][PARTS - 1][kk][e] = w;
                }
            }
        }
    }
    const float scale2 = p.scale * kLog2e, cap2 = p.cap * kLog2e, to_tanh = CAP ? p.scale / p.cap : 0.0f;
    const float into_cap = 2.0f * kLog2e * to_tanh;
    f32x4 acc[RT][DT];
    float top[RT], sum[RT];
    u32 lost[RT];                                      // blocks of V of which it sees one that is NaN, in tiles not seen whole
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        top[t] = kNegInf, sum[t] = 0.0f, lost[t] = 0;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[t][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    for (int k0 = begin; k0 < last; k0 += step) {
        if (fused && off < k0 + TK) insert(k0);
        f32x4 s[RT][NM];
#pragma unroll
        for (int m = 0; m < NM; ++m) {
#pragma unroll
            for (int t = 0; t < RT; ++t) s[t][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int kk = 0; kk < DK; ++kk) {
                const Frag a = qcache::decode<BITS>(&kw[m][kk * W8], qcache::scale_value(kb[m][NSC == 1 ? 0 : kk]), HS{});
#pragma unroll
                for (int i = PARTS - 1; i >= 0; --i)
#pragma unroll
                    for (int t = 0; t < RT; ++t) s[t][m] = mma(a, qf[t][i][kk], s[t][m]);
            }
        }
        const bool whole = N == 1 || k0 + TK <= off + token0 + 1;  // every row sees all of these keys
        if (!whole) {
            bool odd = false;
#pragma unroll
            for (int i = 0; i < NV; ++i) odd |= vb[i] == kNoValue;
            if (__any(odd)) {
                // which rows see blocks that are NaN, as 0 times NaN is NaN to the others too
                for (int j = k0; j < min(k0 + TK, last); ++j) {
                    for (int i = 0; i < (int)scales; ++i) {
                        if ((j < held ? vsc[(int64_t)j * scale_stride + i] : fresh_row(head, 1, j - off)[4 * BITS + i]) != kNoValue)
                            continue;
#pragma unroll
                        for (int t = 0; t < RT; ++t)
                            if (j < lim[t]) lost[t] |= 1u << i;
                    }
                }
#pragma unroll
                for (int i = 0; i < NV; ++i) vb[i] = vb[i] == kNoValue ? 0 : vb[i];
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (!unit_there(i)) continue;
            const float scale = qcache::scale_value(vb[i]);
            HS* to = vt + unit_key(i) * P + 8 * unit_block(i);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<Frag*>(to + e * 8 * NB) = qcache::decode<BITS>(&vw[i][e * W8], scale, HS{});
        }
        if (k0 + step < last) fetch(k0 + step);
        Frag w[RT][PARTS];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
#pragma unroll
            for (int m = 0; m < NM; ++m) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = s[t][m][i];
                    if constexpr (CAP == kNoCap) x *= scale2;
                    else if constexpr (CAP == kCapFine) x = cap2 * fine_tanh(x * to_tanh).t;
                    else x = cap2 - 2.0f * cap2 * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * into_cap));
                    s[t][m][i] = x;
                }
            }
            if (p.slopes) {
                const float base = (float)(pos[t] - k0 - 4 * g);
#pragma unroll
                for (int m = 0; m < NM; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[t][m][i] -= slope2[t] * fabsf(base - (float)(16 * m + i));
            }
            if (!whole || k0 + TK > last) {
                const int left = min(lim[t], last) - k0 - 4 * g;
#pragma unroll
                for (int m = 0; m < NM; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[t][m][i] = 16 * m + i < left ? s[t][m][i] : kNegInf;
            }
            float mx = kNegInf;
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                mx = fmaxf(fmaxf(s[t][m][0], s[t][m][1]), mx);
                mx = fmaxf(fmaxf(s[t][m][2], s[t][m][3]), mx);
            }
            mx = column_max(mx);
            if (__any(mx > top[t] + kRowsSlack)) {
                const float to = fmaxf(mx, top[t]), f = top[t] == to ? 1.0f : __builtin_amdgcn_exp2f(top[t] - to);
                top[t] = to;
                sum[t] *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[t][d] *= f;
            }
            const float ref = top[t] == kNegInf ? 0.0f : top[t];
#pragma unroll
            for (int m = 0; m < NM; ++m) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[t][m][i] = __builtin_amdgcn_exp2f(s[t][m][i] - ref);
                sum[t] += (s[t][m][0] + s[t][m][1]) + (s[t][m][2] + s[t][m][3]);
            }
            if constexpr (PARTS == 1) {
                w[t][0] = frag_tiles(s[t][0], s[t][1], HS{});
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    bf16 u, v, x;
                    three_parts(s[t][e / 4][e % 4], u, v, x);
                    w[t][0][e] = u, w[t][PARTS / 2][e] = v, w[t][PARTS - 1][e] = x;
                }
            }
        }
        // the LDS of a wave is its own, and its operations stay in order
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const Frag a = frag_columns<HE>(vt + 16 * d, P, g, c);
#pragma unroll
            for (int i = PARTS - 1; i >= 0; --i)
#pragma unroll
                for (int t = 0; t < RT; ++t) acc[t][d] = mma(a, w[t][i], acc[t][d]);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }

    // the waves' shares of one tile of rows at a time: out [wave][row][DP + 2]
    float* out = (float*)smem;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const float total = column_sum(sum[t]);
        __syncthreads();
        float* mine = out + (wave * 16 + c) * (DP + 2);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // the dimension that stands in this column
                const int at = 16 * d + 4 * g + i, dim = at % (8 * NB) / 8 * kBlock + at / (8 * NB) * 8 + at % 8;
                mine[dim] = lost[t] >> (dim / kBlock) & 1 ? __builtin_nanf("") : acc[t][d][i];
            }
        }
        if (g == 0) {
            mine[DP] = top[t];
            mine[DP + 1] = total;
        }
        __syncthreads();
        const unsigned row_begin = group * 16 * RT + 16 * t, live = rows > row_begin ? min(rows - row_begin, 16u) : 0;
        for (unsigned at = 0; at < heads; ++at) {
            for (unsigned i = tid; i < live * DP; i += 256) {
                const unsigned r = i / DP, d = i % DP;
                if (d >= D) continue;
                // this head's waves are `heads` apart
                float tops[4], sums[4], o[4], best = kNegInf, all = 0.0f, v = 0.0f;
#pragma unroll
                for (unsigned w = 0; w < 4; ++w) {
                    const float* from = out + ((min(w, shares - 1) * heads + at) * 16 + r) * (DP + 2);
                    tops[w] = from[DP], sums[w] = from[DP + 1], o[w] = from[d];
                    best = fmaxf(best, tops[w]);
                }
#pragma unroll
                for (unsigned w = 0; w < 4; ++w) {
                    if (w >= shares) continue;
                    // a wave without a key that is seen has a sum of 0 and no reference
                    const float f = tops[w] == best ? 1.0f : __builtin_amdgcn_exp2f(tops[w] - best);
                    all += sums[w] * f;
                    v += o[w] * f;
                }
                const unsigned row = row_begin + r, token = row / R, h = (kvh0 + at) * R + row % R;
                const int64_t to = (int64_t)token * H + h;
                if (splits == 1) {
                    y[to * D + d] = (S)((int)token < fresh ? v / all : 0.0f);
                } else {
                    float* left = p.parts + (((int64_t)b * N * H + to) * splits + split) * (D + 4);
                    left[d] = v;
                    if (d == 0) {
                        left[D] = best;
                        left[D + 1] = all;
                    }
                }
            }
        }
    }
}

// What the parts of each row leave, joined: 32 lanes, four dimensions a lane, take every SETS-th part.
// With SETS = 8 a row is a workgroup's, and the first 32 lanes join what the eight leave, in order;
// otherwise a workgroup has eight rows, each with all of its parts.
template <typename E, int SETS>
__global__ __launch_bounds__(256) void qattn_join_kernel(AttnArgs p) {
    typedef typename Elem<E>::S S;
    typedef S S4 __attribute__((ext_vector_type(4)));
    __shared__ __align__(16) float left[SETS == 8 ? 8 : 1][128 + 4];
    const int d = (threadIdx.x & 31) * 4, set = threadIdx.x >> 5;
    const unsigned b = blockIdx.y, rows = (unsigned)(p.N * p.H);
    const unsigned at = SETS == 8 ? blockIdx.x : blockIdx.x * 8 + set, token = at / (unsigned)p.H;
    const int64_t row = (int64_t)b * rows + at;
    const int len = p.lengths[b], fresh = p.fresh ? min(max(p.fresh[b], 0), (int)p.N) : (int)p.N;
    const bool idle = len < 0 || (int64_t)len + fresh > p.M, there = at < rows && d < p.D;
    Joined j{kNegInf, 0.0f, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
    if (!idle && there)
        j = join_parts<SETS, 8>(p.parts + row * p.splits * (p.D + 4), SETS == 8 ? set : 0, (int)p.splits, p.D, d);
    if constexpr (SETS == 8) {
        if (!idle && there) {
            *reinterpret_cast<f32x4*>(&left[set][d]) = j.v;
            if (d == 0) {
                left[set][p.D] = j.top;
                left[set][p.D + 1] = j.total;
            }
        }
        __syncthreads();
        if (set) return;
        j = Joined{kNegInf, 0.0f, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
        if (!idle && there) {
#pragma unroll
            for (int s = 0; s < 8; ++s)
                j.add(left[s][p.D], left[s][p.D + 1], *reinterpret_cast<const f32x4*>(&left[s][d]));
        }
    }
    if (!there) return;
    f32x4 v = j.v / j.total;
    if (idle || (int)token >= fresh) {
        const float none = !idle || len < 0 ? 0.0f : __builtin_nanf("");
        v = f32x4{none, none, none, none};
    }
    *reinterpret_cast<S4*>((S*)p.y + row * p.D + d) = __builtin_convertvector(v, S4);
}

template <typename E, int BITS, int DP, int CAP, int RT>
static int rows_launch(const AttnArgs& p, hipStream_t stream) {
    const int64_t units = p.splits * p.B * ceil_div(p.H / p.G * p.N, 16 * RT), sets = p.G / p.row_splits;
    qattn_rows_kernel<E, BITS, DP, CAP, RT>
        <<<dim3((unsigned)(ceil_div(units, 8) * 8 * sets)), 256, RowsLds<DP>::all(p.row_splits, p.k_new ? p.N : 0, BITS), stream>>>(p);
    const int rc = check_launch("qattn_rows");
    if (rc != FLARE_OK || p.splits == 1) return rc;
    // Eight parts are one lane's loads under way at once and need no second pass: eight tokens (4 bits,
    // 16 heads of 128 over 4) for 64 sequences of 4096 take 54 us for 62 with a workgroup a row, 257
    // tokens (float, 8 heads of 64) behind 1021 23.4 for 27.6. With up to 16 parts that way one token for
    // 16 of 4096 (8 bits, 16 heads of 64) takes 41.3 for 39.7.
    const unsigned rows = (unsigned)(p.N * p.H), sequences = (unsigned)p.B;
    if (p.splits <= 8) qattn_join_kernel<E, 1><<<dim3((rows + 7) / 8, sequences), 256, 0, stream>>>(p);
    else qattn_join_kernel<E, 8><<<dim3(rows, sequences), 256, 0, stream>>>(p);
    return check_launch("qattn_join");
}
template <typename E, int BITS, int DP, int CAP>
static int rows_rt(const AttnArgs& p, int tiles, hipStream_t stream) {
    if constexpr (sizeof(E) == 2)
        if (tiles == 2) return rows_launch<E, BITS, DP, CAP, 2>(p, stream);
    return rows_launch<E, BITS, DP, CAP, 1>(p, stream);
}
template <typename E, int BITS, int DP>
static int rows_dp(const AttnArgs& p, int tiles, hipStream_t stream) {
    if (p.cap == 0.0f) return rows_rt<E, BITS, DP, kNoCap>(p, tiles, stream);
    if constexpr (sizeof(E) == 2)
        if (p.cap <= kCoarseCapMost) return rows_rt<E, BITS, DP, kCap>(p, tiles, stream);
    return rows_rt<E, BITS, DP, kCapFine>(p, tiles, stream);
}
// tiles: of 16 rows a wave owns, 1, or 2 of 16-bit queries (the parts of fp32 ones take three times the registers).
template <typename E, int BITS>
int rows_e(const AttnArgs& p, int tiles, hipStream_t stream) {
    return p.D <= 32   ? rows_dp<E, BITS, 32>(p, tiles, stream)
           : p.D <= 64 ? rows_dp<E, BITS, 64>(p, tiles, stream)
           : p.D <= 96 ? rows_dp<E, BITS, 96>(p, tiles, stream)
                       : rows_dp<E, BITS, 128>(p, tiles, stream);
}

}  // namespace attn
}  // namespace flare
