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
// What the cache holds is exact in bf16, and in fp16 where that is the queries' type.  fp32 queries and
// weights enter as three bf16 parts, 24 bits.
//
// The keys of a sequence are split over `splits` workgroups of four waves by its true length; qattn_join adds
// up what they leave.  A single token's key and value are quantised by the workgroups whose share they are in,
// one of which puts them into the cache.
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

template <typename E, int BITS, int DP, int CAP, int RT>
__global__ __launch_bounds__(256) void qattn_rows_kernel(AttnArgs p) {
    typedef typename Elem<E>::S S;
    typedef typename Held<E>::Type HE;                 // what the products take
    typedef typename Elem<HE>::S HS;
    typedef typename Elem<HE>::Frag Frag;
    using Lds = RowsLds<DP>;
    constexpr int PARTS = Held<E>::parts;
    constexpr int DK = DP / 32, DT = DP / 16, NB = DP / kBlock, P = Lds::P;
    constexpr int TK = BITS == 4 && RT == 1 ? 64 : 32, NM = TK / 16, W8 = BITS / 4;      // W8: words of eight codes
    constexpr int NSC = DK == 3 ? 3 : 1;               // blocks that a lane's dimensions of K may lie in
    constexpr int NVH = (32 * NB + 63) / 64;           // blocks of V a lane takes, of 32 keys
    extern __shared__ __align__(16) char smem[];
    __shared__ u32 new_codes[2][4 * BITS];
    __shared__ u32 new_scales[2][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, c = lane & 15;
    const int D = (int)p.D;
    const int64_t R = p.H / p.G, rows = R * p.N, groups = (rows + 16 * RT - 1) / (16 * RT);
    const int64_t split = blockIdx.x % (unsigned)p.splits, id = blockIdx.x / (unsigned)p.splits;
    const int64_t group = id % groups, kvh = id / groups % p.G, b = id / groups / p.G;
    const bool single = p.k_new != nullptr;            // its key and value are not in the cache yet
    int64_t off = p.lengths[b];
    const int64_t fresh = p.fresh ? clamp_to(p.fresh[b], p.N) : p.N;
    if (off < 0 || off + fresh > p.M) {
        // an idle sequence, or a full cache
        if (p.splits == 1) {
            for (int i = tid; i < 16 * RT * D; i += 256) {
                const int64_t r = group * 16 * RT + i / D;
                if (r < rows)
                    ((S*)p.y)[((b * p.N + r / R) * p.H + kvh * R + r % R) * D + i % D] =
                        (S)(off < 0 ? 0.0f : __builtin_nanf(""));
            }
        }
        return;
    }
    const int64_t n = off + fresh, prefix = p.prefix ? clamp_to(p.prefix[b], n) : 0;
    const int64_t per = ((n + p.splits - 1) / p.splits + 4 * TK - 1) / (4 * TK) * (4 * TK);
    const int64_t first = split * per, last = min(first + per, n);
    const int64_t held = single ? min(last, off) : last;       // what of it memory holds
    const int64_t codes = qcache::row_codes(D, BITS), scales = qcache::row_scales(D);
    uint8_t* kc = (uint8_t*)p.k.p + (b * p.M * p.G + kvh) * codes;
    uint8_t* vc = (uint8_t*)p.v.p + (b * p.M * p.G + kvh) * codes;
    uint8_t* ksc = p.k_scale + (b * p.M * p.G + kvh) * scales;
    uint8_t* vsc = p.v_scale + (b * p.M * p.G + kvh) * scales;
    const int64_t stride = p.G * codes, scale_stride = p.G * scales;

    // the single token's key and value: a quad of lanes a block
    if (single && first <= off && off < last) {
        if (tid < 8 * NB) {
            const int which = tid / (4 * NB), block = tid / 4 % NB, d = block * kBlock + (tid & 3) * 8;
            const S* from = which ? (const S*)p.v_new + b * p.vn_sb + kvh * p.vn_sg
                                  : (const S*)p.k_new + b * p.kn_sb + kvh * p.kn_sg;
            float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
            if (d < D) qcache::load8(reinterpret_cast<const E*>(from) + d, x);
            const u32 byte = qcache::scale_of<BITS>(qcache::quad_max(qcache::top_of(x)), __is_same(E, __half));
            const Codes<BITS> w = qcache::encode<BITS>(x, byte);
#pragma unroll
            for (int i = 0; i < W8; ++i) new_codes[which][d / 8 * W8 + i] = w.w[i];
            if ((tid & 3) == 0) new_scales[which][block] = byte;
            if (group == 0 && d < D) {
                *reinterpret_cast<Codes<BITS>*>((which ? vc : kc) + off * stride + d * BITS / 8) = w;
                if ((tid & 3) == 0) (which ? vsc : ksc)[off * scale_stride + block] = (uint8_t)byte;
            }
        }
        __syncthreads();
    }

    Frag qf[RT][PARTS][DK];
    float slope2[RT];
    int lim[RT], pos[RT];                              // of this lane's rows: the keys it sees are below, and its place
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int64_t r = group * 16 * RT + 16 * t + c, token = r / R, h = kvh * R + r % R;
        const bool live = r < rows && token < fresh;
        pos[t] = (int)(off + token);
        lim[t] = live ? (int)min(n, max(off + token + 1, prefix)) : 0;
        slope2[t] = p.slopes && live ? p.slopes[h] * kLog2e : 0.0f;
#pragma unroll
        for (int kk = 0; kk < DK; ++kk) {
            const int d = 8 * (DK * g + kk);
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

    HS* vt = (HS*)(smem + wave * Lds::v_bytes);
    const bool full = D == DP;
    u32 kw[NM][DK * W8], kb[NM][NSC];
    u32 vw[NM / 2][NVH][BITS], vb[NM / 2][NVH];
    // key (of 32) and block of V of this lane's unit i: keys 0, 2, 1, 3 follow each other, as rows two apart
    // lie half the banks apart
    auto unit_key = [&](int i) {
        const int t = (i * 64 + lane) / NB;
        return (t & ~3) | (t & 1) << 1 | (t >> 1 & 1);
    };
    auto unit_block = [&](int i) { return (i * 64 + lane) % NB; };
    auto fetch = [&](int64_t k0) {
#pragma unroll
        for (int m = 0; m < NM; ++m) {
            const int64_t j = k0 + 16 * m + c;
            const bool there = j < held;
            const uint8_t* row = kc + j * stride + DK * W8 * 4 * g;
#pragma unroll
            for (int i = 0; i < DK * W8; ++i) kw[m][i] = 0;
            if (full) {
                if (there) __builtin_memcpy(kw[m], __builtin_assume_aligned(row, 4), sizeof(kw[m]));
            } else {
#pragma unroll
                for (int kk = 0; kk < DK; ++kk)
                    if (there && 8 * (DK * g + kk) < D)
                        __builtin_memcpy(&kw[m][kk * W8], __builtin_assume_aligned(row + kk * W8 * 4, 4), W8 * 4);
            }
#pragma unroll
            for (int i = 0; i < NSC; ++i) {
                const int block = 8 * (DK * g + i) / kBlock;
                kb[m][i] = there && block < scales ? ksc[j * scale_stride + block] : 0;
            }
        }
#pragma unroll
        for (int h = 0; h < NM / 2; ++h) {
#pragma unroll
            for (int i = 0; i < NVH; ++i) {
                const int64_t j = k0 + 32 * h + unit_key(i);
                const int block = unit_block(i), d = block * kBlock;
                const bool there = i * 64 + lane < 32 * NB && j < held && d < D;
                const uint8_t* row = vc + j * stride + block * (4 * BITS);
#pragma unroll
                for (int w = 0; w < BITS; ++w) vw[h][i][w] = 0;
                if (there) {
                    // a last block may have half the values
                    if (full || d + kBlock <= D) __builtin_memcpy(vw[h][i], __builtin_assume_aligned(row, 8), 4 * BITS);
                    else __builtin_memcpy(vw[h][i], __builtin_assume_aligned(row, 8), 2 * BITS);
                }
                vb[h][i] = there ? vsc[j * scale_stride + block] : 0;
            }
        }
    };
    // the single token's codes, for the lanes that take its place
    auto insert = [&](int64_t k0) {
#pragma unroll
        for (int m = 0; m < NM; ++m) {
            if (k0 + 16 * m + c != off) continue;
#pragma unroll
            for (int i = 0; i < DK * W8; ++i) kw[m][i] = new_codes[0][DK * W8 * g + i];
#pragma unroll
            for (int i = 0; i < NSC; ++i) kb[m][i] = new_scales[0][8 * (DK * g + i) / kBlock];
        }
#pragma unroll
        for (int h = 0; h < NM / 2; ++h) {
#pragma unroll
            for (int i = 0; i < NVH; ++i) {
                if (i * 64 + lane >= 32 * NB || k0 + 32 * h + unit_key(i) != off) continue;
#pragma unroll
                for (int w = 0; w < BITS; ++w) vw[h][i][w] = new_codes[1][unit_block(i) * BITS + w];
                vb[h][i] = new_scales[1][unit_block(i)];
            }
        }
    };

    int64_t k0 = first + wave * TK;
    if (k0 < last) fetch(k0);
    for (; k0 < last; k0 += 4 * TK) {
        if (single && k0 <= off && off < k0 + TK) insert(k0);
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
        // V's first 32 keys to LDS; the rest follow when these have been read
        const int64_t now = k0;
        const bool whole = single || (now + TK <= off + 1);        // every row sees all of these keys
        auto place = [&](int h) {
#pragma unroll
            for (int i = 0; i < NVH; ++i) {
                if (i * 64 + lane >= 32 * NB) continue;
                float scale = qcache::scale_value(vb[h][i]);
                if (!whole && vb[h][i] == kNoValue) scale = 0.0f;
                HS* to = vt + unit_key(i) * P + 8 * unit_block(i);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    *reinterpret_cast<Frag*>(to + e * 8 * NB) = qcache::decode<BITS>(&vw[h][i][e * W8], scale, HS{});
            }
        };
        if (!whole) {
            bool odd = false;
#pragma unroll
            for (int h = 0; h < NM / 2; ++h)
#pragma unroll
                for (int i = 0; i < NVH; ++i) odd |= vb[h][i] == kNoValue;
            if (__any(odd)) {
                // which rows see blocks that are NaN, as 0 times NaN is NaN to the others too
                for (int64_t j = now; j < min(now + TK, last); ++j) {
                    for (int i = 0; i < (int)scales; ++i) {
                        if (vsc[j * scale_stride + i] != kNoValue) continue;
#pragma unroll
                        for (int t = 0; t < RT; ++t)
                            if (j < lim[t]) lost[t] |= 1u << i;
                    }
                }
            }
        }
        place(0);
        u32 vw_rest[NM / 2][NVH][BITS], vb_rest[NM / 2][NVH];
        if constexpr (NM > 2) {
#pragma unroll
            for (int h = 1; h < NM / 2; ++h) {
#pragma unroll
                for (int i = 0; i < NVH; ++i) {
                    vb_rest[h][i] = vb[h][i];
#pragma unroll
                    for (int w = 0; w < BITS; ++w) vw_rest[h][i][w] = vw[h][i][w];
                }
            }
        }
        if (k0 + 4 * TK < last) fetch(k0 + 4 * TK);
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
                const float base = (float)(pos[t] - (int)now - 4 * g);
#pragma unroll
                for (int m = 0; m < NM; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[t][m][i] -= slope2[t] * fabsf(base - (float)(16 * m + i));
            }
            if (!whole || now + TK > last) {
                const int left = min(lim[t], (int)last) - (int)now - 4 * g;
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
        }
#pragma unroll
        for (int h = 0; h < NM / 2; ++h) {
            Frag w[RT][PARTS];
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                if constexpr (PARTS == 1) {
                    w[t][0] = frag_tiles(s[t][2 * h], s[t][2 * h + 1], HS{});
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        bf16 u, v, x;
                        three_parts(s[t][2 * h + e / 4][e % 4], u, v, x);
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
            if constexpr (NM > 2) {
                if (h + 1 < NM / 2) {
#pragma unroll
                    for (int i = 0; i < NVH; ++i) {
                        if (i * 64 + lane >= 32 * NB) continue;
                        float scale = qcache::scale_value(vb_rest[h + 1][i]);
                        if (!whole && vb_rest[h + 1][i] == kNoValue) scale = 0.0f;
                        HS* to = vt + unit_key(i) * P + 8 * unit_block(i);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            *reinterpret_cast<Frag*>(to + e * 8 * NB) =
                                qcache::decode<BITS>(&vw_rest[h + 1][i][e * W8], scale, HS{});
                    }
                }
            }
        }
    }

    // the four waves' shares of one tile of rows at a time: out [wave][row][DP + 2]
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
        for (int i = tid; i < 16 * DP; i += 256) {
            const int r = i / DP, d = i % DP;
            const int64_t row = group * 16 * RT + 16 * t + r;
            if (row >= rows || d >= D) continue;
            const float* o = out + r * (DP + 2);
            constexpr int step = 16 * (DP + 2);
            const float best = fmaxf(fmaxf(o[DP], o[step + DP]), fmaxf(o[2 * step + DP], o[3 * step + DP]));
            float all = 0.0f, v = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                // a wave without a key that is seen has a sum of 0 and no reference
                const float top_w = o[w * step + DP];
                const float f = top_w == best ? 1.0f : __builtin_amdgcn_exp2f(top_w - best);
                all += o[w * step + DP + 1] * f;
                v += o[w * step + d] * f;
            }
            const int64_t token = row / R, h = kvh * R + row % R;
            if (p.splits == 1) {
                ((S*)p.y)[((b * p.N + token) * p.H + h) * D + d] = (S)(token < fresh ? v / all : 0.0f);
            } else {
                float* part = p.parts + (((b * p.N + token) * p.H + h) * p.splits + split) * (D + 4);
                part[d] = v;
                if (d == 0) {
                    part[D] = best;
                    part[D + 1] = all;
                }
            }
        }
    }
}

// A workgroup a row: 32 lanes, four dimensions a lane, take every eighth part, and the first of them
// what the eight leave, in order.
template <typename E>
__global__ __launch_bounds__(256) void qattn_join_kernel(AttnArgs p) {
    typedef typename Elem<E>::S S;
    typedef S S4 __attribute__((ext_vector_type(4)));
    __shared__ __align__(16) float left[8][128 + 4];
    const int64_t row = blockIdx.x, token = row / p.H % p.N, b = row / p.H / p.N, len = p.lengths[b];
    const int64_t fresh = p.fresh ? clamp_to(p.fresh[b], p.N) : p.N;
    const int d = (threadIdx.x & 31) * 4, set = threadIdx.x >> 5;
    const bool idle = len < 0 || len + fresh > p.M;
    if (!idle && d < p.D) {
        const Joined j = join_parts<8, 8>(p.parts + row * p.splits * (p.D + 4), set, (int)p.splits, p.D, d);
        *reinterpret_cast<f32x4*>(&left[set][d]) = j.v;
        if (d == 0) {
            left[set][p.D] = j.top;
            left[set][p.D + 1] = j.total;
        }
    }
    __syncthreads();
    if (set || d >= p.D) return;
    f32x4 v;
    if (idle || token >= fresh) {
        const float none = !idle || len < 0 ? 0.0f : __builtin_nanf("");
        v = f32x4{none, none, none, none};
    } else {
        Joined j{kNegInf, 0.0f, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int s = 0; s < 8; ++s) j.add(left[s][p.D], left[s][p.D + 1], *reinterpret_cast<const f32x4*>(&left[s][d]));
        v = j.v / j.total;
    }
    *reinterpret_cast<S4*>((S*)p.y + row * p.D + d) = __builtin_convertvector(v, S4);
}

template <typename E, int BITS, int DP, int CAP, int RT>
static int rows_launch(const AttnArgs& p, hipStream_t stream) {
    const int64_t groups = ceil_div(p.H / p.G * p.N, 16 * RT);
    qattn_rows_kernel<E, BITS, DP, CAP, RT>
        <<<dim3((unsigned)(p.splits * p.B * p.G * groups)), 256, RowsLds<DP>::bytes, stream>>>(p);
    const int rc = check_launch("qattn_rows");
    if (rc != FLARE_OK || p.splits == 1) return rc;
    qattn_join_kernel<E><<<dim3((unsigned)(p.B * p.N * p.H)), 256, 0, stream>>>(p);
    return check_launch("qattn_join");
}
template <typename E, int BITS, int DP, int CAP>
static int rows_rt(const AttnArgs& p, int tiles, hipStream_t stream) {
    return tiles == 1 ? rows_launch<E, BITS, DP, CAP, 1>(p, stream) : rows_launch<E, BITS, DP, CAP, 2>(p, stream);
}
template <typename E, int BITS, int DP>
static int rows_dp(const AttnArgs& p, int tiles, hipStream_t stream) {
    if (p.cap == 0.0f) return rows_rt<E, BITS, DP, kNoCap>(p, tiles, stream);
    if constexpr (sizeof(E) == 2)
        if (p.cap <= kCoarseCapMost) return rows_rt<E, BITS, DP, kCap>(p, tiles, stream);
    return rows_rt<E, BITS, DP, kCapFine>(p, tiles, stream);
}
// tiles: of 16 rows a wave owns, 1 or 2.
template <typename E, int BITS>
int rows_e(const AttnArgs& p, int tiles, hipStream_t stream) {
    return p.D <= 32   ? rows_dp<E, BITS, 32>(p, tiles, stream)
           : p.D <= 64 ? rows_dp<E, BITS, 64>(p, tiles, stream)
           : p.D <= 96 ? rows_dp<E, BITS, 96>(p, tiles, stream)
                       : rows_dp<E, BITS, 128>(p, tiles, stream);
}

}  // namespace attn
}  // namespace flare
