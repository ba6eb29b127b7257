// flare_attn_step.hip -- softmax attention of one new token a sequence over its cache.
//
// The cache's bytes bound it.  A wave takes 32 keys at a time: K goes from memory straight into
// the A operand of S^T = K Q^T, whose 16 columns are the heads that share these keys, V through
// a stretch of LDS of its own to be read transposed.  The keys of a sequence are split over
// `splits` workgroups of four waves by its true length; attn_join adds up what they leave.  The
// new token's key and value are read from the call's tensors and put into the cache by the one
// workgroup whose share they are in.  64 sequences of 8000 tokens, 4 key heads of 128, bf16: 1.05 GB in
// 182 us, 5.8 TB/s (a copy reads and writes at 4.7, a sum reads at 4.0);
// with a cap 185 us.
#include "flare_attn.h"

namespace flare {
namespace attn {

constexpr int kTile = 32;            // keys a wave takes at a time

template <typename E, int DP>
struct StepLds {
    static constexpr int P = column_pitch<E, DP>();
    static constexpr size_t v_bytes = sizeof(E) * kTile * P;                       // of a wave
    static constexpr size_t o_bytes = sizeof(float) * 16 * (DP + 2);               // of a wave, after the loop
    static constexpr size_t bytes = 4 * (v_bytes > o_bytes ? v_bytes : o_bytes);
};

template <typename E, int DP, bool CAP>
__global__ __launch_bounds__(256) void attn_step_kernel(AttnArgs p) {
    typedef typename Elem<E>::S S;
    typedef typename Elem<E>::Frag Frag;
    using Lds = StepLds<E, DP>;
    constexpr int DK = DP / 32, DT = DP / 16, P = Lds::P;
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, c = lane & 15;
    const int64_t R = p.H / p.G, HG = (R + 15) / 16;
    const int64_t split = blockIdx.x % (unsigned)p.splits, row = blockIdx.x / (unsigned)p.splits;
    const int64_t hg = row % HG, kvh = row / HG % p.G, b = row / HG / p.G;
    const int64_t len = p.lengths[b];
    if (len < 0 || len >= p.M) {
        // an idle row, or a full cache
        if (p.splits == 1) {
            for (int i = tid; i < 16 * (int)p.D; i += 256) {
                const int64_t r = hg * 16 + i / p.D;
                if (r < R)
                    ((S*)p.y)[(b * p.H + kvh * R + r) * p.D + i % p.D] = (S)(len < 0 ? 0.0f : __builtin_nanf(""));
            }
        }
        return;
    }
    const int64_t n = len + 1;
    const int64_t per = ((n + p.splits - 1) / p.splits + 4 * kTile - 1) / (4 * kTile) * (4 * kTile);
    const int64_t first = split * per, last = min(first + per, n);
    const bool head = hg * 16 + c < R;
    const int64_t h = kvh * R + (head ? hg * 16 + c : 0);
    const S* knew = (const S*)p.k_new + b * p.kn_sb + kvh * p.kn_sg;
    const S* vnew = (const S*)p.v_new + b * p.vn_sb + kvh * p.vn_sg;
    S* kc = (S*)p.k.p + (b * p.M * p.G + kvh) * p.D;
    S* vc = (S*)p.v.p + (b * p.M * p.G + kvh) * p.D;
    const int64_t stride = p.G * p.D;
    if (first <= len && len < last && hg == 0) {
        for (int d = tid; d < p.D; d += 256) {
            kc[len * stride + d] = knew[d];
            vc[len * stride + d] = vnew[d];
        }
    }

    Frag qf[DK];
#pragma unroll
    for (int kk = 0; kk < DK; ++kk) {
        const int d = 32 * kk + 8 * g;
        qf[kk] = Frag{};
        if (head && d < p.D) qf[kk] = frag_rows<E>((const S*)p.q.p + b * p.q.sb + h * p.q.sh + d);
    }
    const float scale2 = p.scale * kLog2e, slope2 = p.slopes ? p.slopes[h] * kLog2e : 0.0f;
    const float cap2 = p.cap * kLog2e, to_tanh = CAP ? p.scale / p.cap : 0.0f;
    f32x4 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float top = kNegInf, sum = 0.0f;

    S* vt = (S*)(smem + wave * Lds::v_bytes);
    constexpr int PER = 16 / sizeof(E), CPR = DP / PER, NV = kTile * CPR / 64;
    Frag kf[2][DK];
    u32x4 vr[NV];
    auto fetch = [&](int64_t k0) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const int64_t j = k0 + 16 * m + c;
            const S* row = j == len ? knew : kc + j * stride;
#pragma unroll
            for (int kk = 0; kk < DK; ++kk) {
                const int d = 32 * kk + 8 * g;
                kf[m][kk] = Frag{};
                if (j < last && d < p.D) kf[m][kk] = frag_rows<E>(row + d);
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = i * 64 + lane, col = e % CPR * PER;
            const int64_t j = k0 + e / CPR;
            vr[i] = u32x4{0, 0, 0, 0};
            if (j < last && col < p.D) vr[i] = *reinterpret_cast<const u32x4*>((j == len ? vnew : vc + j * stride) + col);
        }
    };
    int64_t k0 = first + wave * kTile;
    if (k0 < last) fetch(k0);
    for (; k0 < last; k0 += 4 * kTile) {
        f32x4 s[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int kk = 0; kk < DK; ++kk) s[m] = mma(kf[m][kk], qf[kk], s[m]);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = i * 64 + lane;
            *reinterpret_cast<u32x4*>(vt + e / CPR * P + e % CPR * PER) = vr[i];
        }
        if (k0 + 4 * kTile < last) fetch(k0 + 4 * kTile);
        const float base = (float)(int)(len - k0 - 4 * g);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = CAP ? cap2 * fine_tanh(s[m][i] * to_tanh).t : s[m][i] * scale2;
                x -= slope2 * (base - (float)(16 * m + i));
                s[m][i] = k0 + 16 * m + 4 * g + i < last ? x : kNegInf;
            }
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                         fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = column_max(mx);
        const float to = fmaxf(mx, top), f = top == to ? 1.0f : __builtin_amdgcn_exp2f(top - to);
        const float ref = to == kNegInf ? 0.0f : to;
        top = to;
        sum *= f;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] *= f;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[m][i] = __builtin_amdgcn_exp2f(s[m][i] - ref);
                sum += s[m][i];
            }
        }
        const Frag w = frag_tiles(s[0], s[1], S{});
        // the LDS of a wave is its own, and its operations stay in order
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] = mma(frag_columns<E>(vt + 16 * d, P, g, c), w, acc[d]);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    sum = column_sum(sum);

    // the four waves' shares: out [wave][head][DP + 2]
    __syncthreads();
    float* out = (float*)smem;
    {
        float* mine = out + (wave * 16 + c) * (DP + 2);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) mine[16 * d + 4 * g + i] = acc[d][i];
        if (g == 0) {
            mine[DP] = top;
            mine[DP + 1] = sum;
        }
    }
    __syncthreads();
    for (int i = tid; i < 16 * DP; i += 256) {
        const int r = i / DP, d = i % DP;
        if (hg * 16 + r >= R || d >= p.D) continue;
        const float* o = out + r * (DP + 2);
        constexpr int step = 16 * (DP + 2);
        const float t = fmaxf(fmaxf(o[DP], o[step + DP]), fmaxf(o[2 * step + DP], o[3 * step + DP]));
        float total = 0.0f, v = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            // a wave without a key has a sum of 0 and no reference
            const float top_w = o[w * step + DP];
            const float f = top_w == t ? 1.0f : __builtin_amdgcn_exp2f(top_w - t);
            total += o[w * step + DP + 1] * f;
            v += o[w * step + d] * f;
        }
        const int64_t row = b * p.H + kvh * R + hg * 16 + r;
        if (p.splits == 1) {
            ((S*)p.y)[row * p.D + d] = (S)(v / total);
        } else {
            float* part = p.parts + (row * p.splits + split) * (p.D + 4);
            part[d] = v;
            if (d == 0) {
                part[p.D] = first < last ? t : kNegInf;
                part[p.D + 1] = total;
            }
        }
    }
}

// A workgroup a row: 32 lanes, four dimensions a lane, take every eighth part, and the first of them
// what the eight leave, in order.
template <typename E>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs p) {
    typedef typename Elem<E>::S S;
    typedef S S4 __attribute__((ext_vector_type(4)));
    __shared__ __align__(16) float left[8][128 + 4];
    const int64_t row = blockIdx.x, b = row / p.H, len = p.lengths[b];
    const int d = (threadIdx.x & 31) * 4, set = threadIdx.x >> 5;
    const bool idle = len < 0 || len >= p.M;
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
    if (idle) {
        const float none = len < 0 ? 0.0f : __builtin_nanf("");
        v = f32x4{none, none, none, none};
    } else {
        Joined j{kNegInf, 0.0f, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int s = 0; s < 8; ++s) j.add(left[s][p.D], left[s][p.D + 1], *reinterpret_cast<const f32x4*>(&left[s][d]));
        v = j.v / j.total;
    }
    *reinterpret_cast<S4*>((S*)p.y + row * p.D + d) = __builtin_convertvector(v, S4);
}

template <typename E, int DP, bool CAP>
static int step_cap(const AttnArgs& p, hipStream_t stream) {
    constexpr size_t bytes = StepLds<E, DP>::bytes;
    auto kernel = attn_step_kernel<E, DP, CAP>;
    if (bytes > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != hipSuccess) {
            set_error("attn_step: %s", hipGetErrorString(e));
            return FLARE_ERR_LAUNCH;
        }
    }
    const int64_t HG = ceil_div(p.H / p.G, 16);
    kernel<<<dim3((unsigned)(p.splits * p.B * p.G * HG)), 256, bytes, stream>>>(p);
    int rc = check_launch("attn_step");
    if (rc != FLARE_OK || p.splits == 1) return rc;
    attn_join_kernel<E><<<dim3((unsigned)(p.B * p.H)), 256, 0, stream>>>(p);
    return check_launch("attn_join");
}
template <typename E, int DP>
static int step_dp(const AttnArgs& p, hipStream_t stream) {
    return p.cap > 0.0f ? step_cap<E, DP, true>(p, stream) : step_cap<E, DP, false>(p, stream);
}
template <typename E>
static int step_e(const AttnArgs& p, hipStream_t stream) {
    return p.D <= 32   ? step_dp<E, 32>(p, stream)
           : p.D <= 64 ? step_dp<E, 64>(p, stream)
           : p.D <= 96 ? step_dp<E, 96>(p, stream)
                       : step_dp<E, 128>(p, stream);
}
int attn_step(const AttnArgs& p, int dtype, hipStream_t stream) { return FLARE_BY_DTYPE(dtype, step_e, (p, stream)); }

}  // namespace attn
}  // namespace flare
