// flare_scan_bwd.hip -- gradients of the selective state space scan.
//
//   r_t = C_t dyg_t + a_{t+1} r_{t+1}        the gradient of h_t; dyg = dy z sigmoid(z)
//   ddelta_t = sum_s r a h_{t-1} A + x_t sum_s r B_t     dx_t = delta_t sum_s r B_t + D dyg_t
//   dA += r a h_{t-1} delta_t       dB_t = sum_c r delta x      dC_t = sum_c dyg h_t
//
// scan_reverse leaves each chunk's r from behind as if nothing entered it; scan_carries joins
// them; scan_gradient then takes each chunk in stretches between the states that the forward
// kept, the last one first: forward over a stretch, leaving a state every T tokens in LDS, and
// backward over these pieces of T tokens, each recomputed with a_t and a_t h_{t-1} in registers.
//
// There four lanes share a channel (SL = S / 4 states each) and a wave has 16 channels: the
// decays of a piece then take 2 T SL registers, where a lane with all the states of a channel
// would need four times that.  What one lane would do alone for a token (the exponentials of the
// gates, the loads and stores) lane q of a channel does for token q of a piece, and the others read
// it through DPP.  dB and dC are summed over the wave's channels by halving: each step adds two
// values and leaves one, half the lanes' worth of work at a time; the waves' sums meet in LDS and
// the workgroups' in scan_dbc, always in the same order.
//
// Vector instructions bound it, some 34 for an element of the state.  4 x 4096 tokens, 2048
// channels of 16 states, bf16: 654 us with T = 4 and three workgroups of four waves a CU (167
// registers); T = 8 (216 registers, two waves a SIMD) 691, eight waves a workgroup 773 to 881.
#include <type_traits>
#include <utility>

#include "flare_scan.h"

namespace flare {
namespace scan {

// Channel a lane, as scan_chunk: the gradient that leaves the chunk at its front.
template <typename E, int SP>
__global__ __launch_bounds__(256, lane_waves(SP)) void scan_reverse_kernel(ScanArgs p) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t per = (p.Cg + 63) / 64, cb = (int64_t)blockIdx.y * 4 + wave, b = blockIdx.z;
    const int64_t chunk = (int64_t)blockIdx.x + 1;             // nothing is before chunk 0
    if (cb >= p.G * per) return;
    const int64_t g = cb / per, cl = cb % per * 64 + lane, c = g * p.Cg + min(cl, p.Cg - 1);
    const unsigned cu = (unsigned)c;
    const int t0 = (int)(chunk * p.L), t1 = (int)min((chunk + 1) * p.L, p.N);
    const E* dt = (const E*)p.dt + b * p.dt_sb;
    const E* z = p.z ? (const E*)p.z + b * p.z_sb : nullptr;
    const E* dy = (const E*)p.dy + (b * p.N) * p.C;
    const int32_t* ids = p.ids ? p.ids + b * p.N : nullptr;
    scalar_f* bc = scalar_ptr(p.bc + ((b * p.N) * p.G + g) * 2 * SP) + SP;
    const int bc_step = (int)p.G * 2 * SP;
    float r[SP], A2[SP];
#pragma unroll
    for (int s = 0; s < SP; ++s) {
        A2[s] = (p.A2 + s * p.C)[cu];
        r[s] = 0.0f;
    }
    const float bias = p.dt_bias ? p.dt_bias[c] : 0.0f;
    float sum = 0.0f;
    bool cut = false;
    constexpr int U = 4, NB = SP < 16 ? SP : 16;
    E gr[U], dr[U], zr[U];
    auto fetch = [&](int t) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = max(t - u, t0);
            gr[u] = (dy + at * p.C)[cu];
            dr[u] = (dt + at * p.dt_sn)[cu];
            if (z) zr[u] = (z + at * p.z_sn)[cu];
        }
    };
    auto step_of = [&](E raw) {
        const float v = to_f32(raw) + bias;
        return p.softplus ? mix::softplus(v) : v;
    };
    auto rows = [&](int t, int k, float (&C)[NB]) {
        scalar_f* row = bc + (int64_t)t * bc_step + k * NB;
#pragma unroll
        for (int i = 0; i < NB; ++i) C[i] = row[i];
    };
    auto part = [&](float delta, float gy, int k, const float (&C)[NB]) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int s = k * NB + i;
            r[s] = __builtin_amdgcn_exp2f(delta * A2[s]) * (r[s] + gy * C[i]);
        }
    };
    fetch(t1 - 1);
    for (int t4 = t1 - 1; t4 >= t0; t4 -= U) {
        bool plain = t4 - U + 1 >= t0;             // as in scan_chunk
        if (ids && plain) {
            const int id = ids[t4];
            plain = id >= 0 && ids[t4 - 1] == id && ids[t4 - 2] == id && ids[t4 - 3] == id && !begins(ids, t4 - 3);
        }
        if (plain) {
            float gs[U], ds[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                gs[u] = to_f32(gr[u]);
                ds[u] = step_of(dr[u]);
                if (z) {
                    const float zv = to_f32(zr[u]);
                    gs[u] *= zv * mix::sigmoid(zv);
                }
            }
            if (t4 - U >= t0) fetch(t4 - U);
            float Cv[2][NB];
            rows(t4, 0, Cv[0]);
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int k = 0; k < SP / NB; ++k) {
                    const int step = u * (SP / NB) + k, next = step + 1;
                    asm volatile("" ::"s"(Cv[step & 1][0]));
                    if (next < U * (SP / NB)) rows(t4 - next / (SP / NB), next % (SP / NB), Cv[next & 1]);
                    __builtin_amdgcn_sched_barrier(0);
                    part(ds[u], gs[u], k, Cv[step & 1]);
                }
                sum += ds[u];
            }
        } else {
#pragma unroll 1
            for (int t = t4; t >= max(t4 - U + 1, t0); --t) {
                if (!ids || ids[t] >= 0) {
                    const float delta = step_of((dt + t * p.dt_sn)[cu]);
                    float gy = to_f32((dy + (int64_t)t * p.C)[cu]);
                    if (z) {
                        const float zv = to_f32((z + t * p.z_sn)[cu]);
                        gy *= zv * mix::sigmoid(zv);
                    }
#pragma unroll
                    for (int k = 0; k < SP / NB; ++k) {
                        float Cv[NB];
                        rows(t, k, Cv);
                        part(delta, gy, k, Cv);
                    }
                    sum += delta;
                }
                if (ids && begins(ids, t)) {
                    cut = true;
#pragma unroll
                    for (int s = 0; s < SP; ++s) r[s] = 0.0f;
                }
            }
            if (t4 - U >= t0) fetch(t4 - U);
        }
    }
#pragma unroll
    for (int s = 0; s < SP; ++s) (p.carry + ((b * p.NC + chunk - 1) * SP + s) * p.C)[cu] = r[s];
    p.dsum[(b * p.NC + chunk) * p.C + c] = sum;
    if (ids && c == 0) p.cuts[b * p.NC + chunk] = cut;
}

// Slot k - 1 of `carry` holds what leaves chunk k at its front, and then all that enters k - 1.
__global__ __launch_bounds__(256) void scan_carries_kernel(ScanArgs p, int SP) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= p.B * SP * p.C) return;
    const int64_t c = id % p.C, s = id / p.C % SP, b = id / p.C / SP;
    const float A2 = p.A2[s * p.C + c];
    float* slot = p.carry + ((b * p.NC) * SP + s) * p.C + c;
    const int64_t step = SP * p.C;
    const float* dsum = p.dsum + (b * p.NC) * p.C + c;
    float r = 0.0f;
    slot[(p.NC - 1) * step] = 0.0f;
    constexpr int U = 8;
    for (int64_t k0 = p.NC - 1; k0 > 0; k0 -= U) {
        float own[U], dec[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t k = max(k0 - u, (int64_t)1);
            own[u] = slot[(k - 1) * step];
            dec[u] = A2 * dsum[k * p.C];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t k = k0 - u;
            if (k < 1) break;
            r = p.ids && p.cuts[b * p.NC + k] ? own[u] : decayed(r, dec[u]) + own[u];
            slot[(k - 1) * step] = r;
        }
    }
}

__device__ __forceinline__ float lane_xor4(float x) {     // within 8 lanes: mirror, then each quad again
    return mfma::dpp<0x1B>(mfma::dpp<mfma::kRowHalfMirror>(x));
}
__device__ __forceinline__ float lane_xor8(float x) { return mfma::dpp<0x128>(x); }   // row_ror:8

// v[0 .. NV-1] of each lane summed over the 16 channels of the wave (lane bits 2 .. 5).  Leaves
// max(1, NV / 16) values in v; `first` is the index of v[0], `own` whether this lane stores it.
template <int NV>
__device__ __forceinline__ void sum_channels(float (&v)[NV], int lane, int& first, bool& own) {
    first = 0;
    own = true;
    auto sum = [](mix::Halves r) { return r.first + r.second; };
    // NV >= 4: the steps over lane bits 5 and 4 always halve
#pragma unroll
    for (int i = 0; i < NV / 2; ++i) v[i] = sum(mix::swap32(v[i], v[i + NV / 2]));
    first += lane & 32 ? NV / 2 : 0;
#pragma unroll
    for (int i = 0; i < NV / 4; ++i) v[i] = sum(mix::swap16(v[i], v[i + NV / 4]));
    first += lane & 16 ? NV / 4 : 0;
    if constexpr (NV >= 8) {
#pragma unroll
        for (int i = 0; i < NV / 8; ++i) {
            const float a = v[i], b = v[i + NV / 8];
            v[i] = (lane & 8 ? b : a) + lane_xor8(lane & 8 ? a : b);
        }
        first += lane & 8 ? NV / 8 : 0;
    } else {
        v[0] += lane_xor8(v[0]);
        own = own && !(lane & 8);
    }
    if constexpr (NV >= 16) {
#pragma unroll
        for (int i = 0; i < NV / 16; ++i) {
            const float a = v[i], b = v[i + NV / 16];
            v[i] = (lane & 4 ? b : a) + lane_xor4(lane & 4 ? a : b);
        }
        first += lane & 4 ? NV / 16 : 0;
    } else {
        v[0] += lane_xor4(v[0]);
        own = own && !(lane & 4);
    }
}

// a[0 .. 3] of each lane summed over the quad; lane q gets the sum of a[q].
__device__ __forceinline__ float quad_gather(const float (&a)[4], int q) {
    const float lo = (q & 1 ? a[1] : a[0]) + mfma::dpp<mfma::kQuadXor1>(q & 1 ? a[0] : a[1]);
    const float hi = (q & 1 ? a[3] : a[2]) + mfma::dpp<mfma::kQuadXor1>(q & 1 ? a[2] : a[3]);
    return (q & 2 ? hi : lo) + mfma::dpp<mfma::kQuadXor2>(q & 2 ? lo : hi);
}
__device__ __forceinline__ float quad_sum(float x) {
    x += mfma::dpp<mfma::kQuadXor1>(x);
    return x + mfma::dpp<mfma::kQuadXor2>(x);
}
// Lane J of the quad, to all four.
template <int J>
__device__ __forceinline__ float quad_bcast(float x) {
    return mfma::dpp<J * 0x55>(x);
}

// fn(0), fn(1), ... with compile-time indices: register arrays and DPP controls need them.
template <typename F, int... J>
__device__ __forceinline__ void each_token(F&& fn, std::integer_sequence<int, J...>) {
    (fn(std::integral_constant<int, J>{}), ...);
}

constexpr int kWaves = 4;              // 64 channels a workgroup

template <int SP>
struct GradLayout {
    static constexpr int SL = SP / 4;
    static constexpr int T = 4;                          // a token for each lane of a channel
    static constexpr int keep = (int)kept_tokens(SP), pieces = keep / T;
    static constexpr int bc_floats = (int)kBackwardChunkMost * 2 * SP;
    static constexpr int keep_floats = kWaves * pieces * 64 * SL;
    static constexpr int red_floats = kWaves * T * 2 * SP;
    static constexpr size_t bytes = sizeof(float) * (bc_floats + keep_floats + red_floats);
    static_assert(bytes <= 160 * 1024, "LDS of a CU");
};

// One value of each token of a chunk through a buffer descriptor: tokens behind the chunk's last
// one and lanes without a channel load 0 and store nothing, and an address costs one addition.
template <typename E>
struct TokenValues {
    __amdgpu_buffer_rsrc_t r;
    unsigned at, step;               // bytes: this lane's channel, or past everything; a token
    // `base`: the chunk's first token; n tokens `stride` elements apart
    __device__ __forceinline__ TokenValues(const void* base, int n, int64_t stride, int64_t C, int64_t c, bool active)
        : r(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0,
                                              base ? (int)((n - 1) * stride + C) * (int)sizeof(E) : 0, 0x00020000)),
          at(active ? (unsigned)c * (unsigned)sizeof(E) : 0x80000000u), step((unsigned)stride * (unsigned)sizeof(E)) {}
    __device__ __forceinline__ E load(int lane_token, int k) const {
        const unsigned o = at + lane_token * step + k * step;
        if constexpr (sizeof(E) == 2) {
            const unsigned short v = __builtin_amdgcn_raw_buffer_load_b16(r, o, 0, 0);
            return __builtin_bit_cast(E, v);
        } else {
            const unsigned v = __builtin_amdgcn_raw_buffer_load_b32(r, o, 0, 0);
            return __builtin_bit_cast(E, v);
        }
    }
    __device__ __forceinline__ void store(int lane_token, int k, float x) const {
        const unsigned o = at + lane_token * step + k * step;
        if constexpr (sizeof(E) == 2)
            __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, from_f32<E>(x)), r, o, 0, 0);
        else __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, x), r, o, 0, 0);
    }
};

// SL adjacent floats of LDS, aligned to all of them (or 16 bytes).
template <int SL>
__device__ __forceinline__ void lds_row(const float* p, float (&out)[SL]) {
    constexpr int V = SL < 4 ? SL : 4;
    typedef float fv __attribute__((ext_vector_type(V)));
#pragma unroll
    for (int i = 0; i < SL; i += V) {
        const fv v = *reinterpret_cast<const fv*>(p + i);
#pragma unroll
        for (int j = 0; j < V; ++j) out[i + j] = v[j];
    }
}

template <typename E, int SP>
__global__ __launch_bounds__(64 * kWaves) void scan_gradient_kernel(ScanArgs p) {
    using Lay = GradLayout<SP>;
    constexpr int SL = Lay::SL, T = Lay::T, KEEP = Lay::keep;
    // Where a document begins r becomes 0, and a decay of 0 times an infinite r is NaN.  By a branch, or
    // element by element where registers are short: us with either, 16 states (4 x 4096 x 2048) 532,
    // 546; 32 (2 x 2048 x 2048) 258, 261; 64 (2 x 2048 x 1024) 370, 342.
    constexpr bool SELECT = SP == 64;
    extern __shared__ __align__(16) float lds[];
    float* bcs = lds;                                      // [L][2][SP]
    float* keeps = bcs + Lay::bc_floats;                   // [waves][pieces][SL][64]
    float* red = keeps + Lay::keep_floats;                 // [waves][T][2 SP]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane & 3;
    const int64_t per = (p.Cg + 16 * kWaves - 1) / (16 * kWaves);
    const int64_t cb = blockIdx.y, b = blockIdx.z, chunk = blockIdx.x;
    const int64_t g = cb / per, cl = cb % per * 16 * kWaves + wave * 16 + (lane >> 2);
    const bool active = cl < p.Cg;
    const int64_t c = g * p.Cg + (active ? cl : p.Cg - 1);
    const int64_t t0 = chunk * p.L;
    const int n = (int)(min(t0 + p.L, p.N) - t0);          // tokens of this chunk
    const int32_t* ids = p.ids ? p.ids + b * p.N + t0 : nullptr;
    const bool z = p.z != nullptr;
    const int64_t row0 = (b * p.N + t0) * p.C;
    auto values = [&](const void* base, int64_t first, int64_t stride) {
        return TokenValues<E>(base ? (const E*)base + first : nullptr, n, stride, p.C, c, active);
    };
    const auto xs = values(p.x, b * p.x_sb + t0 * p.x_sn, p.x_sn), dts = values(p.dt, b * p.dt_sb + t0 * p.dt_sn, p.dt_sn);
    const auto zs = values(p.z, b * p.z_sb + t0 * p.z_sn, p.z_sn), dys = values(p.dy, row0, p.C);
    const auto dxs = values(p.dx, row0, p.C), ddts = values(p.ddt, row0, p.C), dzs = values(p.dz, row0, p.C);

    const int rows = (n + T - 1) / T * T;                  // tokens behind the last one have B = C = 0
    for (int i = tid; i < rows * 2 * SP; i += 64 * kWaves)
        bcs[i] = i < n * 2 * SP ? p.bc[((b * p.N + t0 + i / (2 * SP)) * p.G + g) * 2 * SP + i % (2 * SP)] : 0.0f;
    __syncthreads();

    float A2[SL], h[SL], r[SL], dA[SL];
    float* keep = keeps + (size_t)wave * Lay::pieces * 64 * SL + lane;
#pragma unroll
    for (int i = 0; i < SL; ++i) {
        const int s = q * SL + i;
        A2[i] = p.A2[s * p.C + c];
        r[i] = active && p.NC > 1 ? p.carry[((b * p.NC + chunk) * SP + s) * p.C + c] : 0.0f;
        dA[i] = 0.0f;
    }
    const float* kept = p.kept + ((b * ((p.N + KEEP - 1) / KEEP) + t0 / KEEP) * SP + q * SL) * p.C + c;
    const float bias = p.dt_bias ? p.dt_bias[c] : 0.0f, skip = p.D ? p.D[c] : 0.0f;
    float dD = 0.0f, dbias = 0.0f;

    // Token q of the piece at k0, as loaded.
    struct Raw {
        E dt, x, dy, z;
        int id;
    };
    auto fetch = [&](Raw& r, int k0, bool all) {
        const int k = max(k0, 0);
        r.dt = dts.load(q, k);
        r.x = xs.load(q, k);
        if (all) r.dy = dys.load(q, k);
        if (all && z) r.z = zs.load(q, k);
        r.id = ids ? ids[min(k + q, n - 1)] : 0;
    };
    // a token that is none has delta = x = 0
    auto step_of = [&](const Raw& r, int k, float& raw, float& delta, float& xv) {
        const bool live = active && k < n && r.id >= 0;
        raw = live ? to_f32(r.dt) + bias : 0.0f;
        delta = live ? (p.softplus ? mix::softplus(raw) : raw) : 0.0f;
        xv = live ? to_f32(r.x) : 0.0f;
        return live;
    };
    auto piece_begins = [&](int k0) {      // bit j: a document begins at token k0 + j
        if (!ids) return 0u;
        const int k = k0 + (lane & (T - 1));
        return (unsigned)__ballot(lane < T && k < n && t0 + k > 0 && ids[k] != ids[k - 1]);
    };
    // h over the piece at k0; `take`(j, i, a, a h) sees each decay and what it leaves.  CUT: a
    // document begins in it.
    auto forward = [&](auto cutc, int k0, unsigned starts, float delta, float du, auto&& take) {
        constexpr bool CUT = decltype(cutc)::value;
        auto token = [&](auto jc) {
            constexpr int j = decltype(jc)::value;
            float B[SL];
            lds_row<SL>(bcs + (k0 + j) * 2 * SP + q * SL, B);
            const float dj = quad_bcast<j>(delta), uj = quad_bcast<j>(du);
            const bool cut = CUT && (starts >> j & 1);
#pragma unroll
            for (int i = 0; i < SL; ++i) {
                float a = __builtin_amdgcn_exp2f(dj * A2[i]), ah = a * h[i];
                if (cut) a = ah = 0.0f;
                take(jc, i, a, ah);
                h[i] = ah + uj * B[i];
            }
        };
        each_token(token, std::make_integer_sequence<int, T>{});
    };

    for (int first = (n - 1) / KEEP * KEEP; first >= 0; first -= KEEP) {
        const int here = min(KEEP, n - first), pieces = (here + T - 1) / T;
#pragma unroll
        for (int i = 0; i < SL; ++i) h[i] = active ? kept[(int64_t)(first / KEEP) * SP * p.C + i * p.C] : 0.0f;
        // forward, keeping the state before each piece
        Raw raws[Lay::pieces - 1];
#pragma unroll
        for (int piece = 0; piece + 1 < Lay::pieces; ++piece)
            if (piece + 1 < pieces) fetch(raws[piece], first + piece * T, false);
        Raw next;
        fetch(next, first + (pieces - 1) * T, true);
#pragma unroll
        for (int i = 0; i < SL; ++i) keep[i * 64] = h[i];
#pragma unroll
        for (int piece = 0; piece + 1 < Lay::pieces; ++piece) {
            if (piece + 1 >= pieces) break;
            const int k0 = first + piece * T;
            float raw, delta, xv;
            step_of(raws[piece], k0 + q, raw, delta, xv);
            const unsigned starts = piece_begins(k0);
            auto nothing = [](auto, int, float, float) {};
            if (starts) forward(std::true_type{}, k0, starts, delta, delta * xv, nothing);
            else forward(std::false_type{}, k0, 0u, delta, delta * xv, nothing);
#pragma unroll
            for (int i = 0; i < SL; ++i) keep[((piece + 1) * SL + i) * 64] = h[i];
        }

        // backward over the pieces
        for (int piece = pieces - 1; piece >= 0; --piece) {
            const int k0 = first + piece * T;
            const Raw now = next;
            fetch(next, k0 - T, true);
            float raw, delta, xv;
            const bool live = step_of(now, k0 + q, raw, delta, xv);
            const float du = delta * xv, dyv = live ? to_f32(now.dy) : 0.0f, zv = live && z ? to_f32(now.z) : 0.0f;
            const float gate = z ? mix::sigmoid(zv) : 1.0f, gy = z ? dyv * zv * gate : dyv;
            float a[T][SL], ah[T][SL];
#pragma unroll
            for (int i = 0; i < SL; ++i) h[i] = keep[(piece * SL + i) * 64];
            const unsigned starts = piece_begins(k0);
            auto hold = [&](auto jc, int i, float av, float ahv) {
                a[decltype(jc)::value][i] = av;
                ah[decltype(jc)::value][i] = ahv;
            };
            if (starts) forward(std::true_type{}, k0, starts, delta, du, hold);
            else forward(std::false_type{}, k0, 0u, delta, du, hold);
            // the tokens in reverse, and then what their lanes do with the sums
            float pA[T], sB[T], lin[T];
            auto back = [&](auto jc) {
                constexpr int j = T - 1 - decltype(jc)::value;
                const float* row = bcs + (k0 + j) * 2 * SP + q * SL;
                const float dj = quad_bcast<j>(delta), uj = quad_bcast<j>(du), gj = quad_bcast<j>(gy);
                float v[2 * SL], B[SL], Cv[SL];
                lds_row<SL>(row, B);
                lds_row<SL>(row + SP, Cv);
                pA[j] = sB[j] = lin[j] = 0.0f;
#pragma unroll
                for (int i = 0; i < SL; ++i) {
                    const float hv = ah[j][i] + uj * B[i];
                    r[i] += Cv[i] * gj;
                    const float w = r[i] * ah[j][i];
                    pA[j] += w * A2[i];
                    dA[i] += w * dj;
                    sB[j] += r[i] * B[i];
                    lin[j] += Cv[i] * hv;
                    v[i] = r[i] * uj;
                    v[SL + i] = gj * hv;
                    r[i] = SELECT && (starts >> j & 1) ? 0.0f : r[i] * a[j][i];
                }
                if (!SELECT && __builtin_expect(starts >> j & 1, 0)) {
#pragma unroll
                    for (int i = 0; i < SL; ++i) r[i] = 0.0f;
                }
                int at;
                bool own;
                sum_channels(v, lane, at, own);
                if (own) {
                    constexpr int NK = SL >= 8 ? SL / 8 : 1;
                    float* out = red + (wave * T + j) * 2 * SP + q * SL;
#pragma unroll
                    for (int m = 0; m < NK; ++m) {
                        const int idx = at + m;              // state idx of B, or idx - SL of C
                        out[idx < SL ? idx : SP + idx - SL] = v[m];
                    }
                }
                if constexpr (j == 0) {
                    const float pq = quad_gather(pA, q) * kLn2, sq = quad_gather(sB, q), lq = quad_gather(lin, q);
                    float ddt = pq + xv * sq;
                    if (p.softplus) ddt *= mix::sigmoid(raw);
                    if (!live) ddt = 0.0f;
                    dbias += ddt;
                    dD += gy * xv;
                    dxs.store(q, k0, live ? delta * sq + gy * skip : 0.0f);
                    ddts.store(q, k0, ddt);
                    if (z) {
                        const float dz = dyv * (lq + skip * xv) * gate * (1.0f + zv * (1.0f - gate));
                        dzs.store(q, k0, live ? dz : 0.0f);
                    }
                }
            };
            each_token(back, std::make_integer_sequence<int, T>{});
            // the piece's dB and dC: the waves' sums, in order
            __syncthreads();
            const int live_tokens = min(T, n - k0);
            float* out = p.dbc + ((cb * p.B + b) * p.N + t0 + k0) * 2 * SP;
            for (int i = tid; i < live_tokens * 2 * SP; i += 64 * kWaves) {
                float s = 0.0f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) s += red[w * T * 2 * SP + i];
                out[i] = s;
            }
            __syncthreads();
        }
    }
    if (!active) return;
    float* par = p.dpar + ((b * p.NC + chunk) * p.C + c) * (SP + 2);
#pragma unroll
    for (int i = 0; i < SL; ++i) par[q * SL + i] = dA[i];
    dD = quad_sum(dD);
    dbias = quad_sum(dbias);
    if (q < 2) par[SP + q] = q ? dbias : dD;
}

// dB and dC of each token: the sum over the channel blocks of its group, in order.
template <typename E>
__global__ __launch_bounds__(256) void scan_dbc_kernel(ScanArgs p, int SP, int64_t per) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= p.B * p.N * p.G * 2 * SP) return;
    const int64_t s = id % (2 * SP), bn = id / (2 * SP) % (p.B * p.N), g = id / (2 * SP) / (p.B * p.N);
    float v = 0.0f;
    for (int64_t k = 0; k < per; ++k) v += p.dbc[((g * per + k) * p.B * p.N + bn) * 2 * SP + s];
    const int64_t col = s % SP;
    if (col >= p.S) return;
    E* out = (E*)(s < SP ? p.dB : p.dC);
    out[(bn * p.G + g) * p.S + col] = from_f32<E>(v);
}

// Where the column sums of [C, SP + 2] go: dA [C, S], dD [C] and ddt_bias [C].
struct PutParams {
    int S, SP;
    float *dA, *dD, *dbias;
    __device__ __forceinline__ void operator()(int64_t col, float v) const {
        const int64_t c = col / (SP + 2), s = col % (SP + 2);
        if (s < S) dA[c * S + s] = v;
        else if (s == SP && dD) dD[c] = v;
        else if (s == SP + 1 && dbias) dbias[c] = v;
    }
};

template <typename E, int SP>
static int backward_go(const ScanArgs& p, hipStream_t stream) {
    int rc;
    if (p.NC > 1) {
        const int64_t blocks = ceil_div(p.G * ceil_div(p.Cg, 64), 4);
        scan_reverse_kernel<E, SP>
            <<<dim3((unsigned)(p.NC - 1), (unsigned)blocks, (unsigned)p.B), 256, 0, stream>>>(p);
        if ((rc = check_launch("scan_reverse")) != FLARE_OK) return rc;
        scan_carries_kernel<<<dim3((unsigned)ceil_div(p.B * SP * p.C, 256)), 256, 0, stream>>>(p, SP);
        if ((rc = check_launch("scan_carries")) != FLARE_OK) return rc;
    }
    using Lay = GradLayout<SP>;
    const int64_t per = ceil_div(p.Cg, 16 * kWaves);
    if (Lay::bytes > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&scan_gradient_kernel<E, SP>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)Lay::bytes);
        if (e != hipSuccess) {
            set_error("scan_gradient: %s", hipGetErrorString(e));
            return FLARE_ERR_LAUNCH;
        }
    }
    scan_gradient_kernel<E, SP><<<dim3((unsigned)p.NC, (unsigned)(p.G * per), (unsigned)p.B), 64 * kWaves, Lay::bytes,
                                  stream>>>(p);
    if ((rc = check_launch("scan_gradient")) != FLARE_OK) return rc;
    scan_dbc_kernel<E><<<dim3((unsigned)ceil_div(p.B * p.N * p.G * 2 * SP, 256)), 256, 0, stream>>>(p, SP, per);
    return check_launch("scan_dbc");
}
template <typename E>
static int backward_e(const ScanArgs& p, int64_t SP, hipStream_t stream) {
    return SP == 8    ? backward_go<E, 8>(p, stream)
           : SP == 16 ? backward_go<E, 16>(p, stream)
           : SP == 32 ? backward_go<E, 32>(p, stream)
                      : backward_go<E, 64>(p, stream);
}

struct BackwardLayout {
    size_t bc, A2, carry, dsum, cuts, dbc, dpar, total;      // in floats
    BackwardLayout(int64_t B, int64_t N, int64_t C, int64_t S, int64_t G, int64_t NC) {
        const int64_t SP = padded_states(S), blocks = G * ceil_div(C / G, 16 * kWaves);
        bc = 0;
        A2 = bc + B * N * G * 2 * SP;
        carry = A2 + SP * C;
        dsum = carry + B * NC * SP * C;
        cuts = dsum + B * NC * C;
        dbc = cuts + B * NC;
        dpar = dbc + blocks * B * N * 2 * SP;
        total = dpar + B * NC * C * (SP + 2);
    }
};

}  // namespace scan
}  // namespace flare

using namespace flare;
using namespace flare::scan;

extern "C" size_t flare_scan_backward_workspace_size(int64_t B, int64_t N, int64_t C, int64_t S, int64_t G,
                                                     int64_t chunk) {
    if (chunk < 1 || G < 1) return 0;
    return BackwardLayout(B, N, C, S, G, ceil_div(N, chunk)).total * sizeof(float);
}

extern "C" int flare_scan_backward(const void* x, const void* dt, const float* A, const void* Bm, const void* Cm,
                                   const float* D, const void* z, const float* dt_bias, int softplus, int dtype,
                                   int64_t B, int64_t N, int64_t C, int64_t S, int64_t G, const int64_t* strides,
                                   const int32_t* document_ids, const void* dy, int64_t chunk, const float* kept,
                                   void* dx, void* ddt, float* dA, void* dB, void* dC, float* dD, void* dz,
                                   float* ddt_bias, void* workspace, size_t workspace_bytes, void* stream) {
    FLARE_REQUIRE(x && dt && A && Bm && Cm && dy && kept && strides && workspace && dx && ddt && dA && dB && dC,
                  "flare_scan_backward: null pointer");
    FLARE_REQUIRE(!z || dz, "flare_scan_backward: z without dz");
    SCAN_REQUIRE_SIZES("flare_scan_backward");
    const int64_t SP = padded_states(S);
    FLARE_REQUIRE(chunk >= 1 && chunk <= kBackwardChunkMost && chunk % kept_tokens(SP) == 0,
                  "flare_scan_backward: chunks of up to %lld tokens, multiples of the kept states' distance",
                  (long long)kBackwardChunkMost);
    ScanArgs p = scan_args(x, dt, A, Bm, Cm, D, z, dt_bias, softplus, B, N, C, S, G, strides);
    p.L = chunk, p.NC = ceil_div(N, chunk);
    for (int i = 1; i < 6; i += 2)
        FLARE_REQUIRE(strides[i] >= 0 && strides[i] < kMostStride,
                      "flare_scan_backward: tokens must be less than 2^22 elements apart");
    const BackwardLayout lay(B, N, C, S, G, p.NC);
    if (workspace_bytes < lay.total * sizeof(float)) {
        set_error("flare_scan_backward: workspace of %zu bytes is too small", workspace_bytes);
        return FLARE_ERR_WORKSPACE;
    }
    float* ws = (float*)workspace;
    p.ids = document_ids, p.dy = dy, p.kept = const_cast<float*>(kept), p.keep = kept_tokens(SP);
    p.dx = dx, p.ddt = ddt, p.dB = dB, p.dC = dC, p.dz = dz;
    p.bc = ws + lay.bc, p.A2 = ws + lay.A2, p.carry = ws + lay.carry, p.dsum = ws + lay.dsum;
    p.cuts = (int32_t*)(ws + lay.cuts), p.dbc = ws + lay.dbc, p.dpar = ws + lay.dpar;
    hipStream_t st = (hipStream_t)stream;
    int rc = launch_pack(p, dtype, SP, st);
    if (rc == FLARE_OK) rc = FLARE_BY_DTYPE(dtype, backward_e, (p, SP, st));
    if (rc != FLARE_OK) return rc;
    return mix::launch_column_sums(p.dpar, B * p.NC, C * (SP + 2), PutParams{(int)S, (int)SP, dA, dD, ddt_bias}, st);
}
