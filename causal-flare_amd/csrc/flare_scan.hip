// flare_scan.hip -- the selective state space scan: forward and single-token step.
//
// scan_chunk: a lane is a channel and holds its S states and rates in registers, so B_t and
// C_t are the same for the whole wave: they are scalar loads, and scalar operands of the
// vector instructions.  An element of the state costs an exponential (8 cycles of a SIMD a wave,
// measured), two products and one or two fused products (4 each), a token a softplus and its gate:
// vector instructions bound it, and both passes over a chunk pay them.  16384 tokens, 2048 channels
// of 16 states, bf16: the chunks' ends 122 us, the output 162 us, where the elements' instructions
// alone are 70 and 84; scan_states 22 us (34 MB read and written).
#include "flare_scan.h"

namespace flare {
namespace scan {

// What the kernels read again and again, laid out once: B and C of every token in fp32 with zeros
// behind S, rows that scalar loads can take whole (padding's rows are 0, whatever they hold); A in
// log2 units and the state before the first chunk, [SP, C] each, so that lanes of neighbouring
// channels read neighbouring words.
template <typename E>
__global__ __launch_bounds__(256) void scan_pack_kernel(ScanArgs p, int SP) {
    int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t rows = p.B * p.N * p.G * 2 * SP, n = (int64_t)SP * p.C;
    if (id < rows) {
        const int s = (int)(id % SP), which = (int)(id / SP % 2);
        const int64_t g = id / (2 * SP) % p.G, t = id / (2 * SP) / p.G % p.N, b = id / (2 * SP) / p.G / p.N;
        float v = 0.0f;
        if (s < p.S && !(p.ids && p.ids[b * p.N + t] < 0)) {
            v = which ? to_f32(((const E*)p.Cm)[b * p.C_sb + t * p.C_sn + g * p.C_sg + s])
                      : to_f32(((const E*)p.Bm)[b * p.B_sb + t * p.B_sn + g * p.B_sg + s]);
        }
        p.bc[id] = v;
        return;
    }
    id -= rows;
    if (id >= n * (1 + p.B)) return;
    const int64_t c = id % p.C, s = id / p.C % SP, b = id / n - 1;
    if (b < 0) p.A2[id] = s < p.S ? p.A[c * p.S + s] * kLog2e : 0.0f;
    else if (p.states) p.states[(b * p.NC * SP + s) * p.C + c] = p.h0 && s < p.S ? p.h0[(b * p.C + c) * p.S + s] : 0.0f;
}

template <typename E>
static int pack_go(const ScanArgs& p, int64_t SP, hipStream_t stream) {
    const int64_t work = p.B * p.N * p.G * 2 * SP + SP * p.C * (1 + p.B);
    scan_pack_kernel<E><<<dim3((unsigned)ceil_div(work, 256)), 256, 0, stream>>>(p, (int)SP);
    return check_launch("scan_pack");
}
int launch_pack(const ScanArgs& p, int dtype, int64_t SP, hipStream_t stream) {
    return FLARE_BY_DTYPE(dtype, pack_go, (p, SP, stream));
}

// One channel block of 64 (within a group) and one chunk a wave.  OUT false: leaves the chunk's
// end state in the next chunk's slot of `states` and its sum of delta in `dsum`.
template <typename E, int SP, bool OUT>
__global__ __launch_bounds__(256, lane_waves(SP)) void scan_chunk_kernel(ScanArgs p) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t per = (p.Cg + 63) / 64, cb = (int64_t)blockIdx.y * 4 + wave, b = blockIdx.z, chunk = blockIdx.x;
    if (cb >= p.G * per) return;
    // Lanes behind the last channel do as that one does, and write what it writes.
    const int64_t g = cb / per, cl = cb % per * 64 + lane, c = g * p.Cg + min(cl, p.Cg - 1);
    const unsigned cu = (unsigned)c;               // the lane's part of every address
    const int len = (int)row_length(p, b), L = (int)p.L;
    const int t0 = (int)chunk * L, t1 = min(t0 + L, len), tn = min(t0 + L, (int)p.N);
    const E* x = (const E*)p.x + b * p.x_sb;
    const E* dt = (const E*)p.dt + b * p.dt_sb;
    const E* z = p.z ? (const E*)p.z + b * p.z_sb : nullptr;
    E* y = (E*)p.y + (b * p.N) * p.C;
    const int32_t* ids = p.ids ? p.ids + b * p.N : nullptr;
    scalar_f* bc = scalar_ptr(p.bc + ((b * p.N) * p.G + g) * 2 * SP);
    const int bc_step = (int)p.G * 2 * SP;

    float h[SP], A2[SP];
#pragma unroll
    for (int s = 0; s < SP; ++s) {
        A2[s] = (p.A2 + s * p.C)[cu];
        h[s] = OUT ? (p.states + ((b * p.NC + chunk) * SP + s) * p.C)[cu] : 0.0f;
    }
    const float bias = p.dt_bias ? p.dt_bias[c] : 0.0f;
    const float skip = OUT && p.D ? p.D[c] : 0.0f;
    float sum = 0.0f;
    bool cut = false;                              // a document begins within the chunk

    constexpr int U = 4, NB = SP < 16 ? SP : 16;
    E xr[U], dr[U], zr[U];
    auto fetch = [&](int t) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = min(t + u, t1 - 1);
            xr[u] = (x + at * p.x_sn)[cu];
            dr[u] = (dt + at * p.dt_sn)[cu];
            if (OUT && z) zr[u] = (z + at * p.z_sn)[cu];
        }
    };
    auto step_of = [&](E raw) {
        const float v = to_f32(raw) + bias;
        return p.softplus ? mix::softplus(v) : v;
    };
    auto rows = [&](int t, int k, float (&B)[NB], float (&C)[NB]) {
        scalar_f* row = bc + (int64_t)t * bc_step + k * NB;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            B[i] = row[i];
            C[i] = OUT ? row[SP + i] : 0.0f;
        }
    };
    auto part = [&](float delta, float xv, int k, const float (&B)[NB], const float (&C)[NB], float (&out)[4]) {
        const float du = delta * xv;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int s = k * NB + i;
            h[s] = __builtin_amdgcn_exp2f(delta * A2[s]) * h[s] + du * B[i];
            if (OUT) out[i & 3] += C[i] * h[s];
        }
    };
    auto keep = [&](int t) {
        if (!OUT || !p.kept || (t & ((int)p.keep - 1))) return;
        int64_t step = p.C;
        asm volatile("" : "+s"(step));             // keeps the 16 addresses out of the loop's registers
        float* to = p.kept + (b * ((p.N + p.keep - 1) / p.keep) + t / (int)p.keep) * SP * step;
#pragma unroll
        for (int s = 0; s < SP; ++s) (to + s * step)[cu] = h[s];
    };
    if (t0 < t1) fetch(t0);
    for (int t4 = t0; t4 < t1; t4 += U) {
        keep(t4);
        // Four tokens of one document run without a branch between them.  The scalar loads of the
        // next NB states are issued once those of the present ones are there.
        bool plain = t4 + U <= t1;
        if (ids && plain) {
            const int id = ids[t4];
            plain = id >= 0 && ids[t4 + 1] == id && ids[t4 + 2] == id && ids[t4 + 3] == id && !begins(ids, t4);
        }
        if (plain) {
            float xs[U], ds[U], gate[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                xs[u] = to_f32(xr[u]);
                ds[u] = step_of(dr[u]);
                gate[u] = 1.0f;
                if (OUT && z) {
                    const float zv = to_f32(zr[u]);
                    gate[u] = zv * mix::sigmoid(zv);
                }
            }
            if (t4 + U < t1) fetch(t4 + U);
            float Bv[2][NB], Cv[2][NB];
            rows(t4, 0, Bv[0], Cv[0]);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float out[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < SP / NB; ++k) {
                    const int step = u * (SP / NB) + k, next = step + 1;
                    asm volatile("" ::"s"(Bv[step & 1][0]));
                    if (next < U * (SP / NB)) rows(t4 + next / (SP / NB), next % (SP / NB), Bv[next & 1], Cv[next & 1]);
                    __builtin_amdgcn_sched_barrier(0);
                    part(ds[u], xs[u], k, Bv[step & 1], Cv[step & 1], out);
                }
                sum += ds[u];
                if (OUT) {
                    const float o = (out[0] + out[1]) + (out[2] + out[3]) + skip * xs[u];
                    (y + (int64_t)(t4 + u) * p.C)[cu] = from_f32<E>(o * gate[u]);
                }
            }
        } else {
#pragma unroll 1
            for (int t = t4; t < min(t4 + U, t1); ++t) {
                if (ids && begins(ids, t)) {
                    cut = true;
#pragma unroll
                    for (int s = 0; s < SP; ++s) h[s] = 0.0f;
                }
                float o = 0.0f;
                if (!ids || ids[t] >= 0) {
                    const float xv = to_f32((x + t * p.x_sn)[cu]), delta = step_of((dt + t * p.dt_sn)[cu]);
                    float out[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int k = 0; k < SP / NB; ++k) {
                        float Bv[NB], Cv[NB];
                        rows(t, k, Bv, Cv);
                        part(delta, xv, k, Bv, Cv, out);
                    }
                    sum += delta;
                    o = (out[0] + out[1]) + (out[2] + out[3]) + skip * xv;
                    if (OUT && z) {
                        const float zv = to_f32((z + t * p.z_sn)[cu]);
                        o *= zv * mix::sigmoid(zv);
                    }
                }
                if (OUT) (y + (int64_t)t * p.C)[cu] = from_f32<E>(o);
            }
            if (t4 + U < t1) fetch(t4 + U);
        }
    }
    if (OUT) {
        for (int t = max(t0, len); t < tn; ++t) (y + (int64_t)t * p.C)[cu] = from_f32<E>(0.0f);
        const int last = len > 0 ? (len - 1) / L : 0;
        if (p.h_fin && chunk == last) {
            float* to = p.h_fin + (b * p.C + c) * p.S;
#pragma unroll
            for (int s = 0; s < SP; ++s)
                if (s < p.S) to[s] = h[s];
        }
    } else {
#pragma unroll
        for (int s = 0; s < SP; ++s) (p.states + ((b * p.NC + chunk + 1) * SP + s) * p.C)[cu] = h[s];
        p.dsum[(b * p.NC + chunk) * p.C + c] = sum;
        if (ids && c == 0) p.cuts[b * p.NC + chunk] = cut;
    }
}

// The state before each chunk from the chunks' end states, in place: slot k + 1 holds chunk k's
// own end state, and then the state before chunk k + 1.
__global__ __launch_bounds__(256) void scan_states_kernel(ScanArgs p, int SP) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= p.B * SP * p.C) return;
    const int64_t c = id % p.C, s = id / p.C % SP, b = id / p.C / SP;
    const float A2 = p.A2[s * p.C + c];
    float* slot = p.states + ((b * p.NC) * SP + s) * p.C + c;
    float h = slot[0];
    const int64_t step = SP * p.C;
    const float* dsum = p.dsum + (b * p.NC) * p.C + c;
    constexpr int U = 8;
    for (int64_t k0 = 0; k0 + 1 < p.NC; k0 += U) {
        float own[U], dec[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t k = min(k0 + u, p.NC - 2);
            own[u] = slot[(k + 1) * step];
            dec[u] = A2 * dsum[k * p.C];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t k = k0 + u;
            if (k + 1 >= p.NC) break;
            // a document's beginning cuts off what came before it
            h = p.ids && p.cuts[b * p.NC + k] ? own[u] : decayed(h, dec[u]) + own[u];
            slot[(k + 1) * step] = h;
        }
    }
}

int launch_states(const ScanArgs& p, int64_t SP, hipStream_t stream) {
    scan_states_kernel<<<dim3((unsigned)ceil_div(p.B * SP * p.C, 256)), 256, 0, stream>>>(p, (int)SP);
    return check_launch("scan_states");
}

template <typename E, int SP>
static int forward_go(const ScanArgs& p, hipStream_t stream) {
    const int64_t blocks = ceil_div(p.G * ceil_div(p.Cg, 64), 4);
    if (p.NC > 1) {
        scan_chunk_kernel<E, SP, false>
            <<<dim3((unsigned)(p.NC - 1), (unsigned)blocks, (unsigned)p.B), 256, 0, stream>>>(p);
        int rc = check_launch("scan_chunk");
        if (rc == FLARE_OK) rc = launch_states(p, SP, stream);
        if (rc != FLARE_OK) return rc;
    }
    scan_chunk_kernel<E, SP, true><<<dim3((unsigned)p.NC, (unsigned)blocks, (unsigned)p.B), 256, 0, stream>>>(p);
    return check_launch("scan_output");
}
template <typename E>
static int forward_e(const ScanArgs& p, int64_t SP, hipStream_t stream) {
    return SP == 8    ? forward_go<E, 8>(p, stream)
           : SP == 16 ? forward_go<E, 16>(p, stream)
           : SP == 32 ? forward_go<E, 32>(p, stream)
                      : forward_go<E, 64>(p, stream);
}

// One token.  Four lanes share a channel, SP / 4 states each, so a wave reads and writes the
// states of 16 channels as one run of memory; the states' bytes bound it.  64 sequences of 2048
// channels of 16 states: 6.5 us, 2.7 TB/s, of which a launch and a chain of loads are some 3.
template <typename E, int SP, bool WHOLE>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanArgs p, const int32_t* mask, float* state) {
    constexpr int SL = SP / 4;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int q = (int)(id & 3);
    if ((id >> 2) >= p.B * p.C) return;                 // whole quads
    const int64_t b = (id >> 2) / p.C, c = (id >> 2) % p.C, g = c / p.Cg;
    float o = 0.0f;
    if (!mask || mask[b]) {
        const int s0 = q * SL;
        float* hp = state + (b * p.C + c) * p.S + s0;
        const float* A = p.A + c * p.S + s0;
        const E* Bm = (const E*)p.Bm + b * p.B_sb + g * p.B_sg + s0;
        const E* Cm = (const E*)p.Cm + b * p.C_sb + g * p.C_sg + s0;
        const float xv = to_f32(((const E*)p.x)[b * p.x_sb + c]);
        float delta = to_f32(((const E*)p.dt)[b * p.dt_sb + c]) + (p.dt_bias ? p.dt_bias[c] : 0.0f);
        float h[SL], av[SL];
        if (WHOLE) {
            typedef float fv __attribute__((ext_vector_type(SL < 4 ? SL : 4)));
            constexpr int V = SL < 4 ? SL : 4;
#pragma unroll
            for (int i = 0; i < SL; i += V) {
                const fv hv = *reinterpret_cast<const fv*>(hp + i), a4 = *reinterpret_cast<const fv*>(A + i);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    h[i + j] = hv[j];
                    av[i + j] = a4[j];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < SL; ++i) {
                h[i] = s0 + i < p.S ? hp[i] : 0.0f;
                av[i] = s0 + i < p.S ? A[i] : 0.0f;
            }
        }
        if (p.softplus) delta = mix::softplus(delta);
        const float du = delta * xv;
#pragma unroll
        for (int i = 0; i < SL; ++i) {
            if (WHOLE || s0 + i < p.S) {
                h[i] = __builtin_amdgcn_exp2f(delta * av[i] * kLog2e) * h[i] + du * to_f32(Bm[i]);
                o += to_f32(Cm[i]) * h[i];
            }
        }
        if (WHOLE) {
            typedef float fv __attribute__((ext_vector_type(SL < 4 ? SL : 4)));
            constexpr int V = SL < 4 ? SL : 4;
#pragma unroll
            for (int i = 0; i < SL; i += V) {
                fv hv;
#pragma unroll
                for (int j = 0; j < V; ++j) hv[j] = h[i + j];
                *reinterpret_cast<fv*>(hp + i) = hv;
            }
        } else {
#pragma unroll
            for (int i = 0; i < SL; ++i)
                if (s0 + i < p.S) hp[i] = h[i];
        }
        o += mfma::dpp<mfma::kQuadXor1>(o);
        o += mfma::dpp<mfma::kQuadXor2>(o);
        if (p.D) o += p.D[c] * xv;
        if (p.z) {
            const float zv = to_f32(((const E*)p.z)[b * p.z_sb + c]);
            o *= zv * mix::sigmoid(zv);
        }
    }
    if (q == 0) ((E*)p.y)[b * p.C + c] = from_f32<E>(o);
}

template <typename E, int SP>
static int step_go(const ScanArgs& p, const int32_t* mask, float* state, hipStream_t stream) {
    const dim3 g((unsigned)ceil_div(p.B * p.C * 4, 256));
    const bool whole = p.S == SP && ((uintptr_t)state & 15) == 0 && ((uintptr_t)p.A & 15) == 0;
    if (whole) scan_step_kernel<E, SP, true><<<g, 256, 0, stream>>>(p, mask, state);
    else scan_step_kernel<E, SP, false><<<g, 256, 0, stream>>>(p, mask, state);
    return check_launch("scan_step");
}
template <typename E>
static int step_e(const ScanArgs& p, const int32_t* mask, float* state, hipStream_t stream) {
    const int64_t SP = padded_states(p.S);
    return SP == 8    ? step_go<E, 8>(p, mask, state, stream)
           : SP == 16 ? step_go<E, 16>(p, mask, state, stream)
           : SP == 32 ? step_go<E, 32>(p, mask, state, stream)
                      : step_go<E, 64>(p, mask, state, stream);
}

}  // namespace scan
}  // namespace flare

using namespace flare;
using namespace flare::scan;

extern "C" int64_t flare_scan_chunk(int64_t B, int64_t N, int64_t C, int64_t S, int64_t G, int for_backward) {
    if (B < 1 || N < 1 || C < 1 || S < 1 || S > 64 || G < 1 || C % G) return 0;
    return chunk_length(B, N, C, G, for_backward != 0);
}
extern "C" int64_t flare_scan_kept_tokens(int64_t S) { return S < 1 || S > 64 ? 0 : kept_tokens(padded_states(S)); }

extern "C" size_t flare_scan_forward_workspace_size(int64_t B, int64_t N, int64_t C, int64_t S, int64_t G,
                                                    int64_t chunk) {
    if (chunk < 1 || N < 1) return 0;
    const int64_t SP = padded_states(S), NC = ceil_div(N, chunk < N ? chunk : N);
    return (size_t)(B * N * G * 2 * SP + SP * C + B * NC * (C * (SP + 1) + 1)) * sizeof(float);
}

extern "C" int flare_scan_forward(const void* x, const void* dt, const float* A, const void* Bm, const void* Cm,
                                  const float* D, const void* z, const float* dt_bias, int softplus, int dtype,
                                  int64_t B, int64_t N, int64_t C, int64_t S, int64_t G, const int64_t* strides,
                                  const int32_t* document_ids, const int32_t* lengths, const float* h0, void* y,
                                  float* h_fin, int64_t chunk, float* kept, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    FLARE_REQUIRE(x && dt && A && Bm && Cm && y && strides && workspace, "flare_scan_forward: null pointer");
    FLARE_REQUIRE(!(document_ids && (lengths || h0 || h_fin)),
                  "flare_scan_forward: document_ids exclude lengths and states");
    FLARE_REQUIRE(!h_fin || h_fin != h0, "flare_scan_forward: the states overlap");
    SCAN_REQUIRE_SIZES("flare_scan_forward");
    FLARE_REQUIRE(chunk >= 1 && (!kept || chunk % kept_tokens(padded_states(S)) == 0),
                  "flare_scan_forward: chunks must be positive, and multiples of the kept states' distance");
    ScanArgs p = scan_args(x, dt, A, Bm, Cm, D, z, dt_bias, softplus, B, N, C, S, G, strides);
    const int64_t SP = padded_states(S);
    p.L = chunk < N ? chunk : N, p.NC = ceil_div(N, p.L);
    if (workspace_bytes < flare_scan_forward_workspace_size(B, N, C, S, G, chunk)) {
        set_error("flare_scan_forward: workspace of %zu bytes is too small", workspace_bytes);
        return FLARE_ERR_WORKSPACE;
    }
    p.ids = document_ids, p.lengths = lengths, p.h0 = h0, p.y = y, p.h_fin = h_fin;
    p.kept = kept, p.keep = kept_tokens(SP);
    p.bc = (float*)workspace;
    p.A2 = p.bc + B * N * G * 2 * SP;
    p.states = p.A2 + SP * C;
    p.dsum = p.states + B * p.NC * SP * C;
    p.cuts = (int32_t*)(p.dsum + B * p.NC * C);
    const int rc = launch_pack(p, dtype, SP, (hipStream_t)stream);
    if (rc != FLARE_OK) return rc;
    return FLARE_BY_DTYPE(dtype, forward_e, (p, SP, (hipStream_t)stream));
}

extern "C" int flare_scan_step(const void* x, const void* dt, const float* A, const void* Bm, const void* Cm,
                               const float* D, const void* z, const float* dt_bias, int softplus, int dtype,
                               int64_t B, int64_t C, int64_t S, int64_t G, const int64_t* strides,
                               const int32_t* mask, float* state, void* y, void* stream) {
    const int64_t N = 1;
    FLARE_REQUIRE(x && dt && A && Bm && Cm && y && strides && state, "flare_scan_step: null pointer");
    SCAN_REQUIRE_SIZES("flare_scan_step");
    ScanArgs p = scan_args(x, dt, A, Bm, Cm, D, z, dt_bias, softplus, B, N, C, S, G, strides);
    p.y = y;
    return FLARE_BY_DTYPE(dtype, step_e, (p, mask, state, (hipStream_t)stream));
}
