// flare_scan.h -- the selective state space scan: what its forward and backward share.
//
//   delta_t = softplus(dt_t + dt_bias), or dt_t + dt_bias            [C]
//   a_t     = exp(delta_t A), 0 where a document begins              [C, S]
//   h_t     = a_t h_{t-1} + delta_t x_t B_t                          [C, S]
//   y_t     = (sum_s C_t h_t + D x_t) z_t sigmoid(z_t)               [C]
//
// Each of G groups of C / G channels has its own B_t and C_t [S].  A token that is none
// (behind the length, or of a negative document id) leaves h alone and has y = 0.
//
// The tokens are cut into chunks that run side by side.  A chunk's decay is exp(A sum delta),
// so its effect on a state is known from its own end state (from 0) and one sum a channel:
//   scan_chunk<false>   end state and sum of delta of each chunk
//   scan_states         the state before each chunk, in order
//   scan_chunk<true>    the chunk again from its state, with y
#pragma once

#include "flare_internal.h"
#include "flare_mix.h"

namespace flare {
namespace scan {

using mix::ceil_div;
using mix::known_dtype;
using mix::kLn2;
using mix::kLog2e;

struct ScanArgs {
    const void *x, *dt, *z, *Bm, *Cm;
    int64_t x_sb, x_sn, dt_sb, dt_sn, z_sb, z_sn, B_sb, B_sn, B_sg, C_sb, C_sn, C_sg;
    const float *A, *D, *dt_bias;       // [C, S], [C], [C]
    const int32_t *ids, *lengths;
    const float* h0;                    // [B, C, S]
    float* h_fin;
    void* y;
    // workspace
    float* bc;                          // [B, N, G, 2, SP]: B_t and C_t in fp32, zeros behind S
    float* A2;                          // [SP, C]: A log2(e), zeros behind S
    float* states;                      // [B, NC, SP, C]: the state before each chunk
    float* dsum;                        // [B, NC, C]
    int32_t* cuts;                      // [B, NC]: whether a document begins within the chunk
    float* kept;                        // [B, ceil(N / keep), SP, C]: the state before every keep-th token
    int64_t keep;
    // backward
    const void* dy;
    void *dx, *ddt, *dz;
    float* carry;                       // [B, NC, SP, C]: the gradient that enters each chunk from behind
    float* dbc;                         // [blocks, B, N, 2, SP]
    float* dpar;                        // [B * NC, C, SP + 2]
    void *dB, *dC;
    int64_t B, N, C, S, G, Cg, NC, L;
    int softplus;
};

__device__ __forceinline__ int64_t row_length(const ScanArgs& p, int64_t b) {
    if (!p.lengths) return p.N;
    const int64_t n = p.lengths[b];
    return n < 0 ? 0 : (n > p.N ? p.N : n);
}
// The state `h` behind a chunk whose tokens sum up to A2 dsum (log2 units).  In two halves, so that
// growth past fp32 leaves a small state what it is token by token; past 2^256 any but 0 is infinite,
// and 0 stays 0.
__device__ __forceinline__ float decayed(float h, float A2dsum) {
    const float e = __builtin_amdgcn_exp2f(0.5f * A2dsum);
    return h == 0.0f ? 0.0f : h * e * e;
}
// Whether token t begins a document.
__device__ __forceinline__ bool begins(const int32_t* ids, int64_t t) { return t > 0 && ids[t] != ids[t - 1]; }

// A pointer whose loads are scalar ones wherever the address is the same for the whole wave.
typedef __attribute__((address_space(4))) const float scalar_f;
__device__ __forceinline__ scalar_f* scalar_ptr(const float* p) { return (scalar_f*)(uintptr_t)p; }

inline int64_t padded_states(int64_t S) { return S <= 8 ? 8 : S <= 16 ? 16 : S <= 32 ? 32 : 64; }

// The backward holds B and C of a chunk in LDS, and recomputes its states from those the forward
// kept: so far apart that what it keeps of a stretch itself stays small.
constexpr int64_t kBackwardChunkMost = 128;
constexpr int64_t kMostStride = 1 << 22;        // between tokens, so that a chunk's offsets fit 31 bits
constexpr int64_t kept_tokens(int64_t SP) { return SP <= 16 ? 32 : SP == 32 ? 16 : 8; }

// Chunk length: some four waves a SIMD (4096 on the card).  Where the channels are too few for
// that a token's latency counts, and chunks go down to 8 tokens (32 for the backward, whose chunks
// hold whole stretches between kept states).  us, forward of 16384 tokens, 2048 channels of 16
// states, with chunks for 2048, 4096 and 8192 waves: 341, 303, 308, more states and less walking over a
// chunk; 257 tokens of 512 channels with chunks of 8 and of 32: 22, 44.
inline int64_t chunk_length(int64_t B, int64_t N, int64_t C, int64_t G, bool backward) {
    const int64_t waves = B * G * ceil_div(C / G, 64), nc = ceil_div(4096, waves), least = backward ? 32 : 8;
    const int64_t L = ceil_div(ceil_div(N, nc), least) * least;
    return backward && L > kBackwardChunkMost ? kBackwardChunkMost : L;
}

// strides: batch and token strides of x, dt, z; batch, token and group strides of B, C (elements).
inline ScanArgs scan_args(const void* x, const void* dt, const float* A, const void* Bm, const void* Cm,
                          const float* D, const void* z, const float* dt_bias, int softplus, int64_t B, int64_t N,
                          int64_t C, int64_t S, int64_t G, const int64_t* st) {
    ScanArgs p = {};
    p.x = x, p.dt = dt, p.z = z, p.Bm = Bm, p.Cm = Cm, p.A = A, p.D = D, p.dt_bias = dt_bias;
    p.x_sb = st[0], p.x_sn = st[1], p.dt_sb = st[2], p.dt_sn = st[3], p.z_sb = st[4], p.z_sn = st[5];
    p.B_sb = st[6], p.B_sn = st[7], p.B_sg = st[8], p.C_sb = st[9], p.C_sn = st[10], p.C_sg = st[11];
    p.B = B, p.N = N, p.C = C, p.S = S, p.G = G, p.Cg = C / G, p.softplus = softplus;
    return p;
}

#define SCAN_REQUIRE_SIZES(name)                                                                              \
    FLARE_REQUIRE(known_dtype(dtype), name ": unknown dtype %d", dtype);                                      \
    FLARE_REQUIRE(B >= 1 && N >= 1 && C >= 1, name ": B, N and C must be positive");                          \
    FLARE_REQUIRE(S >= 1 && S <= 64, name ": 1 to 64 states a channel, got %lld", (long long)S);              \
    FLARE_REQUIRE(G >= 1 && C % G == 0, name ": the channels must divide into the groups of B and C");        \
    FLARE_REQUIRE(B <= 65535 && C <= (1 << 20) && N <= (1 << 30) && B * N <= ((int64_t)1 << 36) / (128 * G),  \
                  name ": too large");                                                                        \
    FLARE_REQUIRE(G * ceil_div(C / G, 64) <= 65535, name ": too many groups")

// Waves a SIMD of the kernels whose lanes hold all SP states of a channel.
constexpr int lane_waves(int SP) { return SP <= 16 ? 4 : SP == 32 ? 2 : 1; }

int launch_pack(const ScanArgs& p, int dtype, int64_t SP, hipStream_t stream);
int launch_states(const ScanArgs& p, int64_t SP, hipStream_t stream);

}  // namespace scan
}  // namespace flare
