// flare_conv.hip -- the short causal convolution: forward, backward and single-token step.
//
//   pre_t = bias + sum_{k < W} w[W-1-k] x_{t-k}      (k back within the same document; before
//                                                      the first token: the cached window, or 0)
//   y_t   = pre_t, or pre_t sigmoid(pre_t)
//   d_t   = dy_t, or dy_t s (1 + pre (1 - s)), s = sigmoid(pre)
//   dx_t  = sum_k w[W-1-k] d_{t+k};   dw[W-1-k] = sum_t d_t x_{t-k};   db = sum_t d_t
//
// Channels are independent, so a thread owns 1, 2 or 4 adjacent channels and walks over a run of
// tokens with the last W inputs in registers.  Bytes bound it: each input
// is read once from memory (the W - 1 rows before a run again, from the L2) and each output
// written once.  4 x 4096 tokens of 2048 channels, bf16, W = 4: 36.4 us, 3.7 TB/s (a copy of as many
// bytes 29 us); the backward, which also recomputes pre_t, 64 us for half again as many, 3.1 TB/s.
// With documents a tap of a channel costs a select more in the forward and two in the backward: 4 x 2011
// x 1024 15 and 26 us, 13 and 19 without; vector instructions are 57% and 78% of their cycles.
#include "flare_internal.h"
#include "flare_mix.h"

namespace flare {
namespace mix {

struct ConvArgs {
    const void* x;
    int64_t x_sb, x_sn;
    const float *weight, *bias;
    const int32_t *ids, *lengths;
    const void* window;
    void *y, *window_out;
    const void* dy;
    void* dx;
    float* partial;
    int64_t B, N, C, tiles;
    int silu, run;
};

// VEC elements of a row as loaded.
template <typename E, int VEC>
struct alignas(VEC * sizeof(E)) Raw {
    E v[VEC];
    __device__ __forceinline__ void load(const E* p) { *this = *reinterpret_cast<const Raw*>(p); }
    __device__ __forceinline__ void get(float (&out)[VEC]) const {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = to_f32(v[i]);
    }
};

__device__ __forceinline__ int64_t row_length(const int32_t* lengths, int64_t b, int64_t N) {
    if (!lengths) return N;
    const int64_t n = lengths[b];
    return n < 0 ? 0 : (n > N ? N : n);
}

// How many tokens before t belong to its document, up to `most`.
__device__ __forceinline__ int tokens_back(const int32_t* ids, int64_t t, int most) {
    int n = 0;
    while (n < most && t - n > 0 && ids[t - n] == ids[t - n - 1]) ++n;
    return n;
}

// `run` tokens a thread; threads of neighbouring channels are neighbours.  U rows are loaded
// while the U before them are computed: what bounds the kernel is how many bytes are under way,
// and eight rows of four channels leave registers for seven waves a SIMD.
template <typename E, int W, int VEC, bool DOCS>
__global__ __launch_bounds__(256) void conv_forward_kernel(ConvArgs p) {
    constexpr int U = 8;
    typedef Raw<E, VEC> R;
    const int64_t groups = p.C / VEC;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= groups * p.tiles * p.B) return;
    const int64_t c = (id % groups) * VEC, tile = id / groups % p.tiles, b = id / groups / p.tiles;
    const int t0 = (int)tile * p.run, N = (int)p.N, end = min(t0 + p.run, N);
    const int len = (int)row_length(p.lengths, b, p.N);
    const E* x = (const E*)p.x + b * p.x_sb + c;
    const E* win = p.window ? (const E*)p.window + b * (W - 1) * p.C + c : nullptr;
    const int32_t* ids = DOCS ? p.ids + b * p.N : nullptr;
    E* y = (E*)p.y + b * p.N * p.C + c;
    // row t of the input: those before the first token come from the window, those that are none are 0
    auto row = [&](int t) {
        R r = {};
        if (t >= 0 && t < len) r.load(x + t * p.x_sn);
        else if (t < 0 && win) r.load(win + (t + W - 1) * p.C);
        return r;
    };
    R raw[U];
    int next_id[U] = {};
    auto fetch = [&](int u, int t) {
        if (t >= end) return;
        raw[u] = row(t);
        if (DOCS) next_id[u] = ids[t];
    };
#pragma unroll
    for (int u = 0; u < U; ++u) fetch(u, t0 + u);
    float w[W][VEC], bias[VEC], in[W][VEC];                    // in[k]: the input k tokens back
#pragma unroll
    for (int k = 1; k < W; ++k) row(t0 - k).get(in[k - 1]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        bias[i] = p.bias ? p.bias[c + i] : 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) w[k][i] = p.weight[(c + i) * W + W - 1 - k];
    }
    int back = DOCS ? tokens_back(ids, t0, W - 1) - 1 : W - 1, last_id = next_id[0];
    for (int t4 = t0; t4 < end; t4 += U) {
        R now[U];
        int id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            now[u] = raw[u];
            id[u] = next_id[u];
            fetch(u, t4 + U + u);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int t = t4 + u;
            if (t >= end) break;
            bool live = t < len;
            if (DOCS) {
                back = id[u] == last_id ? min(back + 1, W - 1) : 0;
                last_id = id[u];
                live = last_id >= 0;
            }
            float out[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
#pragma unroll
                for (int k = W - 1; k > 0; --k) in[k][i] = in[k - 1][i];
            }
            now[u].get(in[0]);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                float s = bias[i];
#pragma unroll
                for (int k = 0; k < W; ++k) s += !DOCS || k <= back ? w[k][i] * in[k][i] : 0.0f;
                if (p.silu) s *= sigmoid(s);
                out[i] = live ? s : 0.0f;
            }
            store_row<E, VEC>(y + (int64_t)t * p.C, out);
        }
    }
    // the window after the last token: inputs len-W+1 .. len-1
    if (p.window_out && tile == 0) {
        E* wo = (E*)p.window_out + b * (W - 1) * p.C + c;
#pragma unroll
        for (int r = 0; r < W - 1; ++r) {
            float v[VEC];
            row(len - (W - 1) + r).get(v);
            store_row<E, VEC>(wo + r * p.C, v);
        }
    }
}

// A thread walks over tokens t0 .. t0+run+W-2: the last W - 1 of them only for the dx of the ones
// before.  It leaves its sums for dw and db in partial [B * tiles][W + 1][C].
template <typename E, int W, int VEC, bool DOCS>
__global__ __launch_bounds__(256) void conv_backward_kernel(ConvArgs p) {
    constexpr int U = 4;
    typedef Raw<E, VEC> R;
    const int64_t groups = p.C / VEC;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= groups * p.tiles * p.B) return;
    const int64_t c = (id % groups) * VEC, tile = id / groups % p.tiles, b = id / groups / p.tiles;
    const int t0 = (int)tile * p.run, N = (int)p.N, end = min(t0 + p.run, N), stop = min(end + W - 1, N);
    const E* x = (const E*)p.x + b * p.x_sb + c;
    const E* dy = (const E*)p.dy + b * p.N * p.C + c;
    E* dx = (E*)p.dx + b * p.N * p.C + c;
    const int32_t* ids = DOCS ? p.ids + b * p.N : nullptr;
    struct Rows {
        R x, dy;
    };
    Rows raw[U];
    int next_id[U] = {};
    auto fetch = [&](int u, int t) {
        raw[u] = {};
        if (t >= stop) return;
        raw[u].x.load(x + t * p.x_sn);
        raw[u].dy.load(dy + (int64_t)t * p.C);
        if (DOCS) next_id[u] = ids[t];
    };
#pragma unroll
    for (int u = 0; u < U; ++u) fetch(u, t0 + u);
    float w[W][VEC], bias[VEC], dw[W][VEC], db[VEC];
    // in[k]: the input k tokens back; acc[k]: the dx so far of the token k back
    float in[W][VEC], acc[W][VEC];
#pragma unroll
    for (int k = 1; k < W; ++k) {
        R r = {};
        if (t0 - k >= 0 && (!DOCS || ids[t0 - k] >= 0)) r.load(x + (t0 - k) * p.x_sn);
        r.get(in[k - 1]);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        bias[i] = p.bias ? p.bias[c + i] : 0.0f;
        db[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) {
            w[k][i] = p.weight[(c + i) * W + W - 1 - k];
            dw[k][i] = acc[k][i] = 0.0f;
        }
    }
    int back = DOCS ? tokens_back(ids, t0, W - 1) - 1 : W - 1, last_id = next_id[0];
    for (int t4 = t0; t4 < end + W - 1; t4 += U) {
        Rows now[U];
        int id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            now[u] = raw[u];
            id[u] = next_id[u];
            fetch(u, t4 + U + u);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int t = t4 + u;
            if (DOCS && t < stop) {
                back = id[u] == last_id ? min(back + 1, W - 1) : 0;
                last_id = id[u];
            }
            const bool live = !DOCS || last_id >= 0;       // padding's rows are 0, whatever they hold
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
#pragma unroll
                for (int k = W - 1; k > 0; --k) {
                    in[k][i] = in[k - 1][i];
                    acc[k][i] = acc[k - 1][i];
                }
                acc[0][i] = 0.0f;
            }
            float ds[VEC];
            now[u].x.get(in[0]);
            now[u].dy.get(ds);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if (DOCS && !live) in[0][i] = ds[i] = 0.0f;
                float d = ds[i];
                if (p.silu) {
                    float s = bias[i];
#pragma unroll
                    for (int k = 0; k < W; ++k) s += !DOCS || k <= back ? w[k][i] * in[k][i] : 0.0f;
                    const float g = sigmoid(s);
                    d *= g * (1.0f + s * (1.0f - g));
                }
#pragma unroll
                for (int k = 0; k < W; ++k) {
                    acc[k][i] += !DOCS || k <= back ? w[k][i] * d : 0.0f;
                    if (t < end) dw[k][i] += !DOCS || k <= back ? d * in[k][i] : 0.0f;
                }
                if (t < end) db[i] += d;
            }
            // token t - (W-1) has all its terms
            const int done = t - (W - 1);
            if (done >= t0 && done < end) store_row<E, VEC>(dx + (int64_t)done * p.C, acc[W - 1]);
        }
    }
    float* out = p.partial + (b * p.tiles + tile) * (W + 1) * p.C + c;
#pragma unroll
    for (int k = 0; k < W; ++k) store_row<float, VEC>(out + (W - 1 - k) * p.C, dw[k]);
    store_row<float, VEC>(out + W * p.C, db);
}

// One token: the window moves on by it in place.  mask 0: nothing changes and y = 0.  64 sequences
// of 2048 channels take 3 us, the latency of a launch and of one load after the other.
template <typename E, int W, int VEC>
__global__ __launch_bounds__(256) void conv_step_kernel(ConvArgs p, const int32_t* mask) {
    const int64_t groups = p.C / VEC;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= groups * p.B) return;
    const int64_t c = (id % groups) * VEC, b = id / groups;
    float out[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = 0.0f;
    if (!mask || mask[b]) {
        E* win = (E*)p.window_out + b * (W - 1) * p.C + c;
        float in[W][VEC];
        load_row<E, VEC>((const E*)p.x + b * p.x_sb + c, in[0]);
#pragma unroll
        for (int k = 1; k < W; ++k) load_row<E, VEC>(win + (W - 1 - k) * p.C, in[k]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            float s = p.bias ? p.bias[c + i] : 0.0f;
#pragma unroll
            for (int k = 0; k < W; ++k) s += p.weight[(c + i) * W + W - 1 - k] * in[k][i];
            if (p.silu) s *= sigmoid(s);
            out[i] = s;
        }
#pragma unroll
        for (int r = 0; r < W - 1; ++r) store_row<E, VEC>(win + r * p.C, in[W - 2 - r]);
    }
    store_row<E, VEC>((E*)p.y + b * p.C + c, out);
}

// Where the column sums of [W + 1][C] go: dw [C, W] and db [C].
struct PutWeights {
    int64_t C;
    int W;
    float *dw, *db;
    __device__ __forceinline__ void operator()(int64_t col, float v) const {
        const int64_t k = col / C, c = col % C;
        if (k < W) dw[c * W + k] = v;
        else if (db) db[c] = v;
    }
};

// Tokens a thread of the backward walks over.  bf16, us with 8, 16, 32 of them, the sums of the weights'
// gradients included: 2^19 elements 10, 11, 16; 2^22 17, 16, 20; 2^23 28, 22, 25; 2^25 94, 71, 69.
static int conv_back_tokens(int64_t B, int64_t N, int64_t C) { return B * N * C >= (int64_t)1 << 24 ? 32 : 16; }

// Adjacent channels a thread takes: four where that leaves `waves` waves or more and the rows are
// aligned to it, two where it does not, and one where rows have no such alignment.  With four and with
// two, us: forward of 2^25 elements 36.4, 40.8, of 2^19 4.6, 4.3; backward of 2^22 22.2, 17.3.
template <typename E>
static int conv_vector(const ConvArgs& p, int64_t runs, int64_t waves) {
    const uintptr_t bits = (uintptr_t)p.x | (uintptr_t)p.y | (uintptr_t)p.window | (uintptr_t)p.window_out |
                           (uintptr_t)p.dy | (uintptr_t)p.dx |
                           ((uintptr_t)p.C | (uintptr_t)p.x_sb | (uintptr_t)p.x_sn) * sizeof(E);
    auto fits = [&](unsigned v) { return bits % (v * sizeof(E)) == 0 && (uintptr_t)p.partial % (v * sizeof(float)) == 0; };
    if (fits(4) && p.B * runs * (p.C / 4) >= waves * 64) return 4;
    return fits(2) ? 2 : 1;
}

template <typename E, int VEC>
static int conv_forward_w(const ConvArgs& p, int64_t W, hipStream_t stream) {
    const dim3 g((unsigned)ceil_div(p.B * (p.C / VEC) * p.tiles, 256));
    auto kernel = W == 2   ? (p.ids ? conv_forward_kernel<E, 2, VEC, true> : conv_forward_kernel<E, 2, VEC, false>)
                  : W == 3 ? (p.ids ? conv_forward_kernel<E, 3, VEC, true> : conv_forward_kernel<E, 3, VEC, false>)
                           : (p.ids ? conv_forward_kernel<E, 4, VEC, true> : conv_forward_kernel<E, 4, VEC, false>);
    kernel<<<g, 256, 0, stream>>>(p);
    return check_launch("conv_forward");
}
template <typename E>
static int conv_forward_e(ConvArgs p, int64_t W, hipStream_t stream) {
    // Long runs read the W - 1 rows before a run less often, short ones spread a small call over the
    // GPU.  bf16, us with runs of 4, 8, 16 tokens: 2^19 elements 4.3, 4.7, 7.0; 2^22 8.2, 8.1, 9.7; 2^23 13.2,
    // 12.7, 14.4; 2^25 43.9, 40.4, 36.4.
    const int64_t work = p.B * p.N * p.C;
    p.run = work >= (int64_t)1 << 24 ? 16 : work >= (int64_t)1 << 22 ? 8 : 4;
    p.tiles = ceil_div(p.N, p.run);
    const int v = conv_vector<E>(p, p.tiles, 2048);
    return v == 1 ? conv_forward_w<E, 1>(p, W, stream) : v == 2 ? conv_forward_w<E, 2>(p, W, stream)
                                                                : conv_forward_w<E, 4>(p, W, stream);
}

template <typename E, int VEC>
static int conv_backward_w(const ConvArgs& p, int64_t W, hipStream_t stream) {
    const dim3 g((unsigned)ceil_div(p.B * (p.C / VEC) * p.tiles, 256));
    auto kernel = W == 2   ? (p.ids ? conv_backward_kernel<E, 2, VEC, true> : conv_backward_kernel<E, 2, VEC, false>)
                  : W == 3 ? (p.ids ? conv_backward_kernel<E, 3, VEC, true> : conv_backward_kernel<E, 3, VEC, false>)
                           : (p.ids ? conv_backward_kernel<E, 4, VEC, true> : conv_backward_kernel<E, 4, VEC, false>);
    kernel<<<g, 256, 0, stream>>>(p);
    return check_launch("conv_backward");
}
template <typename E>
static int conv_backward_e(ConvArgs p, int64_t W, hipStream_t stream) {
    p.run = conv_back_tokens(p.B, p.N, p.C);
    p.tiles = ceil_div(p.N, p.run);
    const int v = conv_vector<E>(p, p.tiles, 4096);
    return v == 1 ? conv_backward_w<E, 1>(p, W, stream) : v == 2 ? conv_backward_w<E, 2>(p, W, stream)
                                                                 : conv_backward_w<E, 4>(p, W, stream);
}

template <typename E, int VEC>
static int conv_step_w(const ConvArgs& p, int64_t W, const int32_t* mask, hipStream_t stream) {
    const dim3 g((unsigned)ceil_div(p.B * (p.C / VEC), 256));
    if (W == 2) conv_step_kernel<E, 2, VEC><<<g, 256, 0, stream>>>(p, mask);
    else if (W == 3) conv_step_kernel<E, 3, VEC><<<g, 256, 0, stream>>>(p, mask);
    else conv_step_kernel<E, 4, VEC><<<g, 256, 0, stream>>>(p, mask);
    return check_launch("conv_step");
}
template <typename E>
static int conv_step_e(const ConvArgs& p, int64_t W, const int32_t* mask, hipStream_t stream) {
    return conv_vector<E>(p, 1, 512) == 1 ? conv_step_w<E, 1>(p, W, mask, stream) : conv_step_w<E, 2>(p, W, mask, stream);
}

static size_t conv_backward_bytes(int64_t B, int64_t N, int64_t C, int64_t W) {
    return (size_t)(B * ceil_div(N, conv_back_tokens(B, N, C))) * (W + 1) * C * sizeof(float);
}

}  // namespace mix
}  // namespace flare

using namespace flare;
using namespace flare::mix;

#define CONV_REQUIRE_SIZES(name)                                                                             \
    FLARE_REQUIRE(known_dtype(dtype), name ": unknown dtype %d", dtype);                                     \
    FLARE_REQUIRE(B >= 1 && N >= 1 && C >= 1, name ": B, N and C must be positive");                         \
    FLARE_REQUIRE(W >= 2 && W <= 4, name ": W must be 2, 3 or 4, got %lld", (long long)W);                   \
    FLARE_REQUIRE(B <= INT32_MAX && N <= (1 << 30) && C <= (1 << 20) && B * N <= ((int64_t)1 << 38) / C,      \
                  name ": too large")

extern "C" int flare_conv_forward(const void* x, int64_t x_stride_b, int64_t x_stride_n, const float* weight,
                                  const float* bias, int silu, int dtype, int64_t B, int64_t N, int64_t C, int64_t W,
                                  const int32_t* document_ids, const int32_t* lengths, const void* window, void* y,
                                  void* window_out, void* stream) {
    CONV_REQUIRE_SIZES("flare_conv_forward");
    FLARE_REQUIRE(x && weight && y, "flare_conv_forward: null pointer");
    FLARE_REQUIRE(!(document_ids && (lengths || window || window_out)),
                  "flare_conv_forward: document_ids exclude lengths and windows");
    FLARE_REQUIRE(!window_out || window_out != window, "flare_conv_forward: the windows overlap");
    ConvArgs p = {};
    p.x = x, p.x_sb = x_stride_b, p.x_sn = x_stride_n, p.weight = weight, p.bias = bias, p.ids = document_ids;
    p.lengths = lengths, p.window = window, p.y = y, p.window_out = window_out, p.B = B, p.N = N, p.C = C;
    p.silu = silu;
    return FLARE_BY_DTYPE(dtype, conv_forward_e, (p, W, (hipStream_t)stream));
}

extern "C" size_t flare_conv_backward_workspace_size(int64_t B, int64_t N, int64_t C, int64_t W) {
    return conv_backward_bytes(B, N, C, W);
}

extern "C" int flare_conv_backward(const void* x, int64_t x_stride_b, int64_t x_stride_n, const float* weight,
                                   const float* bias, int silu, int dtype, int64_t B, int64_t N, int64_t C, int64_t W,
                                   const int32_t* document_ids, const void* dy, void* dx, float* dweight,
                                   float* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    CONV_REQUIRE_SIZES("flare_conv_backward");
    FLARE_REQUIRE(x && weight && dy && dx && dweight && workspace, "flare_conv_backward: null pointer");
    if (workspace_bytes < conv_backward_bytes(B, N, C, W)) {
        set_error("flare_conv_backward: workspace of %zu bytes is too small", workspace_bytes);
        return FLARE_ERR_WORKSPACE;
    }
    ConvArgs p = {};
    p.x = x, p.x_sb = x_stride_b, p.x_sn = x_stride_n, p.weight = weight, p.bias = bias, p.ids = document_ids;
    p.dy = dy, p.dx = dx, p.partial = (float*)workspace, p.B = B, p.N = N, p.C = C, p.silu = silu;
    const int rc = FLARE_BY_DTYPE(dtype, conv_backward_e, (p, W, (hipStream_t)stream));
    if (rc != FLARE_OK) return rc;
    const int64_t rows = B * ceil_div(N, conv_back_tokens(B, N, C)), cols = (W + 1) * C;
    return launch_column_sums(p.partial, rows, cols, PutWeights{C, (int)W, dweight, dbias}, (hipStream_t)stream);
}

extern "C" int flare_conv_step(const void* x, int64_t x_stride_b, const float* weight, const float* bias, int silu,
                               int dtype, int64_t B, int64_t C, int64_t W, const int32_t* mask, void* window, void* y,
                               void* stream) {
    const int64_t N = 1;
    CONV_REQUIRE_SIZES("flare_conv_step");
    FLARE_REQUIRE(x && weight && window && y, "flare_conv_step: null pointer");
    ConvArgs p = {};
    p.x = x, p.x_sb = x_stride_b, p.weight = weight, p.bias = bias, p.window_out = window, p.y = y;
    p.B = B, p.N = 1, p.C = C, p.silu = silu;
    return FLARE_BY_DTYPE(dtype, conv_step_e, (p, W, mask, (hipStream_t)stream));
}
