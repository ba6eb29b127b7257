// flare_attn.hip -- softmax attention: C entry points, id statistics, and writing prompts to caches.
#include "flare_internal.h"
#include "flare_qcache.h"

namespace flare {
namespace attn {

template <typename E> int forward_e(const AttnArgs& p, hipStream_t stream);
template <typename E> int backward_e(const AttnArgs& p, float* delta, float* norms, float* ranges, hipStream_t stream);
template <typename E, int BITS> int forward_bits(const AttnArgs& p, hipStream_t stream);
template <typename E, int BITS> int rows_e(const AttnArgs& p, int tiles, hipStream_t stream);
int attn_step(const AttnArgs& p, int dtype, hipStream_t stream);

// A wave for each 64 tokens.
__global__ __launch_bounds__(64) void attn_ids_kernel(const int32_t* ids, int64_t N, int32_t* stats) {
    const int64_t tile = blockIdx.x, b = blockIdx.y, t = tile * kIdTile + threadIdx.x;
    const bool there = t < N;
    const int id = there ? ids[b * N + t] : 0;
    int lo = there && id >= 0 ? id : INT32_MAX, hi = there && id >= 0 ? id : -1;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        lo = min(lo, __shfl_xor(lo, o, 64));
        hi = max(hi, __shfl_xor(hi, o, 64));
    }
    const bool negative = __any(there && id < 0);
    if (threadIdx.x == 0) {
        int32_t* s = stats + (b * gridDim.x + tile) * 3;
        s[0] = lo, s[1] = hi, s[2] = lo == hi && !negative;
    }
}

// What each block of `rows` queries (blockIdx.y 0) or `key_rows` keys (1) costs: the tiles of ids it
// meets.  A wave a block.
__global__ __launch_bounds__(64) void attn_costs_kernel(AttnArgs p, int rows, int key_rows, int32_t* costs,
                                                        int32_t* key_costs) {
    const bool keys = blockIdx.y != 0;
    const int n = keys ? key_rows : rows, tiles = ((int)p.N + n - 1) / n;
    if ((int64_t)blockIdx.x >= p.B * tiles) return;
    const int b = blockIdx.x / tiles, first = blockIdx.x % tiles * n, all = id_tiles(p.N);
    const IdRange mine = id_block(p, b, first, n);
    const int from = p.causal && keys ? first / kIdTile : 0;
    const int to = p.causal && !keys ? min(all, (first + n + kIdTile - 1) / kIdTile) : all;
    int cost = 0;
    for (int t = from; t < to; t += 64) {
        const int at = t + threadIdx.x;
        cost += __popcll(__ballot(at < to && id_range(p, b, at).meets(mine)));
    }
    if (threadIdx.x == 0) (keys ? key_costs : costs)[blockIdx.x] = cost;
}

constexpr int kMostOrdered = 2048;

// Blocks in falling order of cost, those of one cost as they stand.
__global__ __launch_bounds__(1024) void attn_order_kernel(const int32_t* costs, int n, int32_t* order,
                                                          const int32_t* key_costs, int key_n, int32_t* key_order) {
    __shared__ int c[kMostOrdered];
    if (blockIdx.x) costs = key_costs, n = key_n, order = key_order;
    for (int i = threadIdx.x; i < n; i += 1024) c[i] = costs[i];
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 1024) {
        const int mine = c[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += c[j] > mine || (c[j] == mine && j < i);
        order[rank] = i;
    }
}

// New keys and values to their place behind what each sequence's cache holds.  Nothing of a
// sequence that does not fit.
__global__ __launch_bounds__(256) void attn_append_kernel(Rows k, Rows v, const int32_t* lengths, const int32_t* fresh,
                                                          int64_t B, int64_t N, int64_t M, int64_t row_bytes,
                                                          int64_t G, int64_t size, char* kc, char* vc) {
    const int64_t per = row_bytes / 16, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= B * N * G * per) return;
    const int64_t at = id % per * 16, g = id / per % G, t = id / per / G % N, b = id / per / G / N;
    const int64_t off = lengths[b], n = fresh ? clamp_to(fresh[b], N) : N;
    if (off < 0 || off + n > M || t >= n) return;
    const int64_t to = ((b * M + off + t) * G + g) * row_bytes + at;
    *reinterpret_cast<u32x4*>(kc + to) =
        *reinterpret_cast<const u32x4*>((const char*)k.p + (b * k.sb + t * k.sn + g * k.sh) * size + at);
    *reinterpret_cast<u32x4*>(vc + to) =
        *reinterpret_cast<const u32x4*>((const char*)v.p + (b * v.sb + t * v.sn + g * v.sh) * size + at);
}

static int rows_of_queries(int dtype) { return 64 * q_tiles(dtype == FLARE_F32 ? 4 : 2); }
static int rows_of_keys(int dtype, int64_t D) {
    return 64 * kv_tiles(dtype == FLARE_F32 ? 4 : 2, (int)ceil_div(D, 32) * 32);
}
// Of the id statistics, and of two costs and orders.
static size_t stats_bytes(int64_t B, int64_t N) {
    return (size_t)(B * ceil_div(N, kIdTile) * 3 + 4 * kMostOrdered) * sizeof(int32_t);
}

// Documents make blocks cost very different amounts of work, so that the costly ones have to start
// first; that takes two small launches (some 10 us), and pays where there are more workgroups
// than run at once (512).  16384 tokens in six documents, 16 heads of 128 over 4, us in the rows'
// order and in this: forward 598, 555; dq 749, 693; dk and dv 1121, 1049.
static int launch_ids(AttnArgs& p, int dtype, bool keys, int32_t* stats, hipStream_t stream) {
    if (!p.ids) return FLARE_OK;
    const int tiles = (int)ceil_div(p.N, kIdTile);
    attn_ids_kernel<<<dim3((unsigned)tiles, (unsigned)p.B), 64, 0, stream>>>(p.ids, p.N, stats);
    p.id_stats = stats;
    int rc = check_launch("attn_ids");
    const int rows = rows_of_queries(dtype), key_rows = rows_of_keys(dtype, p.D);
    const int64_t n = p.B * ceil_div(p.N, rows), key_n = keys ? p.B * ceil_div(p.N, key_rows) : 0;
    if (rc != FLARE_OK || n * p.H <= 512 || n > kMostOrdered || key_n > kMostOrdered) return rc;
    int32_t* at = stats + p.B * tiles * 3;
    attn_costs_kernel<<<dim3((unsigned)(n > key_n ? n : key_n), keys ? 2 : 1), 64, 0, stream>>>(p, rows, key_rows, at,
                                                                                             at + kMostOrdered);
    if ((rc = check_launch("attn_costs")) != FLARE_OK) return rc;
    attn_order_kernel<<<dim3(keys ? 2 : 1), 1024, 0, stream>>>(at, (int)n, at + 2 * kMostOrdered, at + kMostOrdered,
                                                               (int)key_n, at + 3 * kMostOrdered);
    p.order = at + 2 * kMostOrdered;
    p.key_order = keys ? at + 3 * kMostOrdered : nullptr;
    return check_launch("attn_order");
}

// Parts that the queries of each block of keys are split into (blocks of keys cost very different
// amounts of work under a causal or document mask): the heads that share them until there are 2048
// workgroups, and then the rows until there are 1024, in parts of 256 or more.  us, the parts' sums
// included: 16384 rows, 16 heads of 128 over 4, two parts 3245, one 3334; 2 x 2048 rows, 16 heads of 64,
// four parts of the rows 113, two 94, one 99.  The keys of each block of rows likewise, for dq: 1024
// workgroups for that call 54 us, 512 (one part) 80.
constexpr int64_t kDqBlocks = 1024;
static void split_backward(AttnArgs& p, int dtype) {
    const int64_t blocks = ceil_div(p.N, rows_of_keys(dtype, p.D));
    const int64_t R = p.H / p.G;
    int64_t want = ceil_div(2048, blocks * p.B * p.G);
    want = want > 8 ? 8 : want;
    const int64_t heads = want < R ? want : R, most = ceil_div(p.N, 256);
    int64_t rows = ceil_div(1024, blocks * p.B * p.G * heads);
    rows = rows * heads > 8 ? ceil_div(8, heads) : rows;
    p.row_splits = rows < most ? rows : most;
    p.splits = heads * p.row_splits;
    const int64_t dq_want = ceil_div(kDqBlocks, ceil_div(p.N, rows_of_queries(dtype)) * p.B * p.H);
    p.dq_splits = dq_want < most ? dq_want : most;
}
static size_t parts_bytes(const AttnArgs& p) {
    return p.splits == 1 ? 0 : (size_t)(p.splits * 2 * p.B * p.N * p.G * p.D) * sizeof(float);
}
static size_t dq_bytes(const AttnArgs& p) {
    return p.dq_splits == 1 ? 0 : (size_t)(p.dq_splits * p.B * p.N * p.H * p.D) * sizeof(float);
}

// Parts that a row's keys are split into in the forward: two workgroups a CU (512) where the rows
// leave less than that, in parts of 512 keys or more.  us, the joining included, with parts and
// without: 64 new tokens behind 8000, 16 heads of 128 over 4, 34 and 274; 2 x 512 behind 3000 55 and 118.
// A round of workgroups under a causal mask alone is as long as its last rows, and two parts even that
// out, up to five quarters of a round.  us without parts and with two, 16 heads of 128 over 4: 4096 rows
// (512 workgroups) 151, 127; 4608 172, 154; 5120 (640) 193, 186; 5632 215, 219; 6400 251, 270.  16 heads of 64:
// 4096 106, 78; 5120 136, 114; 6400 174, 169.  (4096 in documents of 700 tokens 57, 98; with a prefix of 2000
// 155, 153; 2048 behind 2048 in a cache 163, 172.)
static void split_forward(AttnArgs& p, int dtype) {
    const int64_t blocks = ceil_div(p.N, rows_of_queries(dtype)) * p.B * p.H, most = ceil_div(p.M, 512);
    int64_t want = ceil_div(512, blocks);
    if (want < 2 && blocks <= 640 && p.causal && p.M == p.N && !p.ids && !p.prefix) want = 2;
    p.splits = want < most ? want : most;
}
static size_t forward_head_bytes(int64_t B, int64_t N) { return (stats_bytes(B, N) + 255) / 256 * 256; }
static size_t rows_bytes(const AttnArgs& p) {
    return p.splits == 1 ? 0 : (size_t)(p.B * p.H * p.N * p.splits * (p.D + 4)) * sizeof(float);
}

// Workgroups of the step kernel for each sequence's keys: enough for one on each CU (256 on the
// card), whose four waves have the loads under way that its memory takes, and no more than the cache
// has shares of 128 keys.  us, the joining included, for 256, 512 and 1024: 64 sequences of 8000
// tokens, 4 key heads of 128, bf16, 182, 194, 198; 16 of them 47, 48, 50; one 13 with any.
static int64_t step_splits(int64_t B, int64_t M, int64_t H, int64_t G) {
    const int64_t rows = B * G * ceil_div(H / G, 16), s = ceil_div(256, rows), most = ceil_div(M, 128);
    return s < 1 ? 1 : (s > most ? most : s);
}

// Tiles of 16 rows (token, head) a wave of qattn_rows owns.
static int row_tiles(int64_t N, int64_t H, int64_t G, int dtype) { return H / G * N > 16 && dtype != FLARE_F32 ? 2 : 1; }

// Which kernel takes N new tokens over a cache of 8 or 4 bits.  kRows: rows of the heads that share keys, in groups of 16
// or 32, whose codes go straight into operands.  kFused: attn_forward with the codes turned into values as they go to
// LDS, once for each 128 tokens of each head.  kExpanded: attn_forward over 16-bit values that the codes are turned
// into first.
//   A group of 32 rows takes a third of what 128 tokens of a head take.  us, fused and by rows, 16 heads of 128 over 4,
// 4 bits, behind 8192 tokens of 16 sequences: 32 new tokens 177, 86; 64 185, 124; 128 195, 232; behind 1000 of one, 64 31,
// 21.  fp32 queries, 8 heads of 64, behind 4096 of 16: 32 new tokens 106, 55; 512 595, 304: these always go by rows.
//   Values turned into 16 bits once pay from 16 blocks that read them.  us, fused and expanded: 16 x 256 new tokens behind
// 8192, 348, 396; 512 (16 blocks) 684, 689; 2048 2512, 2218; one sequence, 1024 behind 15,300 191, 180; 2048 351, 317.
// That is a tenth of the time for memory that a cache of 4 bits was chosen to save, and rooms count whole, whatever they
// hold: 1 GiB of values at a time, and sequences whose values are more go by their codes.
enum { kRows, kFused, kExpanded };
constexpr int64_t kExpandBlocks = 16, kMostExpanded = (int64_t)1 << 30;      // bytes of values
static int64_t expanded_row(int64_t G, int64_t D) { return 2 * 2 * G * D; }  // of a token, k and v
static int qattn_path(int64_t N, int64_t M, int64_t H, int64_t G, int64_t D, int dtype) {
    const int64_t R = H / G, blocks = R * ceil_div(N, 128);
    if (dtype == FLARE_F32 || ceil_div(R * N, 32) <= 3 * blocks) return kRows;
    return blocks < kExpandBlocks || M * expanded_row(G, D) > kMostExpanded ? kFused : kExpanded;
}
// Sequences that are expanded at a time.
static int64_t expand_slice(int64_t B, int64_t M, int64_t G, int64_t D) {
    const int64_t s = kMostExpanded / (M * expanded_row(G, D));
    return s < 1 ? 1 : (s > B ? B : s);
}
static size_t expanded_bytes(int64_t B, int64_t M, int64_t G, int64_t D) {
    return (size_t)(B * M * expanded_row(G, D) + 255) / 256 * 256;
}

// Key heads of the same tokens that the waves of a workgroup take side by side: their rows share lines of memory, which
// tells where bytes bound the call.  us, one head a workgroup and four: 64 x 8192 tokens, 8 bits, 4 key heads of 128 110,
// 100; 8 of 64 127, 112; in 4 bits 97, 80, and 4 of 128 67, 66; one sequence of 1000 10.6, 13.6, as its keys have fewer
// waves then; 256 x 1024, 4 bits, 4 of 128 36, 44, as one head a workgroup needs no shares to be joined.
static int64_t rows_heads(int64_t B, int64_t M, int64_t G, int tiles) {
    if (tiles > 1 || B * G < 128 || (B * G >= 768 && M < 4096)) return 1;
    return G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1;
}
// Workgroups for each sequence's keys: three on a CU, two where a wave's tiles, parts or codes leave registers for no more,
// with shares of 256 keys a head, or of 128 until there are 32.  us, workgroups of 512, 768 and 1024, 64 x 8192 tokens, 4 key
// heads of 128: 4 bits 75, 66, 69; 8 bits 100, 106, 111; fp32 queries 80, 99, 86; five tokens, 8 bits, 16 x 8192
// 45, 55, 54 (with a launch to write them).  16 x 4096 in 8 bits, 16 heads of 64 43, 39, 41.  Shares of 128 and
// of 256 for one sequence of 1000 10.0, 11.1; of 4000 10.5, 11.7; of 16384 (128 and 64 of them) 14.4, 12.5.
static int64_t rows_splits(int64_t B, int64_t N, int64_t M, int64_t H, int64_t G, int64_t D, int dtype, int bits) {
    const int tiles = row_tiles(N, H, G, dtype);
    const int64_t heads = rows_heads(B, M, G, tiles), rows = B * (G / heads) * ceil_div(H / G * N, 16 * tiles);
    const bool three = tiles == 1 && dtype != FLARE_F32 && D * bits <= 512;
    const int64_t s = ceil_div(three ? 768 : 512, rows), small = ceil_div(M, 128);
    int64_t most = ceil_div(M, 256 / heads);
    if (heads == 1 && most < 32) most = small < 32 ? small : 32;
    return s < 1 ? 1 : (s > most ? most : s);
}
// Workgroups of the largest launch of a call.  (Where attn_forward splits its keys there are few.)
static int64_t qattn_blocks(int64_t B, int64_t N, int64_t M, int64_t H, int64_t G, int64_t D, int dtype, int bits) {
    const int path = qattn_path(N, M, H, G, D, dtype), tiles = row_tiles(N, H, G, dtype);
    if (path != kRows)
        return ceil_div(N, rows_of_queries(dtype)) * H * (path == kFused ? B : expand_slice(B, M, G, D));
    const int64_t units = rows_splits(B, N, M, H, G, D, dtype, bits) * B * ceil_div(H / G * N, 16 * tiles);
    return ceil_div(units, 8) * 8 * (G / rows_heads(B, M, G, tiles));
}
template <typename E>
static int qattn_rows(const AttnArgs& p, int bits, int tiles, hipStream_t stream) {
    return bits == 8 ? rows_e<E, 8>(p, tiles, stream) : rows_e<E, 4>(p, tiles, stream);
}
template <typename E>
static int qattn_forward(const AttnArgs& p, int bits, hipStream_t stream) {
    return bits == 8 ? forward_bits<E, 8>(p, stream) : forward_bits<E, 4>(p, stream);
}

// attn_forward's splits over values turned into 16 bits.  Where its blocks are more than a round of workgroups (512) but
// less than one and a half, or may be many without a row that is real, two parts even the last round out.  us, one part
// and two, 16 heads of 128 over 4: 4608 rows (576 blocks) behind 8000 625, 545; 5120 707, 574; 6144 (768) 777, 661; 8192
// (1024) 929, 937; 2700 to 4096 real rows of 4096 (512) behind 11000 610, 494; all of 4 x 1024 behind 7000 (512) 314, 334.
static void split_expanded(AttnArgs& p, int dtype, bool ragged) {
    split_forward(p, dtype);
    const int64_t blocks = ceil_div(p.N, rows_of_queries(dtype)) * p.B * p.H;
    if (p.splits == 1 && p.M > 512 && blocks <= 768 && (blocks > 512 || ragged)) p.splits = 2;
}

static int qattn_expanded(const AttnArgs& all, int dtype, int bits, void* workspace, hipStream_t stream) {
    // one slice of sequences after another, in the same workspace
    const int64_t slice = expand_slice(all.B, all.M, all.G, all.D), row = all.G * all.D, codes = row * bits / 8;
    const int64_t scales = all.G * qcache::row_scales(all.D);
    for (int64_t b = 0; b < all.B; b += slice) {
        AttnArgs p = all;
        p.B = slice < all.B - b ? slice : all.B - b;
        const int64_t held = b * p.M;
        p.q.p = (const char*)all.q.p + b * p.q.sb * 2, p.y = (char*)all.y + b * p.N * p.H * p.D * 2;
        p.lengths = all.lengths + b, p.fresh = all.fresh ? all.fresh + b : nullptr;
        p.prefix = all.prefix ? all.prefix + b : nullptr;
        p.k.p = (const char*)all.k.p + held * codes, p.v.p = (const char*)all.v.p + held * codes;
        p.k_scale = all.k_scale + held * scales, p.v_scale = all.v_scale + held * scales;
        char* k = (char*)workspace;
        char* v = k + slice * p.M * row * 2;
        int rc = qcache::qcache_expand(p, dtype, bits, k, v, stream);
        if (rc != FLARE_OK) return rc;
        p.k = {k, p.M * row, row, p.D}, p.v = {v, p.M * row, row, p.D};
        split_expanded(p, dtype, p.fresh != nullptr);
        p.parts = (float*)(k + expanded_bytes(slice, p.M, p.G, p.D));
        rc = dtype == FLARE_BF16 ? forward_e<__hip_bfloat16>(p, stream) : forward_e<__half>(p, stream);
        if (rc != FLARE_OK) return rc;
    }
    return FLARE_OK;
}

}  // namespace attn
}  // namespace flare

using namespace flare;
using namespace flare::attn;

#define ATTN_REQUIRE_SIZES(name)                                                                                  \
    FLARE_REQUIRE(known_dtype(dtype), name ": unknown dtype %d", dtype);                                          \
    FLARE_REQUIRE(B >= 1 && N >= 1 && M >= 1 && H >= 1 && G >= 1, name ": sizes must be positive");               \
    FLARE_REQUIRE(H % G == 0, name ": the query heads must divide into the key heads");                           \
    FLARE_REQUIRE(D >= 16 && D <= 128 && D % 16 == 0, name ": head dimension %lld is not a multiple of 16 up to " \
                  "128", (long long)D);                                                                           \
    FLARE_REQUIRE(N <= (1 << 30) && M <= (1 << 30) && B <= 65535 && H <= 65535 && B * H <= (1 << 24) &&           \
                  (N + 63) / 64 * B * H <= (1 << 26) && H * D < kMostStride, name ": too large");            \
    FLARE_REQUIRE(softcap == 0.0f || (softcap >= kLeastCap && softcap <= kMostCap),                                \
                  name ": the cap must be 0 (none) or between 2^-100 and 2^100")

static AttnArgs attn_args(const void* q, const void* k, const void* v, const int64_t* st, int64_t B, int64_t N,
                          int64_t M, int64_t H, int64_t G, int64_t D, float scale, float softcap,
                          const float* slopes) {
    AttnArgs p = {};
    p.q = {q, st[0], st[1], st[2]}, p.k = {k, st[3], st[4], st[5]}, p.v = {v, st[6], st[7], st[8]};
    p.B = B, p.N = N, p.M = M, p.H = H, p.G = G, p.D = D, p.scale = scale, p.cap = softcap, p.slopes = slopes;
    return p;
}

extern "C" size_t flare_attn_forward_workspace_size(int64_t B, int64_t N, int64_t M, int64_t H, int64_t D, int dtype) {
    if (B < 1 || N < 1 || M < 1 || H < 1) return 0;
    AttnArgs p = {};
    p.B = B, p.N = N, p.M = M, p.H = H, p.D = D, p.causal = 1;       // which needs the most
    split_forward(p, dtype);
    return forward_head_bytes(B, N) + rows_bytes(p);
}

extern "C" int flare_attn_forward(const void* q, const void* k, const void* v, const int64_t* strides, int dtype,
                                  int64_t B, int64_t N, int64_t M, int64_t H, int64_t G, int64_t D, float scale,
                                  float softcap, const float* slopes, int causal, const int32_t* document_ids,
                                  const int32_t* prefix_lengths, const int32_t* lengths, const int32_t* new_lengths,
                                  void* y, void* y_rest, float* lse, void* workspace, size_t workspace_bytes,
                                  void* stream) {
    FLARE_REQUIRE(q && k && v && strides && y, "flare_attn_forward: null pointer");
    ATTN_REQUIRE_SIZES("flare_attn_forward");
    FLARE_REQUIRE(lengths || M == N, "flare_attn_forward: as many keys as queries without a cache");
    FLARE_REQUIRE(!(document_ids && lengths), "flare_attn_forward: document_ids exclude a cache");
    FLARE_REQUIRE(lengths || !new_lengths, "flare_attn_forward: new_lengths without lengths");
    AttnArgs p = attn_args(q, k, v, strides, B, N, M, H, G, D, scale, softcap, slopes);
    const uintptr_t out = (uintptr_t)y | (uintptr_t)y_rest;
    FLARE_REQUIRE(aligned(p.q, dtype) && aligned(p.k, dtype) && aligned(p.v, dtype) && (out & 15) == 0,
                  "flare_attn_forward: rows must be 16-byte aligned and less than 2^22 elements apart");
    p.causal = causal, p.ids = document_ids, p.prefix = prefix_lengths, p.lengths = lengths, p.fresh = new_lengths;
    p.y = y, p.y_rest = y_rest, p.lse = lse;
    split_forward(p, dtype);
    p.parts = (float*)((char*)workspace + forward_head_bytes(B, N));
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < forward_head_bytes(B, N) + rows_bytes(p)) {
        set_error("flare_attn_forward: workspace of %zu bytes is too small or not 16-byte aligned", workspace_bytes);
        return FLARE_ERR_WORKSPACE;
    }
    const int rc = launch_ids(p, dtype, false, (int32_t*)workspace, (hipStream_t)stream);
    if (rc != FLARE_OK) return rc;
    return FLARE_BY_DTYPE(dtype, forward_e, (p, (hipStream_t)stream));
}

// delta, fp16's norms and ranges, and the id statistics.
static int64_t norms_floats(int64_t B, int64_t N, int64_t H, int dtype) { return dtype == FLARE_F16 ? B * H * N : 0; }
static int64_t ranges_floats(int64_t B, int64_t N, int dtype) {
    return dtype == FLARE_F16 ? B * ceil_div(N, kIdTile) * 2 : 0;
}
static size_t backward_head_bytes(int64_t B, int64_t N, int64_t H, int dtype) {
    const int64_t floats = B * H * N + norms_floats(B, N, H, dtype) + ranges_floats(B, N, dtype);
    return ((size_t)floats * sizeof(float) + stats_bytes(B, N) + 255) / 256 * 256;
}
extern "C" size_t flare_attn_backward_workspace_size(int64_t B, int64_t N, int64_t H, int64_t G, int64_t D, int dtype) {
    if (B < 1 || N < 1 || H < 1 || G < 1 || H % G) return 0;
    AttnArgs p = {};
    p.B = B, p.N = N, p.H = H, p.G = G, p.D = D;
    split_backward(p, dtype);
    return backward_head_bytes(B, N, H, dtype) + parts_bytes(p) + dq_bytes(p);
}

extern "C" int flare_attn_backward(const void* q, const void* k, const void* v, const int64_t* strides, int dtype,
                                   int64_t B, int64_t N, int64_t H, int64_t G, int64_t D, float scale, float softcap,
                                   const float* slopes, int causal, const int32_t* document_ids,
                                   const int32_t* prefix_lengths, const void* y, const void* y_rest,
                                   const float* lse, const void* dy,
                                   void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
                                   void* stream) {
    const int64_t M = N;
    FLARE_REQUIRE(q && k && v && strides && y && lse && dy && dq && dk && dv && workspace,
                  "flare_attn_backward: null pointer");
    ATTN_REQUIRE_SIZES("flare_attn_backward");
    AttnArgs p = attn_args(q, k, v, strides, B, N, M, H, G, D, scale, softcap, slopes);
    const uintptr_t out = (uintptr_t)y | (uintptr_t)y_rest | (uintptr_t)dy | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv;
    FLARE_REQUIRE(aligned(p.q, dtype) && aligned(p.k, dtype) && aligned(p.v, dtype) && (out & 15) == 0 &&
                  ((uintptr_t)workspace & 15) == 0,
                  "flare_attn_backward: rows must be 16-byte aligned and less than 2^22 elements apart");
    if (workspace_bytes < flare_attn_backward_workspace_size(B, N, H, G, D, dtype)) {
        set_error("flare_attn_backward: workspace of %zu bytes is too small", workspace_bytes);
        return FLARE_ERR_WORKSPACE;
    }
    float* delta = (float*)workspace;
    float* norms = delta + B * H * N;
    float* ranges = norms + norms_floats(B, N, H, dtype);
    int32_t* stats = (int32_t*)(ranges + ranges_floats(B, N, dtype));
    p.causal = causal, p.ids = document_ids, p.prefix = prefix_lengths;
    p.y = const_cast<void*>(y), p.y_rest = const_cast<void*>(y_rest), p.lse = const_cast<float*>(lse), p.dy = dy;
    p.delta = delta, p.norms = norms, p.ranges = ranges;
    p.dq = dq, p.dk = dk, p.dv = dv;
    split_backward(p, dtype);
    p.parts = (float*)((char*)workspace + backward_head_bytes(B, N, H, dtype));
    p.dq_parts = (float*)((char*)p.parts + parts_bytes(p));
    const int rc = launch_ids(p, dtype, true, stats, (hipStream_t)stream);
    if (rc != FLARE_OK) return rc;
    return FLARE_BY_DTYPE(dtype, backward_e, (p, delta, norms, ranges, (hipStream_t)stream));
}

extern "C" int flare_attn_append(const void* k, const void* v, const int64_t* strides, int dtype, int64_t B, int64_t N,
                                 int64_t M, int64_t G, int64_t D, const int32_t* lengths, const int32_t* new_lengths,
                                 void* k_cache, void* v_cache, void* stream) {
    const int64_t H = G;
    const float softcap = 0.0f;
    FLARE_REQUIRE(k && v && strides && lengths && k_cache && v_cache, "flare_attn_append: null pointer");
    ATTN_REQUIRE_SIZES("flare_attn_append");
    const Rows kr = {k, strides[0], strides[1], strides[2]}, vr = {v, strides[3], strides[4], strides[5]};
    FLARE_REQUIRE(aligned(kr, dtype) && aligned(vr, dtype) && (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0,
                  "flare_attn_append: rows must be 16-byte aligned and less than 2^22 elements apart");
    const int64_t size = dtype == FLARE_F32 ? 4 : 2, work = B * N * G * (D * size / 16);
    FLARE_REQUIRE(work <= (int64_t)INT32_MAX * 256, "flare_attn_append: too large");
    attn_append_kernel<<<dim3((unsigned)ceil_div(work, 256)), 256, 0, (hipStream_t)stream>>>(
        kr, vr, lengths, new_lengths, B, N, M, D * size, G, size, (char*)k_cache, (char*)v_cache);
    return check_launch("attn_append");
}

extern "C" size_t flare_attn_step_workspace_size(int64_t B, int64_t M, int64_t H, int64_t G, int64_t D) {
    if (B < 1 || M < 1 || G < 1 || H % G) return 0;
    const int64_t s = step_splits(B, M, H, G);
    return s == 1 ? 0 : (size_t)(B * H * s * (D + 4)) * sizeof(float);
}

extern "C" int flare_attn_step(const void* q, const void* k, const void* v, const int64_t* strides, int dtype,
                               int64_t B, int64_t M, int64_t H, int64_t G, int64_t D, float scale, float softcap,
                               const float* slopes, const int32_t* lengths, void* k_cache, void* v_cache, void* y,
                               void* workspace, size_t workspace_bytes, void* stream) {
    const int64_t N = 1;
    FLARE_REQUIRE(q && k && v && strides && lengths && k_cache && v_cache && y, "flare_attn_step: null pointer");
    ATTN_REQUIRE_SIZES("flare_attn_step");
    const int64_t none[9] = {};
    AttnArgs p = attn_args(q, k_cache, v_cache, none, B, N, M, H, G, D, scale, softcap, slopes);
    p.q.sb = strides[0], p.q.sh = strides[1];
    p.k_new = k, p.kn_sb = strides[2], p.kn_sg = strides[3];
    p.v_new = v, p.vn_sb = strides[4], p.vn_sg = strides[5];
    const Rows kr = {k, strides[2], 0, strides[3]}, vr = {v, strides[4], 0, strides[5]};
    FLARE_REQUIRE(aligned(p.q, dtype) && aligned(kr, dtype) && aligned(vr, dtype) && aligned(p.k, dtype) &&
                  aligned(p.v, dtype) && ((uintptr_t)y & 15) == 0,
                  "flare_attn_step: rows must be 16-byte aligned and less than 2^22 elements apart");
    p.splits = step_splits(B, M, H, G);
    if (workspace_bytes < flare_attn_step_workspace_size(B, M, H, G, D) ||
        (p.splits > 1 && (!workspace || ((uintptr_t)workspace & 15)))) {
        set_error("flare_attn_step: workspace of %zu bytes is too small or not 16-byte aligned", workspace_bytes);
        return FLARE_ERR_WORKSPACE;
    }
    p.lengths = lengths, p.y = y, p.parts = (float*)workspace;
    return attn_step(p, dtype, (hipStream_t)stream);
}

extern "C" size_t flare_qattn_workspace_size(int64_t B, int64_t N, int64_t M, int64_t H, int64_t G, int64_t D, int dtype,
                                             int bits) {
    if (B < 1 || N < 1 || M < 1 || H < 1 || G < 1 || D < 1 || H % G) return 0;
    const int path = qattn_path(N, M, H, G, D, dtype);
    if (path == kRows) {
        const int64_t s = rows_splits(B, N, M, H, G, D, dtype, bits);
        return s == 1 ? 0 : (size_t)(B * N * H * s * (D + 4)) * sizeof(float);
    }
    AttnArgs p = {};
    p.B = path == kFused ? B : expand_slice(B, M, G, D), p.N = N, p.M = M, p.H = H, p.D = D, p.causal = 1;
    size_t most = 0;
    // (the last slice may be smaller and split its keys more often)
    for (const int64_t left = path == kFused ? B : B % p.B ? B % p.B : p.B;; p.B = left) {
        if (path == kFused) split_forward(p, dtype);
        else split_expanded(p, dtype, true);
        most = rows_bytes(p) > most ? rows_bytes(p) : most;
        if (p.B == left) break;
    }
    return most + (path == kFused ? 0 : expanded_bytes(expand_slice(B, M, G, D), M, G, D));
}

extern "C" int flare_qattn(const void* q, const void* k, const void* v, const int64_t* strides, int dtype, int bits, int64_t B,
                           int64_t N, int64_t M, int64_t H, int64_t G, int64_t D, float scale, float softcap,
                           const float* slopes, const int32_t* prefix_lengths, const int32_t* lengths,
                           const int32_t* new_lengths, void* k_cache, void* k_scale, void* v_cache, void* v_scale, void* y,
                           void* workspace, size_t workspace_bytes, void* stream) {
    FLARE_REQUIRE(q && k && v && strides && lengths && k_cache && k_scale && v_cache && v_scale && y,
                  "flare_qattn: null pointer");
    ATTN_REQUIRE_SIZES("flare_qattn");
    FLARE_REQUIRE(bits == 4 || bits == 8, "flare_qattn: %d bits; 4 or 8", bits);
    FLARE_REQUIRE(N * H <= (1 << 30) && N * G <= (1 << 27) &&
                  qattn_blocks(B, N, M, H, G, D, dtype, bits) <= mix::kMostBlocks, "flare_qattn: too large");
    AttnArgs p = attn_args(q, k_cache, v_cache, strides, B, N, M, H, G, D, scale, softcap, slopes);
    const Rows kr = {k, strides[3], strides[4], strides[5]}, vr = {v, strides[6], strides[7], strides[8]};
    const uintptr_t held = (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)y;
    FLARE_REQUIRE(aligned(p.q, dtype) && aligned(kr, dtype) && aligned(vr, dtype) && (held & 15) == 0,
                  "flare_qattn: rows must be 16-byte aligned and less than 2^22 elements apart");
    if (workspace_bytes < flare_qattn_workspace_size(B, N, M, H, G, D, dtype, bits) ||
        (workspace_bytes && (!workspace || ((uintptr_t)workspace & 15)))) {
        set_error("flare_qattn: workspace of %zu bytes is too small or not 16-byte aligned", workspace_bytes);
        return FLARE_ERR_WORKSPACE;
    }
    p.k_scale = (uint8_t*)k_scale, p.v_scale = (uint8_t*)v_scale;
    p.lengths = lengths, p.fresh = new_lengths, p.prefix = prefix_lengths, p.causal = 1;
    p.y = y, p.parts = (float*)workspace;
    const int path = qattn_path(N, M, H, G, D, dtype);
    // a few tokens' keys and values are quantised on the way
    if (N <= 16 && path == kRows) {
        p.k_new = k, p.kn_sb = strides[3], p.kn_sn = strides[4], p.kn_sg = strides[5];
        p.v_new = v, p.vn_sb = strides[6], p.vn_sn = strides[7], p.vn_sg = strides[8];
    } else {
        const int rc = flare_qcache_write(k, v, strides + 3, dtype, bits, B, N, M, G, D, lengths, new_lengths, k_cache,
                                          k_scale, v_cache, v_scale, stream);
        if (rc != FLARE_OK) return rc;
    }
    if (path == kRows) {
        p.splits = rows_splits(B, N, M, H, G, D, dtype, bits), p.row_splits = rows_heads(B, M, G, row_tiles(N, H, G, dtype));
        return FLARE_BY_DTYPE(dtype, qattn_rows, (p, bits, row_tiles(N, H, G, dtype), (hipStream_t)stream));
    }
    if (path == kExpanded) return qattn_expanded(p, dtype, bits, workspace, (hipStream_t)stream);
    split_forward(p, dtype);
    return dtype == FLARE_BF16 ? qattn_forward<__hip_bfloat16>(p, bits, (hipStream_t)stream)
                               : qattn_forward<__half>(p, bits, (hipStream_t)stream);
}
