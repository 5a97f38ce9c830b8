// Attention of one new token per sequence over a paged F16 key-value cache.
//
// For query head h of sequence s, with key-value head h / group,
//   y = sum_t w_t v_t / sum_t w_t,   w_t = exp(scale * q . k_t - m),
// m the running maximum: one pass over keys and values, sums and statistics in
// F32, exponents in base 2 (log2(e) goes into q).
//
// A workgroup takes one key-value head of one sequence (all of its query heads,
// so that the cache is read once) over one chunk of its tokens; its four (one, eight) waves
// take steps of 32 tokens in turn. Both products run on
// v_mfma_f32_16x16x32_f16 with the cache's rows as one operand:
//   scores  [16 tokens x 16 columns] += K rows (as stored)  x  q columns
//   outputs [16 values x 16 columns] += V transposed        x  weight columns
// The score tiles leave lane (column c, group G) with tokens 4G..4G+3 of both
// tiles of a step; V rows are loaded in that token order, so the weights go into the
// second product where they are. A lane loads 8 consecutive values of 8 tokens
// (16 lanes read whole rows) and picks value j of each by v_perm_b32: 32 per
// step at width 128, against 1024 multiply-adds per lane and query head.
//
// Columns. The tile's 16 columns are 8 query heads twice: a factor x is split
// into fp16 parts x = hi + lo (hi 11 bits, lo the next 11), hi in column c and lo in
// column c + 8 of one tile; the two columns' sums are added at the end. So F32
// queries and weights cost no instruction more than F16 ones with 8 query heads
// or fewer, and errors stay at 2^-22 (against 64 bits 1.0e-7 relative over 4096 tokens, where
// products in F32 one by one leave 2.0e-7). q is scaled by a power of two
// (max |scale q| in [2^9, 2^11)) and the weights by 2^14, so that what the low
// parts lose below 2^-24 stays far below that. Where a factor is not 0 its high part is not either, so that infinite
// keys and values meet it as they would an F32 number.
//
// What bounds it: reading the cache (4 * width bytes per token and head). A step's K rows
// are reloaded behind its scores and its V rows behind its second product, so a wave has 8
// to 16 KiB on their way at any time, three workgroups to a CU; one sequence of 32768 tokens x 8 heads takes
// 24.6 us (5.5 TB/s) and 4.6 for the join. Long ragged rows go to attend_even, below: 32 sequences of up to
// 4096 tokens x 32 heads of 128 (1.2 GB) 183 us, 6.6 TB/s, what a kernel that only reads reaches. Below some
// ten MB it is the chain of latencies (length and pages, rows, two products, the waves' sums): 33 tokens x 32 heads
// 5.9 us of kernel.
//
// Sequences of more than one chunk leave (sum w v, m, sum w) per chunk in the
// workspace; a second launch joins them in order, so results do not
// depend on the order in which chunks end. (Joined by the workgroup that ends last instead, the sums have to
// go past the XCDs' own L2s: 1 x 32768 tokens 49 us against 29, and 100 with fences that write the L2s back.)
#include "device_common.h"
#include "launch.h"
#include "paged.h"

#include <algorithm>

namespace {

using kk::half8;
using kk::kWave;
using kk::PoolView;

typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4, kWideWaves = 8;
constexpr int kThreads = kWaves * kWave;
constexpr int kStep = 32;                // tokens of a wave's step
constexpr int kMinChunk = kWaves * kStep;
constexpr int kMaxChunk = 512, kMaxChunkMany = 1024;
constexpr int kMostChunks = 65535;       // the grid's limit
constexpr int64_t kMostIds = 8000;       // page ids of a chunk in LDS, 32 KB
constexpr int kRowSteps = 1;             // what beginning a row counts in a share
constexpr int kMostEven = 1024;          // sequences whose lengths a workgroup of attend_even goes through
constexpr float kWeightScale = 16384.0f; // of the weights' F16 parts
constexpr float kLeastPart = 0x1p-24f;    // the least F16 above 0
constexpr float kLeastWeight = 0x1p100f;  // p times this is above kLeastPart for every normal p

struct AttendArgs {
    const _Float16 *k, *v;
    const int *table, *lengths;
    const void *q;
    void *y;
    float *part_o, *part_ml;             // [sequence][query head][chunk]: width sums; m and sum w
    int *status;
    PoolView pool;
    int64_t q_stride, y_stride;
    int query_heads, group, tiles, longest, window, row_pages, chunk, chunks, f16, q_wide;
    float scale_log2;
    // attend_even: (sequence, four heads) -> where the row's sums stand in the workspace, and of how many workgroups
    int2 *spans;
    kk::FastDiv shares;                  // attend_even's workgroups
    int sequences;
};

// A word that no lane writes during the launch, read through the scalar cache.
__device__ __forceinline__ int scalar_load(const int *p) {
    return *(const __attribute__((address_space(4))) int *)(p);
}

__device__ __forceinline__ int length_of(const AttendArgs &a, int s, bool tell) {
    int len = scalar_load(a.lengths + s);
    if (len < 0 || len > a.longest) {
        if (tell) kk::report(a.status, kk::kBadIndex);
        len = len < 0 ? 0 : a.longest;
    }
    return len;
}

__device__ __forceinline__ void store_output(const AttendArgs &a, int64_t at, float v) {
    if (a.f16) static_cast<_Float16 *>(a.y)[at] = static_cast<_Float16>(v);   // the one rounding of an F16 output
    else static_cast<float *>(a.y)[at] = v;
}

// Lane moves across the four groups of 16 lanes (each pairs with both others' sums).
__device__ __forceinline__ float across_groups_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float across_groups_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// The value of the lane eight columns on (row_ror:8): a column's other part.
__device__ __forceinline__ float other_part(float v) { return kk::dpp_move<0x128>(v); }
// Both parts' sum, in the high part's lanes; where that is infinite (infinite values), the low part has NaN or the other sign.
__device__ __forceinline__ float both_parts(float high) {
    const float low = other_part(high);
    return fabsf(high) == INFINITY ? high : high + low;
}

// Eight values of a row of q (16-byte loads where a.q_wide allows).
__device__ __forceinline__ void load_query(const AttendArgs &a, int64_t at, float (&v)[8]) {
    if (a.f16) {
        const _Float16 *q = static_cast<const _Float16 *>(a.q) + at;
        if (a.q_wide) {
            const half8 x = *reinterpret_cast<const half8 *>(q);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(x[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(q[i]);
        }
    } else {
        const float *q = static_cast<const float *>(a.q) + at;
        if (a.q_wide) {
            const float4v x = *reinterpret_cast<const float4v *>(q), y = *reinterpret_cast<const float4v *>(q + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = x[i], v[i + 4] = y[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = q[i];
        }
    }
}

// A lane's part of a cache row; ONCE: with the non-temporal hint.
template <typename T, bool ONCE>
__device__ __forceinline__ T load_row(const _Float16 *p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const T *>(p));
    else return *reinterpret_cast<const T *>(p);
}

// The exponent of a float's size: 128 for what is not finite, -127 for 0 and subnormal ones.
__device__ __forceinline__ int exponent_of(float v) { return static_cast<int>((__float_as_uint(v) >> 23) & 0xff) - 127; }

// q columns: column c is head c % 8 of each tile, its high (c < 8) or low part; the scores times `undo` are in base 2.
template <int D32, int NT, bool FULL>
__device__ __forceinline__ void split_queries(float scale_log2, int heads, int width, int c, int G, const float (&q)[NT][D32][8],
                                              half8 (&qf)[NT][D32], float (&undo)[NT]) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const bool column = nt * 8 + (c & 7) < heads;
        float top = 0.0f;
#pragma unroll
        for (int d = 0; d < D32; ++d)
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, FULL || d * 32 + G * 8 < width ? fabsf(q[nt][d][i]) : 0.0f);
        const int size = exponent_of(across_groups_max(top));
        // 2^e with top * |scale| * 2^e in [2^9, 2^11); beside an infinite value every finite one stays finite
        const int e = max(-126, min(126, min(9 - size, 110) - exponent_of(scale_log2)));
        undo[nt] = ldexpf(1.0f, -e);
        const float factor = column ? ldexpf(scale_log2, e) : 0.0f;
#pragma unroll
        for (int d = 0; d < D32; ++d) {
            const float by = FULL || d * 32 + G * 8 < width ? factor : 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = q[nt][d][i] * by;
                // a value other than 0 keeps a high part other than 0 for infinite keys, as the weights do
                const _Float16 high = static_cast<_Float16>(__builtin_amdgcn_fmed3f(x, x * 0x1p127f, copysignf(kLeastPart, x)));
                qf[nt][d][i] = c < 8 ? high : static_cast<_Float16>(x - static_cast<float>(high));
            }
        }
    }
}

// A step's scores to weights, high and low parts as the second product's columns; the maxima and sums so far move
// along. there(i): whether the lane's token i counts, asked where `masked`.
template <int VW, int NT, typename There>
__device__ __forceinline__ void weigh(const float4v (&scores)[NT][2], const float (&undo)[NT], bool masked, There there, int c,
                                      float (&m)[NT], float (&l)[NT], float4v (&acc)[NT][VW], half8 (&pf)[NT]) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float sc[8], sum = 0.0f, top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float part = scores[nt][i / 4][i % 4];
            sc[i] = (part + other_part(part)) * undo[nt];
            sum += sc[i];
        }
        if (__any(!(fabsf(sum) < INFINITY))) {
            // infinite keys or queries: the high part's infinity, as F32 products have it
            // (its low part gives NaN or the other sign)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float part = scores[nt][i / 4][i % 4], other = other_part(part);
                const float high = c < 8 ? part : other;
                if (fabsf(high) == INFINITY) sc[i] = high;
            }
        }
        if (masked) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sc[i] = there(i) ? sc[i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, sc[i]);
        top = fmaxf(m[nt], across_groups_max(top));
        if (__any(top > m[nt])) {
            const float alpha = top > m[nt] ? __builtin_amdgcn_exp2f(m[nt] - top) : 1.0f;   // 0 from no token yet
            l[nt] *= alpha;
#pragma unroll
            for (int j = 0; j < VW; ++j) acc[nt][j] *= alpha;
            m[nt] = top;
        }
        // scaled after the exponential: an exponent of 14 and a difference holds 2^-20 of it, 3e-7 of the weight
        const float from = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float p = __builtin_amdgcn_exp2f(sc[i] - from) * kWeightScale;
            l[nt] += p;
            // A weight above 0 keeps a high part above 0, which takes an infinite value to its infinity (the low part
            // takes it off again: finite values lose nothing)
            const float part = __builtin_amdgcn_fmed3f(p, p * kLeastWeight, kLeastPart);
            const _Float16 high = static_cast<_Float16>(part);
            pf[nt][i] = c < 8 ? high : static_cast<_Float16>(p - static_cast<float>(high));
        }
    }
}

// The second product: value j of a lane's eight tokens, picked out of their rows, times the weights.
template <int VW, int NT>
__device__ __forceinline__ void add_values(const uint32_t (&vr)[8][VW / 2], const half8 (&pf)[NT], float4v (&acc)[NT][VW]) {
#pragma unroll
    for (int j = 0; j < VW; ++j) {
        union { uint32_t u[4]; half8 h; } vf;
        const int word = (j / 8) * 4 + (j % 8) / 2;
        const uint32_t pick = j & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int u = 0; u < 4; ++u) vf.u[u] = __builtin_amdgcn_perm(vr[2 * u + 1][word], vr[2 * u][word], pick);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            acc[nt][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf.h, pf[nt], acc[nt][j], 0, 0, 0);
    }
}

// D32: 32-value pieces of a head (width <= 32 * D32; FULL: equal). VW: values a lane loads of a V
// row (16 lanes: width <= 16 * VW). NT: column tiles (8 query heads each). UNI: page_tokens % 16
// == 0, so that a half step of 16 tokens lies in one page: its address is scalar, its page id a
// scalar load. Otherwise the chunk's page ids wait in LDS and each lane finds its rows there.
template <int D32, int VW, int NT, bool UNI, bool FULL, bool ONCE, int WAVES>
__global__ __launch_bounds__(WAVES * kWave) void attend(AttendArgs a) {
    static_assert(VW == 4 || VW == 8 || VW == 16, "4, 8 or 2 x 8 values of a V row per lane");
    constexpr int VP = VW < 8 ? VW : 8;              // values of one load
    constexpr int VR = VW / 2;                       // dwords of a lane's part of a V row
    constexpr int DPad = 16 * VW;
    constexpr int kGroup = WAVES * kWave;
    extern __shared__ float lds[];
    const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int c = lane & 15, G = lane >> 4;
    int s = blockIdx.y, chunk = blockIdx.z, kvh = blockIdx.x, tile = 0;
    if (a.tiles > 1) {
        // Workgroups go round the eight XCDs: numbered so that the tiles of one chunk, which read the same rows, are a
        // multiple of eight apart, on one XCD and its L2, and start together (last: fewer than eight chunks)
        const uint32_t number = blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z);
        const uint32_t items = gridDim.x / a.tiles * gridDim.y * gridDim.z, even = items & ~7u;
        const bool whole = number < even * a.tiles;
        const uint32_t side = whole ? 8 : items - even, at = whole ? number : number - even * a.tiles;
        const uint32_t set = at / (side * a.tiles), in_set = at - set * side * a.tiles;
        tile = in_set / side;
        const uint32_t item = (whole ? set * 8 : even) + in_set - tile * side, heads_of_cache = gridDim.x / a.tiles;
        const uint32_t row_chunk = item / heads_of_cache;
        kvh = item - row_chunk * heads_of_cache;
        chunk = row_chunk / gridDim.y;
        s = row_chunk - chunk * gridDim.y;
    }
    // Workgroups also go round the CUs, wherever one has room: parts that are there first (part number slowest: those
    // past a sequence's end come last and at once), and sequences turned within each eight, so that long and
    // short ones that take turns do not meet on the same CUs (64 sequences of 1000 tokens x 6 heads where
    // `longest` is 32768: 41 us, in order of sequences and their parts 54; 96 x 8 heads of 80, every other one of 2048 tokens,
    // the rest of half as many at most: 70, in that order 72, not turned 83)
    const int eight = s / 8, first_of = eight * 8, size = min(8, static_cast<int>(gridDim.y) - first_of);
    s = first_of + (s - first_of + eight + eight / 4 + chunk) % size;
    const int head0 = kvh * a.group + tile * 8 * NT;                        // first query head
    const int heads = min(8 * NT, a.group - tile * 8 * NT);
    const int width = FULL ? 32 * D32 : a.pool.width;

    // a part past the sequence's end, before it asks for anything
    if (chunk > 0 && a.window == 0 && chunk * a.chunk >= scalar_load(a.lengths + s)) return;
    // the queries' values are on their way while the sequence's length and pages are read
    float q[NT][D32][8];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int h = nt * 8 + (c & 7);
        const int64_t q_row = s * a.q_stride + (int64_t)(head0 + (h < heads ? h : 0)) * width;
#pragma unroll
        for (int d = 0; d < D32; ++d) load_query(a, q_row + (FULL || d * 32 + G * 8 < width ? d * 32 + G * 8 : 0), q[nt][d]);
    }

    const int len = length_of(a, s, tid == 0 && chunk == 0 && kvh == 0 && tile == 0);
    const int first = a.window > 0 ? max(0, len - a.window) : 0;
    const int base = first & ~(kStep - 1);
    const int begin = base + chunk * a.chunk;
    const int end = min(len, begin + a.chunk);
    const bool single = len - base <= a.chunk;
    if (begin >= end) {
        if (chunk == 0)                              // no tokens: zeros
            for (int i = tid; i < heads * width; i += kGroup)
                store_output(a, s * a.y_stride + (int64_t)(head0 + i / width) * width + i % width, 0.0f);
        return;
    }
    const int lo = max(first, begin), hi = end - 1;  // first and last token of the chunk
    const int *row = a.table + (int64_t)s * a.row_pages;

    // !UNI: page ids of the chunk; a bad one is reported and its tokens left out
    int *page_ids = reinterpret_cast<int *>(lds);
    const int page0 = a.pool.per_page.div(lo);
    bool holes = false;
    if constexpr (!UNI) {
        const int last_page = a.pool.per_page.div(hi);
        bool bad = false;
        for (int i = tid; i <= last_page - page0; i += kGroup) {
            int id = row[page0 + i];
            if (static_cast<unsigned>(id) >= static_cast<unsigned>(a.pool.pages)) {
                bad = true;
                id = -1;
            }
            page_ids[i] = id;
        }
        if (bad) kk::report(a.status, kk::kBadPage);
        holes = __syncthreads_or(bad);
    }

    const _Float16 *k_head = a.k + (int64_t)kvh * a.pool.head_stride;
    const _Float16 *v_head = a.v + (int64_t)kvh * a.pool.head_stride;

    // the registers of a step: its K rows as A operands, its V rows as loaded
    half8 kf[2][D32];
    uint32_t vr[8][VR];
    // UNI: where the step's two halves stand, and whether their pages exist
    struct Halves {
        int64_t at[2];
        bool ok[2];
    };
    auto find = [&](int t0) {
        Halves w;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int t = min(max(t0 + half * 16, lo & ~15), hi & ~15);
            const int p = a.pool.per_page.div(t);
            int id = scalar_load(row + p);
            w.ok[half] = static_cast<unsigned>(id) < static_cast<unsigned>(a.pool.pages);
            if (!w.ok[half]) {
                if (lane == 0) kk::report(a.status, kk::kBadPage);
                id = 0;
            }
            w.at[half] = (int64_t)id * a.pool.page_stride + (int64_t)(t - p * a.pool.page_tokens) * a.pool.token_stride;
        }
        return w;
    };
    // !UNI: the row of token t, moved into the chunk
    auto row_of = [&](int t) -> int64_t {
        t = min(max(t, lo), hi);
        const int p = a.pool.per_page.div(t);
        return (int64_t)max(page_ids[p - page0], 0) * a.pool.page_stride +
               (int64_t)(t - p * a.pool.page_tokens) * a.pool.token_stride;
    };
    // a lane's token of V register i, which is also the token of its score i
    auto token_of = [&](int t0, int i) { return t0 + (i < 4 ? 0 : 16) + G * 4 + (i & 3); };
    const uint32_t k_lane = static_cast<uint32_t>(c * a.pool.token_stride) + G * 8;
    const uint32_t v_lane = static_cast<uint32_t>(G * 4 * a.pool.token_stride);
    auto load_k = [&](int t0, const Halves &w) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            int64_t at = 0;
            if constexpr (!UNI) at = row_of(t0 + half * 16 + c);
#pragma unroll
            for (int d = 0; d < D32; ++d) {
                const bool in = FULL || d * 32 + G * 8 < width;
                const _Float16 *p = UNI ? k_head + w.at[half] + (k_lane + (in ? d * 32 : 0)) - (in ? 0 : G * 8)
                                        : k_head + at + (in ? d * 32 + G * 8 : 0);
                const half8 x = load_row<half8, ONCE>(p);
                kf[half][d] = in ? x : half8{0, 0, 0, 0, 0, 0, 0, 0};
            }
        }
    };
    auto load_v = [&](int t0, const Halves &w) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            int64_t at = 0;
            if constexpr (!UNI) at = row_of(token_of(t0, i));
#pragma unroll
            for (int part = 0; part < VW / VP; ++part) {
                // a column past the width gives values past it, which are not stored: any part of the row will do (zeros
                // in its place make the wave wait for the row here: 64 x 1024 tokens x 8 heads of 80 34.6 us, with them 2 more)
                const int col = part * 128 + c * VP;
                const bool in = (FULL && 16 * VW == 32 * D32) || col < width;
                const _Float16 *p = UNI ? v_head + w.at[i / 4] + (i & 3) * a.pool.token_stride + (v_lane + (in ? col : 0))
                                        : v_head + at + (in ? col : 0);
                if constexpr (VW == 4) {
                    const uint2v x = load_row<uint2v, ONCE>(p);
                    vr[i][0] = x[0], vr[i][1] = x[1];
                } else {
                    const uint4v x = load_row<uint4v, ONCE>(p);
#pragma unroll
                    for (int u = 0; u < 4; ++u) vr[i][part * 4 + u] = x[u];
                }
            }
        }
    };

    int t0 = begin + wave * kStep;
    const bool any = t0 < end;
    Halves here{}, next{};
    if (any) {
        if constexpr (UNI) here = find(t0);
        load_k(t0, here);
        load_v(t0, here);
    }
    __builtin_amdgcn_sched_barrier(0);

    half8 qf[NT][D32];
    float undo[NT];
    split_queries<D32, NT, FULL>(a.scale_log2, heads, width, c, G, q, qf, undo);

    float4v acc[NT][VW];
    float m[NT], l[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt] = -INFINITY;
        l[nt] = 0.0f;
#pragma unroll
        for (int j = 0; j < VW; ++j) acc[nt][j] = float4v{0, 0, 0, 0};
    }

    if (any) for (;;) {
        const int t1 = t0 + WAVES * kStep;
        const bool more = t1 < end;
        if constexpr (UNI) if (more) next = find(t1);
        // a step with tokens that are not the chunk's, or whose page is missing
        const bool masked = t0 < lo || t0 + kStep > end || (UNI ? !(here.ok[0] && here.ok[1]) : holes);
        auto there = [&](int i) {
            const int t = token_of(t0, i);
            bool ok = t >= lo && t <= hi;
            if constexpr (UNI) ok = ok && here.ok[i / 4];
            else ok = ok && page_ids[a.pool.per_page.div(min(max(t, lo), hi)) - page0] >= 0;
            return ok;
        };

        float4v scores[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            scores[nt][0] = scores[nt][1] = float4v{0, 0, 0, 0};
#pragma unroll
            for (int d = 0; d < D32; ++d) {
                scores[nt][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[0][d], qf[nt][d], scores[nt][0], 0, 0, 0);
                scores[nt][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[1][d], qf[nt][d], scores[nt][1], 0, 0, 0);
            }
        }
        // the next step's K rows are on their way during the weights and the second product, its V rows
        // during the next scores
        __builtin_amdgcn_sched_barrier(0);
        if (more) load_k(t1, next);
        __builtin_amdgcn_sched_barrier(0);

        half8 pf[NT];
        weigh<VW, NT>(scores, undo, masked, there, c, m, l, acc, pf);
        if (masked) {                                // 0 * NaN would reach the sums
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool ok = there(i);
#pragma unroll
                for (int u = 0; u < VR; ++u) vr[i][u] = ok ? vr[i][u] : 0;
            }
        }
        add_values<VW, NT>(vr, pf, acc);
        if (!more) break;
        __builtin_amdgcn_sched_barrier(0);
        load_v(t1, next);
        __builtin_amdgcn_sched_barrier(0);
        t0 = t1;
        here = next;
    }
    if constexpr (!UNI) __syncthreads();             // page_ids are read; the sums go over them

    // the waves' sums side by side, then one sum per value
    float *wave_ml = lds, *wave_o = lds + WAVES * NT * 8 * 2;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const float total = across_groups_sum(l[nt]);
        const int h = nt * 8 + c;
        const bool mine = c < 8 && h < heads;
        if (mine && G == 0) {
            wave_ml[(wave * NT * 8 + h) * 2] = m[nt];
            wave_ml[(wave * NT * 8 + h) * 2 + 1] = total;
        }
        // row 4G + r of product j is value VP * (4G + r) + j % 8 of half j / 8
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < VW; j += 4) {
                float4v v;
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = both_parts(acc[nt][j + u][r]);
                if (mine)
                    *reinterpret_cast<float4v *>(wave_o + (wave * heads + h) * DPad + (j / 8) * 128 + (4 * G + r) * VP +
                                                 j % 8) = v;
            }
    }
    __syncthreads();
    for (int i = tid; i < heads * width; i += kGroup) {
        const int h = i / width, d = i - h * width;
        float top = -INFINITY, total = 0.0f, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = fmaxf(top, wave_ml[(w * NT * 8 + h) * 2]);
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float mw = wave_ml[(w * NT * 8 + h) * 2];
            const float scale = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - top);
            total += scale * wave_ml[(w * NT * 8 + h) * 2 + 1];
            sum += scale * wave_o[(w * heads + h) * DPad + d];
        }
        if (single) {
            store_output(a, s * a.y_stride + (int64_t)(head0 + h) * width + d, total == 0.0f ? 0.0f : sum / total);
        } else {
            const int64_t at = ((int64_t)s * a.query_heads + head0 + h) * a.chunks + chunk;
            a.part_o[at * width + d] = sum;
            if (d == 0) {
                a.part_ml[at * 2] = top;
                a.part_ml[at * 2 + 1] = total;
            }
        }
    }
}

// The steps of a row: from the one that holds its first token on.
__device__ __forceinline__ int base_of(const AttendArgs &a, int len) {
    return (a.window > 0 ? max(0, len - a.window) : 0) & ~(kStep - 1);
}
__device__ __forceinline__ int steps_of(const AttendArgs &a, int len) { return (len - base_of(a, len) + kStep - 1) / kStep; }

// Sum over the lanes up to this one: within 16 lanes by row shifts, then the rows' last lanes on.
template <int CONTROL, int ROWS>
__device__ __forceinline__ int add_shifted(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CONTROL, ROWS, 0xf, false);
}
__device__ __forceinline__ int sum_to_lane(int v) {
    v = add_shifted<0x111, 0xf>(v);
    v = add_shifted<0x112, 0xf>(v);
    v = add_shifted<0x114, 0xf>(v);
    v = add_shifted<0x118, 0xf>(v);
    v = add_shifted<0x142, 0xa>(v);
    return add_shifted<0x143, 0xc>(v);
}

// The part of one workgroup of attend_even: of all steps in the order (sequence, four heads, step), `left` from `at` on.
// A row's first kRowSteps steps are empty: what it costs to begin it.
struct Share {
    int at, left;
    int s, four, step;                               // where `at` is
    int per, extra;                                  // steps of a share; the first `extra` shares have one more
    __device__ __forceinline__ int holder(int step_number) const {
        const int cut = extra * (per + 1);
        return step_number < cut ? step_number / (per + 1) : extra + (step_number - cut) / per;
    }
};

__device__ __forceinline__ Share share_of(const AttendArgs &a, int number, int fours, int lane, bool tell) {
    auto steps = [&](int s) {
        if (s >= a.sequences) return 0;
        int len = a.lengths[s];
        if (len < 0 || len > a.longest) {
            if (tell) kk::report(a.status, kk::kBadIndex);
            len = len < 0 ? 0 : a.longest;
        }
        const int n = steps_of(a, len);
        return n ? (n + kRowSteps) * fours : 0;
    };
    const int mine = steps(lane), mine_to_lane = sum_to_lane(mine);        // of the first 64 sequences; more are read twice
    int total = __builtin_amdgcn_readlane(mine_to_lane, kWave - 1);
    if (a.sequences > kWave) {
        int more = 0;
#pragma unroll 4
        for (int s = lane + kWave; s < a.sequences; s += kWave) more += steps(s);
        total += __builtin_amdgcn_readlane(sum_to_lane(more), kWave - 1);
    }
    Share r;
    r.per = max(static_cast<int>(a.shares.div(total)), 1);
    r.extra = max(0, total - r.per * static_cast<int>(a.shares.d));
    r.at = number * r.per + min(number, r.extra);
    r.left = max(0, min(r.per + (number < r.extra ? 1 : 0), total - r.at));
    if (r.left == 0) return r;
    int before = 0;
    for (int s0 = 0;; s0 += kWave) {                 // ends: at < total
        const int own = s0 == 0 ? mine : steps(s0 + lane), sum = s0 == 0 ? mine_to_lane : sum_to_lane(own);
        if (const uint64_t past = __ballot(before + sum > r.at)) {
            const int found = __builtin_ctzll(past);
            const int held = __builtin_amdgcn_readlane(own, found);
            const int in_row = r.at - before - __builtin_amdgcn_readlane(sum, found) + held, per_four = held / fours;
            r.s = s0 + found;
            r.four = in_row / per_four;
            r.step = in_row - r.four * per_four;
            return r;
        }
        before += __builtin_amdgcn_readlane(sum, kWave - 1);
    }
}

// The same sums by one workgroup to a CU (width 64: two), each an equal share of the steps of all rows. Its waves take four
// neighbouring key-value heads, so that what it reads lies together in either order within a page (64 x 4096 tokens x 8
// heads, token by token: 195 us by `attend`, 5.5 TB/s; 168 so, 6.4), and a wave's sums are its head's: no barrier, no LDS.
// Four waves with a step on its way each keep up with the memory (two workgroups to a CU: 172 for 165 with 64 x 4096 head by
// head; width 64: 91 for 95). A new row costs a chain of latencies - length, page, rows - of some 4 us: the next row is
// looked up while this one's first rows are on their way, its first rows are asked for behind this one's last scores, and
// beginning it counts as a step of a share (64 sequences ragged to 2048 x 8 heads: 63 us without all that, 58 with).
template <int D32, int VW>
__global__ __launch_bounds__(kThreads, 1) void attend_even(AttendArgs a) {
    constexpr int VP = VW < 8 ? VW : 8, VR = VW / 2, width = 32 * D32;
    const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int c = lane & 15, G = lane >> 4;
    const int fours = a.pool.heads / kWaves, heads = a.group;
    const Share share = share_of(a, blockIdx.x, fours, lane, blockIdx.x == 0 && wave == 0);
    if (share.left == 0 || share.step + share.left <= kRowSteps) return;     // (or ends among a row's empty steps)

    // what a share has of one row
    struct Run {
        int s, four, step, steps, take;              // the row's steps, and this run's from `step` on, empty ones included
        int lo, hi, t0;                              // its tokens, and the first of its first step
        const int *row;
        const _Float16 *k, *v;
    };
    auto run_at = [&](int s, int four, int step, int left) {
        Run r;
        const int len = length_of(a, s, false), base = base_of(a, len), kvh = four * kWaves + wave;
        r.s = s;
        r.four = four;
        r.step = step;
        r.steps = (len - base + kStep - 1) / kStep + kRowSteps;
        r.take = min(left, r.steps - step);
        r.t0 = base + max(0, step - kRowSteps) * kStep;
        r.lo = max(r.t0, a.window > 0 ? len - a.window : 0);
        r.hi = min(len, base + (step + r.take - kRowSteps) * kStep) - 1;
        r.row = a.table + (int64_t)s * a.row_pages;
        r.k = a.k + (int64_t)kvh * a.pool.head_stride;
        r.v = a.v + (int64_t)kvh * a.pool.head_stride;
        return r;
    };
    auto run_after = [&](const Run &r, int left) {   // left > 0: there is a row with tokens
        int s = r.s, four = r.four + 1;
        if (four == fours) {
            four = 0;
            do ++s;
            while (length_of(a, s, false) == 0);
        }
        return run_at(s, four, 0, left);
    };

    half8 kf[2][D32];
    uint32_t vr[8][VR];
    struct Halves {
        int64_t at[2];
        bool ok[2];
    };
    auto find = [&](const Run &r, int t0) {
        Halves w;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int t = min(max(t0 + half * 16, r.lo & ~15), r.hi & ~15);
            const int p = a.pool.per_page.div(t);
            int id = scalar_load(r.row + p);
            w.ok[half] = static_cast<unsigned>(id) < static_cast<unsigned>(a.pool.pages);
            if (!w.ok[half]) {
                if (lane == 0) kk::report(a.status, kk::kBadPage);
                id = 0;
            }
            w.at[half] = (int64_t)id * a.pool.page_stride + (int64_t)(t - p * a.pool.page_tokens) * a.pool.token_stride;
        }
        return w;
    };
    const uint32_t k_lane = static_cast<uint32_t>(c * a.pool.token_stride) + G * 8;
    const uint32_t v_lane = static_cast<uint32_t>(G * 4 * a.pool.token_stride);
    auto load_k = [&](const _Float16 *k, const Halves &w) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int d = 0; d < D32; ++d) kf[half][d] = load_row<half8, true>(k + w.at[half] + (k_lane + d * 32));
    };
    auto load_v = [&](const _Float16 *v, const Halves &w) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int part = 0; part < VW / VP; ++part) {
                const int col = part * 128 + c * VP;
                const bool in = 16 * VW == width || col < width;
                const _Float16 *p = v + w.at[i / 4] + (i & 3) * a.pool.token_stride + (v_lane + (in ? col : 0));
                if constexpr (VW == 4) {
                    const uint2v x = load_row<uint2v, true>(p);
                    vr[i][0] = x[0], vr[i][1] = x[1];
                } else {
                    const uint4v x = load_row<uint4v, true>(p);
#pragma unroll
                    for (int u = 0; u < 4; ++u) vr[i][part * 4 + u] = x[u];
                }
            }
    };
    float q[1][D32][8];
    auto load_queries = [&](const Run &r) {
        const int64_t at = r.s * a.q_stride + (int64_t)((r.four * kWaves + wave) * a.group + (c & 7) % heads) * width;
#pragma unroll
        for (int d = 0; d < D32; ++d) load_query(a, at + d * 32 + G * 8, q[0][d]);
    };

    Run now = run_at(share.s, share.four, share.step, share.left);
    load_queries(now);
    Halves here = find(now, now.t0);
    load_k(now.k, here);
    load_v(now.v, here);
    __builtin_amdgcn_sched_barrier(0);
    half8 qf[1][D32];
    float undo[1], m[1], l[1];
    float4v acc[1][VW];
    auto start = [&] {
        split_queries<D32, 1, true>(a.scale_log2, heads, width, c, G, q, qf, undo);
        m[0] = -INFINITY;
        l[0] = 0.0f;
#pragma unroll
        for (int j = 0; j < VW; ++j) acc[0][j] = float4v{0, 0, 0, 0};
    };
    int left = share.left, t0 = now.t0, run_from = share.at;     // run_from: the number of the run's first step
    // where the next run begins, found while this one's first rows are on their way
    bool again;
    Run then;
    Halves first_of_then;
    auto look_ahead = [&] {
        again = left - now.take > kRowSteps;
        if (again) {
            then = run_after(now, left - now.take);
            first_of_then = find(then, then.t0);
        }
    };
    look_ahead();
    start();

    for (;;) {
        const bool last = t0 + kStep > now.hi;       // the run's last step
        const bool more = !last || again;
        Halves next = first_of_then;
        if (!last) next = find(now, t0 + kStep);
        const _Float16 *k_next = last ? then.k : now.k, *v_next = last ? then.v : now.v;
        const bool masked = t0 < now.lo || t0 + kStep > now.hi + 1 || !(here.ok[0] && here.ok[1]);
        auto there = [&](int i) {
            const int t = t0 + (i < 4 ? 0 : 16) + G * 4 + (i & 3);
            return t >= now.lo && t <= now.hi && here.ok[i / 4];
        };
        float4v scores[1][2] = {{float4v{0, 0, 0, 0}, float4v{0, 0, 0, 0}}};
#pragma unroll
        for (int d = 0; d < D32; ++d) {
            scores[0][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[0][d], qf[0][d], scores[0][0], 0, 0, 0);
            scores[0][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[1][d], qf[0][d], scores[0][1], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (more) load_k(k_next, next);
        if (last && more) load_queries(then);
        __builtin_amdgcn_sched_barrier(0);
        half8 pf[1];
        weigh<VW, 1>(scores, undo, masked, there, c, m, l, acc, pf);
        if (masked) {                                // 0 * NaN would reach the sums
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool ok = there(i);
#pragma unroll
                for (int u = 0; u < VR; ++u) vr[i][u] = ok ? vr[i][u] : 0;
            }
        }
        add_values<VW, 1>(vr, pf, acc);
        __builtin_amdgcn_sched_barrier(0);
        if (more) load_v(v_next, next);
        __builtin_amdgcn_sched_barrier(0);
        if (last) {
            // sums to the output, or to place (workgroup + row): consecutive for the workgroups of one row
            const int row = now.s * fours + now.four, slot = blockIdx.x + row, head0 = (now.four * kWaves + wave) * a.group;
            const bool single = now.step <= kRowSteps && now.step + now.take == now.steps;
            if (now.step <= kRowSteps && tid == 0)
                a.spans[row] = int2{slot, share.holder(run_from - now.step + now.steps - 1) - static_cast<int>(blockIdx.x) + 1};
            const float total = across_groups_sum(l[0]);
            const int64_t at = ((int64_t)slot * kWaves + wave) * a.group + c;
            const bool mine = c < heads;
            if (mine && G == 0 && !single) {
                a.part_ml[at * 2] = m[0];
                a.part_ml[at * 2 + 1] = total;
            }
            // row 4G + r of product j is value VP * (4G + r) + j % 8 of half j / 8
#pragma unroll
            for (int j = 0; j < VW; j += 4)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = (j / 8) * 128 + (4 * G + r) * VP + j % 8;
                    float4v v;
#pragma unroll
                    for (int u = 0; u < 4; ++u) v[u] = both_parts(acc[0][j + u][r]);
                    if (!mine || d >= width) continue;
                    if (single) {
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            store_output(a, now.s * a.y_stride + (int64_t)(head0 + c) * width + d + u,
                                         total == 0.0f ? 0.0f : v[u] / total);
                    } else {
                        *reinterpret_cast<float4v *>(a.part_o + at * width + d) = v;
                    }
                }
            if (!more) return;
            run_from += now.take;
            left -= now.take;
            now = then;
            look_ahead();
            start();
            t0 = now.t0;
        } else {
            t0 += kStep;
        }
        here = next;
    }
}

// Joins the chunks of one query head: y = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i. Weights by
// one thread per chunk; then groups of threads take the chunks in turn, 4 values
// each, and the groups' sums are added in order.
constexpr int kJoinRun = 1024;                       // chunks whose weights wait in LDS at a time
template <int THREADS, bool EVEN>
__global__ __launch_bounds__(THREADS) void join_chunks(AttendArgs a) {
    __shared__ float weights[kJoinRun];
    __shared__ float4v sums[THREADS];
    __shared__ float reduce[THREADS / kWave];
    const int h = blockIdx.x, s = blockIdx.y, width = a.pool.width, tid = threadIdx.x;
    const int len = length_of(a, s, false);
    int n, step;                                     // chunks, and how many places they are apart
    int64_t at;
    if constexpr (EVEN) {
        const int kvh = h / a.group;
        const int2 span = a.spans[s * (a.pool.heads / kWaves) + kvh / kWaves];
        if (len == 0) {                              // no tokens: zeros
            for (int i = tid; i < width; i += THREADS) store_output(a, s * a.y_stride + (int64_t)h * width + i, 0.0f);
            return;
        }
        n = span.y;
        step = kWaves * a.group;
        at = (int64_t)span.x * step + kvh % kWaves * a.group + h - kvh * a.group;
    } else {
        n = (len - base_of(a, len) + a.chunk - 1) / a.chunk;
        step = 1;
        at = ((int64_t)s * a.query_heads + h) * a.chunks;
    }
    if (n <= 1) return;                              // written by its one chunk
    const float2 *ml = reinterpret_cast<const float2 *>(a.part_ml) + at;
    const float4v *o = reinterpret_cast<const float4v *>(a.part_o + at * width);
    const int vectors = width / 4, groups = THREADS / vectors;
    const int group = tid / vectors, at4 = tid - group * vectors;

    float top = -INFINITY;
    for (int i = tid; i < n; i += THREADS) top = fmaxf(top, ml[(int64_t)i * step].x);
    top = kk::wave_max(top);
    if (tid % kWave == 0) reduce[tid / kWave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / kWave; ++w) top = fmaxf(top, reduce[w]);
    __syncthreads();

    float total = 0.0f;
    float4v sum{0, 0, 0, 0};
    for (int i0 = 0; i0 < n; i0 += kJoinRun) {
        const int run = min(kJoinRun, n - i0);
        for (int i = tid; i < run; i += THREADS) {
            const float2 x = ml[(int64_t)(i0 + i) * step];
            const float w = x.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x.x - top);
            weights[i] = w;
            total += w * x.y;
        }
        // the values of up to 8 chunks a thread are on their way before the weights are known
        for (int j0 = group; j0 < run || j0 == group; j0 += 8 * groups) {
            float4v v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int i = j0 + u * groups;
                v[u] = group < groups && i < run ? o[(int64_t)(i0 + i) * step * vectors + at4] : float4v{0, 0, 0, 0};
            }
            if (j0 == group) __syncthreads();
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int i = j0 + u * groups;
                if (group < groups && i < run) sum += weights[i] * v[u];
            }
        }
        __syncthreads();
    }
    total = kk::wave_sum(total);
    if (tid % kWave == 0) reduce[tid / kWave] = total;
    sums[tid] = sum;
    __syncthreads();
    total = 0.0f;
#pragma unroll
    for (int w = 0; w < THREADS / kWave; ++w) total += reduce[w];
    if (tid < vectors) {
        for (int g = 1; g < groups; ++g) sum += sums[g * vectors + tid];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            store_output(a, s * a.y_stride + (int64_t)h * width + tid * 4 + i, total == 0.0f ? 0.0f : sum[i] / total);
    }
}

// Whether the 16 tokens of a half step are in one page; lane offsets within them are 32-bit.
bool in_halves(const kunlun::KVCacheLayout &c) { return c.page_tokens % 16 == 0 && c.token_stride < (1 << 26); }

struct Plan {
    int group, nt, tiles, chunk, chunks;
    bool halves, once, wide, narrow;
    int shares;                                      // attend_even: workgroups, else 0
};

Plan plan_of(const kunlun::KVCacheLayout &c, const kunlun::PagedAttentionLayout &p, int cus) {
    Plan r;
    r.halves = in_halves(c);
    r.group = p.query_heads / c.heads;
    r.nt = r.group > 8 && c.width <= 128 ? 2 : 1;
    r.tiles = (r.group + 8 * r.nt - 1) / (8 * r.nt);
    const int longest = p.window > 0 ? std::min<int64_t>(p.longest, (int64_t)p.window + kStep - 1) : p.longest;
    const int64_t rows = (int64_t)p.sequences * c.heads * r.tiles;
    // No split, so no second launch: eight waves to a workgroup for rows of up to 512 tokens, or 1024 where they
    // leave few CUs idle, four for more rows of up to 512 (us, against the split or shares: 4 x 160 / 320 / 512 tokens x 8
    // heads 7.8 / 8.6 / 9.6, split 11.1 / 11.2 / 11.5; eight waves at 768 12.6, split 11.5; 32 x 512 / 1024 x 8 heads
    // 13.8 / 26.8, split 18.4, shares 30.8).
    const int whole = kMaxChunk + kStep;             // a window starts up to kStep - 1 tokens early
    r.wide = r.nt == 1 && c.width <= 128 && rows <= cus && longest > kMinChunk &&
             longest <= (rows > cus / 2 ? 2 * whole : whole);
    const int64_t least = r.wide ? longest : rows > cus && longest <= whole ? longest : kMinChunk;
    // Otherwise two workgroups' tokens to a CU, in parts of one size: of up to 512 tokens (1 x 32768 tokens x 8 heads
    // 29.3 us, of 256 32.2); with two rows and more to a CU whole rows of up to 1024 (64 x 640 / 1024 tokens x 8 heads
    // 29.6 / 44, in shares 36 / 50) and, above, at least three parts of up to 1024, where shares do not take them (two parts,
    // three, four: 64 x 2048 x 8 heads of 80 uniform 46.7, 44.6, 45.7, full 75.0, 70.7, 74.0; pages of 24 tokens 64.3,
    // 61.4, 62.9 and 106.6, 107.7, 108.9; 96 x 2048 x 6 heads of 128 70.0, 67.9, 64.6 and 109.9, 107.7, 108.6); of
    // workgroups that a CU holds one or two of instead of three, twice as many tokens (64 x 2048 x 8 heads of 160 143
    // whole, 168 in three parts, uniform 114 and 104; groups of 16 query heads 94 and 119, 68 and 72).
    const int many = c.width > 128 || r.nt == 2 ? 2 * kMaxChunkMany : kMaxChunkMany;
    const int64_t most = rows >= 2 * cus ? many : kMaxChunk;
    const int64_t wanted = std::min<int64_t>((longest * rows + 2 * cus - 1) / (2 * cus), most);
    const int64_t split = std::max({wanted, least, (int64_t)(longest + kMostChunks - 1) / kMostChunks});
    const int64_t least_parts = rows >= 2 * cus && longest > many ? 3 : 1;
    // and a bound on the workgroups that find no tokens where `longest` is far above the lengths
    // (but page ids that wait in LDS have to fit)
    const int64_t id_parts = r.halves ? 1 : (longest + kMostIds * c.page_tokens - 1) / (kMostIds * (int64_t)c.page_tokens);
    const int64_t most_parts = std::max({(1 << 12) / rows, least_parts, id_parts});
    const int64_t asked = std::max((longest + split - 1) / split, least_parts);
    const int64_t parts = std::max(std::min(asked, most_parts), id_parts), chunk = (longest + parts - 1) / parts;
    r.chunk = static_cast<int>((chunk + kMinChunk - 1) / kMinChunk * kMinChunk);
    r.chunks = (longest + r.chunk - 1) / r.chunk;
    // One wave to a workgroup for many rows of up to four steps (512 sequences x 8 heads: 2 / 64 / 128 tokens 31 / 40 / 55 us
    // on four waves, 17 / 33 / 54 on one, 256 tokens 97 / 100; 64 x 8: 128 tokens 10.4 / 11.3; width 256, 60 x 64 tokens x 32
    // heads 60 / 32)
    r.narrow = r.nt == 1 && rows > 2 * cus && longest <= 4 * kStep;
    // The non-temporal hint, for reads of whole cache lines that fill more than a quarter of the 256 MiB cache with
    // nothing that is read again (us by `attend`, with the hint and without: 64 x 1024 x 8 heads 44 / 50; 96 x 2048 x 6 104 /
    // 117, in token order 111 / 119; 64 x 1024 x 8 of 64 24.7 / 27.1; 16 x 1024 x 8, 67 MB, 20.0 / 18.4; tiles that read the
    // same rows, 256 x 2048 with 32 query heads on one, 79 / 65; rows that share lines, 64 x 1024 x 8 of 80, 38.7 / 34.6).
    r.once = r.tiles == 1 && (int64_t)p.sequences * longest * c.heads * c.width * 4 > (64 << 20);
    // Equal shares where rows would be split and there is enough to read (us, by `attend` and in shares, 8 heads of 128, head by
    // head / token by token: 64 sequences uniform to 1536 48 and 43 / 52 and 43, to 4096 98 and 88 / 115 and 91; 16 to
    // 2048 24.6 and 21.1 / 26.6 and 20.8, all 2048 29.7 and 31.9 / 32.2 and 32.1; width 256, 16 to 16384 202 and 150; 1 x
    // 131072 94 and 88). One sequence is even by itself, until the last round of its parts counts little (1 x 32768
    // 29.2 and 31.1). Where `longest` is far above the lengths the shares lose 3 to 4 us (64 to 153 of 1536: 13.0 and 16.4;
    // 64 of 1000, of 32768: 48 and 52). Rows that one workgroup takes whole stay with it (64 x 1024 44 and 50, uniform to
    // 1024 33 and 35), unless they lie token by token (256 x 1024 190 and 170, uniform 118 and 107, 64 x 1024 50 and 51, 37
    // and 35) or few workgroups fit on a CU (width 256, 64 uniform to 768 / 2048 56 and 50 / 126 and 94; width 192 43 and 45
    // / 97 and 83, all 2048 132 and 138).
    const bool together = c.head_stride < c.token_stride;
    const bool share_whole = !r.wide && (c.width > 128 ? longest > kMaxChunk : together && longest > 6 * kMinChunk);
    r.shares = 0;
    if ((r.chunks > 1 || share_whole) && r.halves && r.once && r.nt == 1 && c.heads % kWaves == 0 &&
        (c.width % 64 == 0 || c.width == 96) && p.sequences <= kMostEven &&
        (p.sequences > 1 || (int64_t)longest * c.heads * c.width * 4 > (256 << 20)) &&
        (int64_t)p.sequences * c.heads * (longest / kStep + 3) < INT32_MAX)
        r.shares = c.width <= 64 ? 2 * cus : cus;
    return r;
}

template <int D32, int VW, int NT, bool UNI, bool FULL, bool ONCE, int WAVES>
hipError_t launch(const AttendArgs &a, const Plan &p, int sequences, int heads, hipStream_t stream) {
    const size_t ids = UNI ? 0 : (p.chunk / a.pool.page_tokens + 2) * sizeof(int);
    const size_t sums = (size_t)WAVES * (NT * 8 * 2 + std::min(p.group, 8 * NT) * 16 * VW) * sizeof(float);
    const size_t lds = std::max(ids, sums);          // up to 33 KiB
    hipLaunchKernelGGL((attend<D32, VW, NT, UNI, FULL, ONCE, WAVES>), dim3(heads * p.tiles, sequences, p.chunks),
                       dim3(WAVES * kWave), lds, stream, a);
    return hipGetLastError();
}

template <int D32, int VW, int NT, int WAVES>
hipError_t launch_tiles(const AttendArgs &a, const Plan &p, int sequences, int heads, hipStream_t stream) {
    if (!p.halves) return launch<D32, VW, NT, false, false, false, WAVES>(a, p, sequences, heads, stream);
    if (a.pool.width != 32 * D32) return launch<D32, VW, NT, true, false, false, WAVES>(a, p, sequences, heads, stream);
    if constexpr (WAVES == kWaves) {
        if (p.once) return launch<D32, VW, NT, true, true, true, WAVES>(a, p, sequences, heads, stream);
    }
    return launch<D32, VW, NT, true, true, false, WAVES>(a, p, sequences, heads, stream);
}

template <int D32, int VW>
hipError_t launch_width(const AttendArgs &a, const Plan &p, int sequences, int heads, hipStream_t stream) {
    if (p.shares) {                                  // before any other choice: the join reads what only this kernel writes
        if (a.pool.width != 32 * D32 || !p.halves || p.nt != 1) return hipErrorInvalidValue;
        hipLaunchKernelGGL((attend_even<D32, VW>), dim3(p.shares), dim3(kThreads), 0, stream, a);
        return hipGetLastError();
    }
    if (p.narrow) return launch_tiles<D32, VW, 1, 1>(a, p, sequences, heads, stream);
    if constexpr (VW <= 8) {
        if (p.nt == 2) return launch_tiles<D32, VW, 2, kWaves>(a, p, sequences, heads, stream);
        if (p.wide) return launch_tiles<D32, VW, 1, kWideWaves>(a, p, sequences, heads, stream);
    }
    return launch_tiles<D32, VW, 1, kWaves>(a, p, sequences, heads, stream);
}

// Places of attend_even's sums: every workgroup begins one and every row, for each of its four heads' query heads.
size_t even_parts(const kunlun::KVCacheLayout &c, const kunlun::PagedAttentionLayout &p, const Plan &r) {
    return ((size_t)p.sequences * (c.heads / kWaves) + r.shares) * kWaves * r.group;
}

} // namespace

extern "C" size_t kk_paged_attention_workspace_bytes(const kunlun::KVCacheLayout &c, const kunlun::PagedAttentionLayout &p,
                                          int cus) {
    const Plan r = plan_of(c, p, cus);
    if (r.shares)
        return even_parts(c, p, r) * (c.width + 2) * sizeof(float) + (size_t)p.sequences * (c.heads / kWaves) * sizeof(int2);
    return r.chunks == 1 ? 0 : (size_t)p.sequences * p.query_heads * r.chunks * (c.width + 2) * sizeof(float);
}

extern "C" const char *kk_paged_attention_route(const kunlun::KVCacheLayout &c, const kunlun::PagedAttentionLayout &p,
                                                int cus) {
    const Plan r = plan_of(c, p, cus);
    return r.shares ? "paged_attention_even" : r.chunks > 1 ? "paged_attention_split" : "paged_attention";
}

extern "C" int kk_paged_attention(void *y, const void *q, const void *k, const void *v, const int *table, const int *lengths,
                       const kunlun::KVCacheLayout &c, const kunlun::PagedAttentionLayout &p, void *workspace,
                       int *status, int cus, hipStream_t stream) {
    const Plan r = plan_of(c, p, cus);
    if (c.width <= 0 || c.width > 256 || c.width % 8 || p.sequences > 65535 || r.chunks > kMostChunks ||
        ((r.chunks > 1 || r.shares) && !workspace))
        return hipErrorInvalidValue;
    AttendArgs a;
    a.k = static_cast<const _Float16 *>(k);
    a.v = static_cast<const _Float16 *>(v);
    a.table = table;
    a.lengths = lengths;
    a.q = q;
    a.y = y;
    a.part_o = static_cast<float *>(workspace);
    const size_t parts = r.shares ? even_parts(c, p, r) : (size_t)p.sequences * p.query_heads * r.chunks;
    a.part_ml = a.part_o + parts * c.width;
    a.spans = reinterpret_cast<int2 *>(a.part_ml + parts * 2);
    a.shares = kk::FastDiv(std::max(r.shares, 1));
    a.sequences = p.sequences;
    a.status = status;
    a.pool = PoolView(c);
    a.q_stride = p.q_stride;
    a.y_stride = p.y_stride;
    a.query_heads = p.query_heads;
    a.group = r.group;
    a.tiles = r.tiles;
    a.longest = p.longest;
    a.window = p.window;
    a.row_pages = p.row_pages;
    a.chunk = r.chunk;
    a.chunks = r.chunks;
    a.f16 = p.type == kunlun::InputType::f16;
    a.q_wide = (uintptr_t)q % 16 == 0 && p.q_stride % (a.f16 ? 8 : 4) == 0;
    a.scale_log2 = p.scale * kLog2E;
    hipError_t rc;
    if (c.width <= 64) rc = launch_width<2, 4>(a, r, p.sequences, c.heads, stream);
    else if (c.width <= 96) rc = launch_width<3, 8>(a, r, p.sequences, c.heads, stream);
    else if (c.width <= 128) rc = launch_width<4, 8>(a, r, p.sequences, c.heads, stream);
    else if (c.width <= 192) rc = launch_width<6, 16>(a, r, p.sequences, c.heads, stream);
    else rc = launch_width<8, 16>(a, r, p.sequences, c.heads, stream);
    if (rc != hipSuccess || (r.chunks == 1 && !r.shares)) return rc;
    // one wave where there is little to join
    const bool little = r.shares ? r.shares <= 4 * (int64_t)p.sequences * (c.heads / kWaves) : r.chunks <= 4;
    const dim3 grid(p.query_heads, p.sequences);
    if (r.shares && little) hipLaunchKernelGGL((join_chunks<kWave, true>), grid, dim3(kWave), 0, stream, a);
    else if (r.shares) hipLaunchKernelGGL((join_chunks<kThreads, true>), grid, dim3(kThreads), 0, stream, a);
    else if (little) hipLaunchKernelGGL((join_chunks<kWave, false>), grid, dim3(kWave), 0, stream, a);
    else hipLaunchKernelGGL((join_chunks<kThreads, false>), grid, dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}
