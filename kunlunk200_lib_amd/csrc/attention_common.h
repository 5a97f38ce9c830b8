// What the attention kernels over paged caches share: arguments, a query's two F16 parts and the scores they give,
// equal shares of all rows' steps, and the join of parts. Internal linkage: each kernel file has its own copy.
#pragma once

#include "device_common.h"
#include "paged.h"

namespace {

using kk::half8;
using kk::kWave;
using kk::PoolView;

typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kStep = 32;                // tokens of a wave's step
constexpr float kLeastPart = 0x1p-24f;    // the least F16 above 0

struct AttendArgs {
    const void *k, *v;
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

// What a workgroup takes of a launch over (key-value heads x tiles of query heads, sequences, parts).
struct Part {
    int s, chunk, kvh, tile;
};
__device__ __forceinline__ Part part_of(const AttendArgs &a) {
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
    return {s, chunk, kvh, tile};
}

// A word that no lane writes during the launch, read through the scalar cache.
template <typename T>
__device__ __forceinline__ T scalar_load(const T *p) {
    return *(const __attribute__((address_space(4))) T *)(p);
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

// Eight values of a row of q (16-byte loads where a.q_wide allows); F16 as they are in the first four registers, so that
// nothing waits for them here.
__device__ __forceinline__ void load_query(const AttendArgs &a, int64_t at, float4v (&v)[2]) {
    if (a.f16) {
        const _Float16 *q = static_cast<const _Float16 *>(a.q) + at;
        if (a.q_wide) {
            v[0] = *reinterpret_cast<const float4v *>(q);
        } else {
            half8 x;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = q[i];
            v[0] = __builtin_bit_cast(float4v, x);
        }
    } else {
        const float *q = static_cast<const float *>(a.q) + at;
        if (a.q_wide) {
            v[0] = *reinterpret_cast<const float4v *>(q);
            v[1] = *reinterpret_cast<const float4v *>(q + 4);
        } else {
            v[0] = float4v{q[0], q[1], q[2], q[3]};
            v[1] = float4v{q[4], q[5], q[6], q[7]};
        }
    }
}

// A lane's part of a cache row; ONCE: with the non-temporal hint.
template <typename T, bool ONCE>
__device__ __forceinline__ T load_row(const void *p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(static_cast<const T *>(p));
    else return *static_cast<const T *>(p);
}

// The exponent of a float's size: 128 for what is not finite, -127 for 0 and subnormal ones.
__device__ __forceinline__ int exponent_of(float v) { return static_cast<int>((__float_as_uint(v) >> 23) & 0xff) - 127; }

// q columns: column c is head c % 8 of each tile, its high (c < 8) or low part; the scores times `undo` are in base 2.
// in(d): whether the lane's piece d of a row is within the width. `loaded`: as load_query left it.
template <int D32, int NT, typename In>
__device__ __forceinline__ void split_queries(bool f16, float scale_log2, int heads, int c, In in,
                                              const float4v (&loaded)[NT][D32][2], half8 (&qf)[NT][D32], float (&undo)[NT]) {
    float q[NT][D32][8];
    if (f16) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int d = 0; d < D32; ++d)
#pragma unroll
                for (int i = 0; i < 8; ++i) q[nt][d][i] = static_cast<float>(__builtin_bit_cast(half8, loaded[nt][d][0])[i]);
    } else {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int d = 0; d < D32; ++d)
#pragma unroll
                for (int i = 0; i < 8; ++i) q[nt][d][i] = loaded[nt][d][i / 4][i % 4];
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const bool column = nt * 8 + (c & 7) < heads;
        float top = 0.0f;
#pragma unroll
        for (int d = 0; d < D32; ++d)
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, in(d) ? fabsf(q[nt][d][i]) : 0.0f);
        const int size = exponent_of(across_groups_max(top));
        // 2^e with top * |scale| * 2^e in [2^9, 2^11); beside an infinite value every finite one stays finite
        const int e = max(-126, min(126, min(9 - size, 110) - exponent_of(scale_log2)));
        undo[nt] = ldexpf(1.0f, -e);
        const float factor = column ? ldexpf(scale_log2, e) : 0.0f;
#pragma unroll
        for (int d = 0; d < D32; ++d) {
            const float by = in(d) ? factor : 0.0f;
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

// A step's scores, both parts together.
__device__ __forceinline__ void whole_scores(const float4v (&scores)[2], float undo, int c, float (&sc)[8]) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float part = scores[i / 4][i % 4];
        sc[i] = (part + other_part(part)) * undo;
        sum += sc[i];
    }
    if (__any(!(fabsf(sum) < INFINITY))) {
        // infinite keys or queries: the high part's infinity, as F32 products have it
        // (its low part gives NaN or the other sign)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float part = scores[i / 4][i % 4], other = other_part(part);
            const float high = c < 8 ? part : other;
            if (fabsf(high) == INFINITY) sc[i] = high;
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
// A row's first ROW_STEPS steps are empty: what it costs to begin it.
struct Share {
    int at, left;
    int s, four, step;                               // where `at` is
    int per, extra;                                  // steps of a share; the first `extra` shares have one more
    __device__ __forceinline__ int holder(int step_number) const {
        const int cut = extra * (per + 1);
        return step_number < cut ? step_number / (per + 1) : extra + (step_number - cut) / per;
    }
};

// Sequence s's length as a lane reads it.
__device__ __forceinline__ int lane_length(const AttendArgs &a, int s, bool tell) {
    int len = a.lengths[s];
    if (len < 0 || len > a.longest) {
        if (tell) kk::report(a.status, kk::kBadIndex);
        len = len < 0 ? 0 : a.longest;
    }
    return len;
}

template <int ROW_STEPS, typename Length>
__device__ __forceinline__ Share share_of(const AttendArgs &a, int number, int fours, int lane, Length length) {
    auto steps = [&](int s) {
        if (s >= a.sequences) return 0;
        const int n = steps_of(a, length(s));
        return n ? (n + ROW_STEPS) * fours : 0;
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

} // namespace
