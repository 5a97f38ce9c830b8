// New tokens into a paged key-value cache of e4m3 codes with an F32 scale for every block of tokens and head, their
// queries and keys turned by their position's angles on the way, and tokens read back out of it.
//
// Storing. A block's scale is the least power of two 2^e, e >= -64, that takes the largest value of its new tokens to at most
// 448, the codes' largest, or the scale that its earlier tokens have, where that is larger; where it grows the
// earlier codes move down with it. By powers of two that loses nothing above the subnormal codes (2^-6 of the scale and
// below), so a block filled token by token holds what it would hold filled at once, up to those. A value is rounded
// once: keys are turned in F64, where products of F32 factors are exact, and reach F32 rounded to odd, so that rounding
// that to a code's four bits rounds the F64 value (in F32 throughout one code in 2^19 is the neighbour of the nearest).
//
// The first new token of a block finds which follow it; its GROUP lanes (16 to 256, by the block's values) hold all of
// the block's new values of one head in registers between the largest and the codes. The other tokens' lanes leave at once.
// One launch with the queries in front; bound by the bytes it reads and writes.
#include "device_common.h"
#include "kv_rows.h"
#include "launch.h"
#include "paged.h"

namespace {

using kk::kWave;
using kk::PoolView;

constexpr int kThreads = 256;
constexpr int kLeastExponent = -64;      // of a scale

typedef float float2v __attribute__((ext_vector_type(2)));

struct F8Args {
    uint8_t *k_pool, *v_pool;
    float *k_scales, *v_scales;
    void *q_out;
    const void *q, *k, *v;
    const int *sequence, *position, *lengths, *table;
    const float *cosine, *sine;
    int *status;
    PoolView pool;
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    kk::FastDiv q_units_per_token, units_per_head, heads_per_token;   // heads_per_token: keys' and values'
    int tokens, sequences, row_pages, query_heads, rotary, positions;
    int block_log2, blocks;              // tokens of a scale are 2^block_log2; scales of a page and head
    uint32_t q_units, q_groups;          // 8-value units of all queries, and the workgroups that take them
    int64_t items;                       // tokens x heads_per_token
};

// Where token i goes: its sequence and position, or why it goes nowhere.
struct Place {
    int s, pos;
    bool out, bad;                       // left out; reported
};
__device__ __forceinline__ Place place_of(const F8Args &a, int i) {
    Place r{a.sequence ? a.sequence[i] : i, -1, true, false};
    if (r.s < 0) return r;
    r.bad = r.s >= a.sequences;
    if (r.bad) return r;
    r.pos = a.position ? a.position[i] : a.lengths[r.s] - 1;
    if (r.pos < 0) return r;
    r.bad = a.pool.per_page.div(r.pos) >= static_cast<uint32_t>(a.row_pages) || (a.rotary > 0 && r.pos >= a.positions);
    r.out = r.bad;
    return r;
}

__device__ __forceinline__ bool page_of(const F8Args &a, const Place &at, int &page) {
    page = a.table[(int64_t)at.s * a.row_pages + a.pool.per_page.div(at.pos)];
    return static_cast<unsigned>(page) < static_cast<unsigned>(a.pool.pages);
}

// d to F32, rounded to odd: towards zero, with the last bit set where that is not exact.
__device__ __forceinline__ float to_odd(double d) {
    const float y = static_cast<float>(d);
    const double back = static_cast<double>(y);
    if (back == d || !(fabs(d) < INFINITY)) return y;
    const uint32_t bits = __float_as_uint(y) - (fabs(back) > fabs(d) ? 1u : 0u);
    return __uint_as_float(bits | 1u);
}

// Unit u of a head: 8 values, of which the first 2 * pairs are turned pairs; element(i) is value i's place in the head.
// VEC: consecutive values, or of a head turned in halves 4 of the first half and their partners.
template <typename T, bool HALVES, bool VEC>
struct Unit {
    int u, half, pairs;
    bool turned;
    __device__ __forceinline__ Unit(int unit, int rotary) : u(unit), half(rotary / 2) {
        pairs = min(4, max(0, half - u * 4));
        turned = pairs > 0;
    }
    __device__ __forceinline__ int element(int i) const {
        if (VEC) return HALVES && turned ? (i < 4 ? u * 4 + i : half + u * 4 + i - 4) : u * 8 + i;
        if (i >= 2 * pairs) return u * 8 + i;
        const int j = u * 4 + i / 2;
        return HALVES ? (i & 1 ? half + j : j) : 2 * j + (i & 1);
    }
    // the places in the unit of pair j's values
    __device__ __forceinline__ int low(int j) const { return VEC && HALVES ? j : 2 * j; }
    __device__ __forceinline__ int high(int j) const { return VEC && HALVES ? j + 4 : 2 * j + 1; }
    __device__ __forceinline__ void load(const T *from, float (&x)[8]) const {
        if constexpr (VEC) {
            kk::load_values<T, 4>(from + element(0), x, 0);
            kk::load_values<T, 4>(from + element(4), x, 4);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(from[element(i)]);
        }
    }
    // turn(a, b, cos, sin) on every pair
    template <typename Turn>
    __device__ __forceinline__ void each_pair(const float *cosine, const float *sine, float (&x)[8], Turn turn) const {
        if constexpr (VEC) {
            if (!turned) return;
            float cs[8], sn[8];
            kk::load_values<float, 4>(cosine + u * 4, cs, 0);
            kk::load_values<float, 4>(sine + u * 4, sn, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) turn(x[low(j)], x[high(j)], cs[j], sn[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < pairs) turn(x[2 * j], x[2 * j + 1], cosine[u * 4 + j], sine[u * 4 + j]);
        }
    }
};

template <typename T, bool HALVES, bool VEC>
__device__ __forceinline__ void turn_query(const F8Args &a) {
    const uint32_t number = blockIdx.x * kThreads + threadIdx.x;
    if (number >= a.q_units) return;
    const int token = a.q_units_per_token.div(number), in_token = number - token * a.q_units_per_token.d;
    const int head = a.units_per_head.div(in_token);
    const Place at = place_of(a, token);
    int page;
    if (at.out || !page_of(a, at, page)) return;     // reported with the keys
    const Unit<T, HALVES, VEC> unit(in_token - head * a.units_per_head.d, a.rotary);
    float x[8];
    unit.load(static_cast<const T *>(a.q) + token * a.q_stride + head * a.pool.width, x);
    const int64_t angles = (int64_t)at.pos * unit.half;
    unit.each_pair(a.cosine + angles, a.sine + angles, x, [](float &p, float &r, float cs, float sn) {
        const float y = fmaf(p, cs, -(r * sn));
        r = fmaf(p, sn, r * cs);
        p = y;
    });
    T *to = static_cast<T *>(a.q_out) + token * a.q_out_stride + head * a.pool.width;
    if constexpr (VEC) {
        kk::store_values<T, 4>(to + unit.element(0), x, 0);
        kk::store_values<T, 4>(to + unit.element(4), x, 4);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) to[unit.element(i)] = static_cast<T>(x[i]);
    }
}

// The least scale that takes a size of these bits to 448 = 1.75 * 2^8; NaN for what is not finite.
__device__ __forceinline__ float least_scale(uint32_t bits) {
    if (bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    const int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return __uint_as_float(static_cast<uint32_t>(max(e, kLeastExponent) + 127) << 23);
}

__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d) {
    return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}
__device__ __forceinline__ void eight_values(uint2 codes, float scale, float (&x)[8]) {
    const float2v a = __builtin_amdgcn_cvt_pk_f32_fp8(codes.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(codes.x, true);
    const float2v c = __builtin_amdgcn_cvt_pk_f32_fp8(codes.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8(codes.y, true);
    x[0] = a[0] * scale, x[1] = a[1] * scale, x[2] = b[0] * scale, x[3] = b[1] * scale;
    x[4] = c[0] * scale, x[5] = c[1] * scale, x[6] = d[0] * scale, x[7] = d[1] * scale;
}

// UNITS: units a lane holds at most.
template <typename T, bool HALVES, bool VEC, int GROUP, int UNITS>
__global__ __launch_bounds__(kThreads) void append_f8(F8Args a) {
    if (blockIdx.x < a.q_groups) {
        turn_query<T, HALVES, VEC>(a);
        return;
    }
    constexpr int kLanes = GROUP < kWave ? GROUP : kWave;                 // of the group that are in one wave
    __shared__ uint32_t tops[kThreads / kWave];
    const int64_t number = (int64_t)(blockIdx.x - a.q_groups) * (kThreads / GROUP) + threadIdx.x / GROUP;
    if (number >= a.items) return;
    const int lane = threadIdx.x % GROUP, in_wave = threadIdx.x % kLanes;
    const uint32_t item = static_cast<uint32_t>(number);
    const int token = a.heads_per_token.div(item), hk = item - token * a.heads_per_token.d;
    const bool is_k = hk < a.pool.heads;
    const int h = is_k ? hk : hk - a.pool.heads;
    const Place at = place_of(a, token);
    if (at.out) {
        if (at.bad && hk == 0 && lane == 0) kk::report(a.status, kk::kBadIndex);
        return;
    }
    const int block_tokens = 1 << a.block_log2;
    const int page_at = a.pool.per_page.div(at.pos), within = at.pos - page_at * a.pool.page_tokens;
    const int earlier = within & (block_tokens - 1);                      // tokens of the block before this one
    // Whether a token before this one in the block is among the entries before it (that one's lanes, or an earlier one's,
    // have this one too), and which of those that may follow do; entries in between may be left out.
    auto names = [&](int distance) {
        const Place x = place_of(a, token + distance);
        return !x.out && x.s == at.s && x.pos == at.pos + distance;
    };
    const bool precedes = in_wave < min(earlier, token) && names(-1 - in_wave);
    const bool follows = in_wave == 0 || (in_wave < min(block_tokens - earlier, a.tokens - token) && names(in_wave));
    const int shift = static_cast<int>(threadIdx.x % kWave) - in_wave;
    const uint64_t own = (kLanes < kWave ? (uint64_t(1) << kLanes % kWave) - 1 : ~uint64_t(0));
    if ((__ballot(precedes) >> shift) & own) return;
    const uint64_t members = (__ballot(follows) >> shift) & own;
    int page;
    if (!page_of(a, at, page)) {
        if (hk == 0 && lane == 0) kk::report(a.status, kk::kBadPage);
        return;
    }
    const int units = a.units_per_head.d, fresh = (kWave - __builtin_clzll(members)) * units;     // up to the last one's end
    const T *from = (is_k ? static_cast<const T *>(a.k) + token * a.k_stride : static_cast<const T *>(a.v) + token * a.v_stride) +
                    h * a.pool.width;
    const int64_t stride = is_k ? a.k_stride : a.v_stride;
    const int rotary = is_k ? a.rotary : 0;
    float x[UNITS][8];
    uint32_t top = 0;
#pragma unroll
    for (int n = 0; n < UNITS; ++n) {
        const int number = lane + n * GROUP;
        if (number >= fresh) break;
        const int j = a.units_per_head.div(number);
        if (!(members >> j & 1)) continue;
        const Unit<T, HALVES, VEC> unit(number - j * units, rotary);
        unit.load(from + j * stride, x[n]);
    }
#pragma unroll
    for (int n = 0; n < UNITS; ++n) {
        const int number = lane + n * GROUP;
        if (number >= fresh) break;
        const int j = a.units_per_head.div(number);
        if (!(members >> j & 1)) continue;
        const Unit<T, HALVES, VEC> unit(number - j * units, rotary);
        const int64_t angles = (int64_t)(at.pos + j) * unit.half;
        unit.each_pair(a.cosine + angles, a.sine + angles, x[n], [](float &p, float &r, float cs, float sn) {
            const double dp = p, dr = r, dc = cs, ds = sn;
            p = to_odd(fma(dp, dc, -(dr * ds)));
            r = to_odd(fma(dp, ds, dr * dc));
        });
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[n][i]) & 0x7fffffffu);
    }
#pragma unroll
    for (int offset = kLanes / 2; offset > 0; offset >>= 1)
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), offset, kWave)));
    if constexpr (GROUP > kWave) {
        if (in_wave == 0) tops[threadIdx.x / kWave] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / kWave; ++w) top = max(top, tops[w]);
    }

    float *scale_at = (is_k ? a.k_scales : a.v_scales) + ((int64_t)page * a.pool.heads + h) * a.blocks + (within >> a.block_log2);
    uint8_t *block = (is_k ? a.k_pool : a.v_pool) + page * a.pool.page_stride + h * a.pool.head_stride +
                     (int64_t)(within - earlier) * a.pool.token_stride;
    float scale = least_scale(top);
    if (earlier > 0) {
        const float old = *scale_at;
        if (!(old <= scale) && scale == scale) scale = old;               // (a scale that is not a number stays)
        if (scale > old) {
            const float down = old / scale;
            for (int number = lane; number < earlier * units; number += GROUP) {
                const int j = a.units_per_head.div(number);
                uint2 *codes = reinterpret_cast<uint2 *>(block + j * a.pool.token_stride + (number - j * units) * 8);
                float y[8];
                eight_values(*codes, down, y);
                *codes = make_uint2(four_codes(y[0], y[1], y[2], y[3]), four_codes(y[4], y[5], y[6], y[7]));
            }
        }
        if constexpr (GROUP > kWave) __syncthreads();                     // every wave has read the old scale
    }
    if (lane == 0) *scale_at = scale;
    const float by = 1.0f / scale;
#pragma unroll
    for (int n = 0; n < UNITS; ++n) {
        const int number = lane + n * GROUP;
        if (number >= fresh) break;
        const int j = a.units_per_head.div(number);
        if (!(members >> j & 1)) continue;
        const Unit<T, HALVES, VEC> unit(number - j * units, rotary);
        uint8_t *to = block + (earlier + j) * a.pool.token_stride;
        const uint32_t low = four_codes(x[n][0] * by, x[n][1] * by, x[n][2] * by, x[n][3] * by);
        const uint32_t high = four_codes(x[n][4] * by, x[n][5] * by, x[n][6] * by, x[n][7] * by);
        if constexpr (VEC) {
            if (HALVES && unit.turned) {
                *reinterpret_cast<uint32_t *>(to + unit.element(0)) = low;
                *reinterpret_cast<uint32_t *>(to + unit.element(4)) = high;
            } else {
                *reinterpret_cast<uint2 *>(to + unit.element(0)) = make_uint2(low, high);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) to[unit.element(i)] = static_cast<uint8_t>((i < 4 ? low : high) >> (i % 4 * 8));
        }
    }
}

template <typename T, bool HALVES, bool VEC>
int launch(const F8Args &a, hipStream_t stream) {
    const int units = a.units_per_head.d << a.block_log2;                 // of a whole block, up to 2048
    const int group = units <= 16 ? 16 : units <= 32 ? 32 : units <= 4 * kWave ? 64 : 256;
    const int64_t groups = a.q_groups + (a.items + kThreads / group - 1) / (kThreads / group);
    if (groups > INT32_MAX / kThreads) return hipErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(groups));
    if (group == 16) hipLaunchKernelGGL((append_f8<T, HALVES, VEC, 16, 1>), grid, dim3(kThreads), 0, stream, a);
    else if (group == 32) hipLaunchKernelGGL((append_f8<T, HALVES, VEC, 32, 1>), grid, dim3(kThreads), 0, stream, a);
    else if (group == 64) hipLaunchKernelGGL((append_f8<T, HALVES, VEC, 64, 4>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((append_f8<T, HALVES, VEC, 256, 8>), grid, dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

// Token i of the list: its keys' and values' codes times their scales, rounded once where rows are F16. A thread takes 8
// values.
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void read_f8(F8Args a, T *k_out, T *v_out) {
    const int64_t number = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (number >= a.items) return;
    const uint32_t item = a.units_per_head.div(static_cast<uint32_t>(number));
    const int u = static_cast<uint32_t>(number) - item * a.units_per_head.d;
    const int token = a.heads_per_token.div(item), hk = item - token * a.heads_per_token.d;
    const bool is_k = hk < a.pool.heads;
    const int h = is_k ? hk : hk - a.pool.heads;
    const Place at = place_of(a, token);
    if (at.out) {
        if (at.bad && hk == 0 && u == 0) kk::report(a.status, kk::kBadIndex);
        return;
    }
    int page;
    if (!page_of(a, at, page)) {
        if (hk == 0 && u == 0) kk::report(a.status, kk::kBadPage);
        return;
    }
    const int within = at.pos - a.pool.per_page.div(at.pos) * a.pool.page_tokens;
    const float scale = (is_k ? a.k_scales : a.v_scales)[((int64_t)page * a.pool.heads + h) * a.blocks + (within >> a.block_log2)];
    const uint8_t *codes = (is_k ? a.k_pool : a.v_pool) + page * a.pool.page_stride + h * a.pool.head_stride +
                           within * a.pool.token_stride + u * 8;
    float x[8];
    eight_values(*reinterpret_cast<const uint2 *>(codes), scale, x);
    T *to = (is_k ? k_out + token * a.k_stride : v_out + token * a.v_stride) + h * a.pool.width + u * 8;
    if constexpr (VEC) {
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 8; i += N) kk::store_values<T, N>(to + i, x, i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) to[i] = static_cast<T>(x[i]);
    }
}

F8Args args_of(const void *k_pool, const void *v_pool, const float *k_scales, const float *v_scales, const int *sequence,
               const int *position, const int *lengths, const int *table, const kunlun::KVCacheF8Layout &f8, int tokens,
               int sequences, int row_pages, int *status) {
    const kunlun::KVCacheLayout &c = f8.cache;
    F8Args a{};
    a.k_pool = static_cast<uint8_t *>(const_cast<void *>(k_pool));
    a.v_pool = static_cast<uint8_t *>(const_cast<void *>(v_pool));
    a.k_scales = const_cast<float *>(k_scales);
    a.v_scales = const_cast<float *>(v_scales);
    a.sequence = sequence;
    a.position = position;
    a.lengths = lengths;
    a.table = table;
    a.status = status;
    a.pool = PoolView(c);
    a.units_per_head = kk::FastDiv(static_cast<uint32_t>(c.width / 8));
    a.heads_per_token = kk::FastDiv(static_cast<uint32_t>(2 * c.heads));
    a.tokens = tokens;
    a.sequences = sequences;
    a.row_pages = row_pages;
    a.block_log2 = __builtin_ctz(f8.block_tokens);
    a.blocks = c.page_tokens / f8.block_tokens;
    return a;
}

} // namespace

extern "C" int kk_kv_append_f8(void *k_pool, void *v_pool, float *k_scales, float *v_scales, void *q_out, const void *q,
                               const void *k, const void *v, const int *sequence, const int *position, const int *lengths,
                               const int *table, const float *cosine, const float *sine,
                               const kunlun::KVCacheF8Layout &f8, const kunlun::KVAppendLayout &p, int *status,
                               hipStream_t stream) {
    const kunlun::KVCacheLayout &c = f8.cache;
    const int64_t query_heads = q ? p.query_heads : 0, per_head = c.width / 8;
    if ((query_heads + 2 * (int64_t)c.heads) * per_head * p.tokens > INT32_MAX - 1024 || f8.block_tokens <= 0 ||
        f8.block_tokens > 64 || c.width > 256)
        return hipErrorInvalidValue;
    F8Args a = args_of(k_pool, v_pool, k_scales, v_scales, sequence, position, lengths, table, f8, p.tokens, p.sequences,
                       p.row_pages, status);
    a.q_out = q_out;
    a.q = q;
    a.k = k;
    a.v = v;
    a.cosine = cosine;
    a.sine = sine;
    a.q_stride = p.q_stride;
    a.k_stride = p.k_stride;
    a.v_stride = p.v_stride;
    a.q_out_stride = p.q_out_stride;
    a.query_heads = static_cast<int>(query_heads);
    a.rotary = p.rotary;
    a.positions = p.positions;
    a.q_units_per_token = kk::FastDiv(static_cast<uint32_t>(query_heads ? query_heads * per_head : 1));
    a.q_units = static_cast<uint32_t>(query_heads * per_head * p.tokens);
    a.q_groups = (a.q_units + kThreads - 1) / kThreads;
    a.items = (int64_t)p.tokens * 2 * c.heads;
    const bool f16 = p.type == kunlun::InputType::f16, halves = p.pairs == kunlun::RotaryPairs::halves;
    // loads and stores of 4 values: rows on 4 values, the rotated part whole units
    const int64_t strides = p.k_stride | p.v_stride | (q ? p.q_stride | p.q_out_stride : 0);
    const uintptr_t rows = (uintptr_t)k | (uintptr_t)v | (uintptr_t)q | (q ? (uintptr_t)q_out : 0);
    const bool vec = p.rotary % 8 == 0 && strides % 4 == 0 && rows % (f16 ? 8 : 16) == 0 &&
                     (p.rotary == 0 || ((uintptr_t)cosine | (uintptr_t)sine) % 16 == 0);
    if (f16 && halves) return vec ? launch<_Float16, true, true>(a, stream) : launch<_Float16, true, false>(a, stream);
    if (f16) return vec ? launch<_Float16, false, true>(a, stream) : launch<_Float16, false, false>(a, stream);
    if (halves) return vec ? launch<float, true, true>(a, stream) : launch<float, true, false>(a, stream);
    return vec ? launch<float, false, true>(a, stream) : launch<float, false, false>(a, stream);
}

extern "C" int kk_kv_read_f8(void *k_out, void *v_out, const void *k_pool, const void *v_pool, const float *k_scales,
                             const float *v_scales, const int *sequence, const int *position, const int *lengths,
                             const int *table, const kunlun::KVCacheF8Layout &f8, const kunlun::KVReadLayout &p, int *status,
                             hipStream_t stream) {
    const kunlun::KVCacheLayout &c = f8.cache;
    F8Args a = args_of(k_pool, v_pool, k_scales, v_scales, sequence, position, lengths, table, f8, p.tokens, p.sequences,
                       p.row_pages, status);
    a.k_stride = p.k_stride;
    a.v_stride = p.v_stride;
    a.items = (int64_t)p.tokens * 2 * c.heads * (c.width / 8);
    if (a.items > INT32_MAX - 1024) return hipErrorInvalidValue;
    const bool f16 = p.type == kunlun::InputType::f16;
    const bool vec = ((uintptr_t)k_out | (uintptr_t)v_out) % 16 == 0 && (p.k_stride | p.v_stride) % (f16 ? 8 : 4) == 0;
    const dim3 grid(static_cast<unsigned>((a.items + kThreads - 1) / kThreads));
    _Float16 *kh = static_cast<_Float16 *>(k_out), *vh = static_cast<_Float16 *>(v_out);
    float *kf = static_cast<float *>(k_out), *vf = static_cast<float *>(v_out);
    if (f16 && vec) hipLaunchKernelGGL((read_f8<_Float16, true>), grid, dim3(kThreads), 0, stream, a, kh, vh);
    else if (f16) hipLaunchKernelGGL((read_f8<_Float16, false>), grid, dim3(kThreads), 0, stream, a, kh, vh);
    else if (vec) hipLaunchKernelGGL((read_f8<float, true>), grid, dim3(kThreads), 0, stream, a, kf, vf);
    else hipLaunchKernelGGL((read_f8<float, false>), grid, dim3(kThreads), 0, stream, a, kf, vf);
    return hipGetLastError();
}
