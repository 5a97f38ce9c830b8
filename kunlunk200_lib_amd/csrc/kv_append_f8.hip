// New tokens into a paged key-value cache of e4m3 codes with an F32 scale for every block of tokens and head, their
// queries and keys turned by their position's angles on the way, and tokens read back out of it.
//
// Storing. A block's scale is the least power of two 2^e, e >= -64, that takes the largest value of its new tokens to at most
// 448, the codes' largest, or the scale that its earlier tokens have, where that is as large in size; where it grows the
// earlier codes move down with it. By powers of two that loses nothing above the subnormal codes (2^-6 of the scale and
// below), so a block filled token by token holds what it would hold filled at once, up to those. A value is rounded
// once: keys are turned in F64, where products of F32 factors are exact, and reach F32 rounded to odd, so that rounding
// that to a code's four bits rounds the F64 value (in F32 throughout one code in 2^19 is the neighbour of the nearest). Beside
// an earlier scale that is no power of two, which only another producer leaves, the quotient goes through F32 rounded to odd
// too; of a turned key it is that of the F32 value, for which the F64 one would have to stay in registers.
//
// The first new token of a block finds which follow it. Its lanes, a wave or less for a few tokens as in decoding, a
// workgroup of up to 1024 for more, hold all of the block's new values of one head in registers between the largest and the
// codes; the others leave at once.
// One launch, the queries' workgroups among the others; bound by the bytes it reads and writes where there are many (2047
// tokens of 32 + 8 heads of 128 in F32, 88 MB: 20.3 us), by its chain of look-ups, values, their largest and codes where there
// are few (32 tokens of 32 heads 6.6 us).
#include "device_common.h"
#include "kv_rows.h"
#include "launch.h"
#include "paged.h"

#include <algorithm>
#include <type_traits>

namespace {

using kk::kWave;
using kk::PoolView;

constexpr int kThreads = 256;
constexpr int kLeastExponent = -64;      // of a scale
constexpr int kMostGroups = 2048;        // that look through one entry each
constexpr int kMostWaves = 16;           // of a workgroup
constexpr int kPlaces = 4096;            // of a checking workgroup's table, 16 KB: no fewer workgroups fit on a CU
constexpr int kCheckedAhead = 4;         // entries of a thread on their way

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
    kk::FastDiv q_units_per_token;
    kk::FastDiv units_per_head;          // append: of 8 values; read: pieces of 16 bytes
    kk::FastDiv heads_per_token;         // append: keys' and values'; read: a token's parts
    int tokens, sequences, row_pages, query_heads, rotary, positions;
    int block_log2, blocks;              // tokens of a scale are 2^block_log2; scales of a page and head
    uint32_t q_units;                    // units of kQueryHeads query heads, of all tokens
    uint32_t check_groups;               // workgroups that look for blocks whose tokens stand apart
    uint32_t large_groups;               // workgroups for many new tokens of a block
    uint32_t q_step;                     // the queries' share of all workgroups, of 2^32
    int window;                          // append: entries that a group of lanes looks through
    uint32_t items;                      // append: windows x heads_per_token; read: tokens x parts of one
    uint32_t first;                      // read: the launch's first item
};

// Where token i goes: its sequence and position, or why it goes nowhere.
struct Place {
    int s, pos;
    bool out, bad;                       // left out; reported too
};
__device__ __forceinline__ Place place_of(const F8Args &a, int i) {
    // both loads on their way at once (without positions there are no sequences either: token i is the newest of sequence i)
    const int s = a.sequence ? a.sequence[i] : i, pos = a.position ? a.position[i] : a.lengths[i] - 1;
    const bool bad = s >= a.sequences || (s >= 0 && pos >= 0 && (a.pool.per_page.div(pos) >= static_cast<uint32_t>(a.row_pages) ||
                                                                 (a.rotary > 0 && pos >= a.positions)));
    return Place{s, pos, bad || s < 0 || pos < 0, bad};
}

// The page of a token that is not left out; it may be one that the pool does not have.
__device__ __forceinline__ int page_of(const F8Args &a, const Place &at) {
    return a.table[(int64_t)at.s * a.row_pages + a.pool.per_page.div(at.pos)];
}
__device__ __forceinline__ bool in_pool(const F8Args &a, int page) {
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
    // turn(low, high, cos, sin) for every pair's places in the unit
    template <typename Turn>
    __device__ __forceinline__ void each_pair(const float *cosine, const float *sine, Turn turn) const {
        if constexpr (VEC) {
            if (!turned) return;
            float cs[8], sn[8];
            kk::load_values<float, 4>(cosine + u * 4, cs, 0);
            kk::load_values<float, 4>(sine + u * 4, sn, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) turn(low(j), high(j), cs[j], sn[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < pairs) turn(2 * j, 2 * j + 1, cosine[u * 4 + j], sine[u * 4 + j]);
        }
    }
};

// The same unit of kQueryHeads neighbouring query heads of a token, which share its angles.
constexpr int kQueryHeads = 4;
template <typename T, bool HALVES, bool VEC>
__device__ __forceinline__ void turn_queries(const F8Args &a, uint32_t number) {
    if (number >= a.q_units) return;
    const int token = a.q_units_per_token.div(number), in_token = number - token * a.q_units_per_token.d;
    const int head_group = a.units_per_head.div(in_token), first = head_group * kQueryHeads;
    const int heads = min(kQueryHeads, a.query_heads - first);
    const Place at = place_of(a, token);
    if (at.out) return;                              // reported with the keys
    const int page = page_of(a, at);
    const Unit<T, HALVES, VEC> unit(in_token - head_group * a.units_per_head.d, a.rotary);
    float x[kQueryHeads][8];
#pragma unroll
    for (int n = 0; n < kQueryHeads; ++n)
        unit.load(static_cast<const T *>(a.q) + token * a.q_stride + (first + min(n, heads - 1)) * a.pool.width, x[n]);
    const int64_t angles = (int64_t)at.pos * unit.half;
    unit.each_pair(a.cosine + angles, a.sine + angles, [&](int low, int high, float cs, float sn) {
#pragma unroll
        for (int n = 0; n < kQueryHeads; ++n) {
            const float p = x[n][low], r = x[n][high];
            x[n][low] = fmaf(p, cs, -(r * sn));
            x[n][high] = fmaf(p, sn, r * cs);
        }
    });
    if (!in_pool(a, page)) return;                   // reported with the keys
#pragma unroll
    for (int n = 0; n < kQueryHeads; ++n) {
        if (n >= heads) break;
        T *to = static_cast<T *>(a.q_out) + token * a.q_out_stride + (first + n) * a.pool.width;
        if constexpr (VEC) {
            kk::store_values<T, 4>(to + unit.element(0), x[n], 0);
            kk::store_values<T, 4>(to + unit.element(4), x[n], 4);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) to[unit.element(i)] = static_cast<T>(x[n][i]);
        }
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
// A product to F32, rounded to odd: a code times a scale has up to 28 bits, and rounded to the nearest F32 first, 6 in 10^5 of
// them would reach F16 one step off. (The remainder is not exact for products below 2^-125, which are 0 in F16 and as codes;
// a product past F32's range becomes its largest number.)
__device__ __forceinline__ float times_to_odd(float a, float b) {
    const float y = a * b, rest = fmaf(a, b, -y);
    const uint32_t bits = __float_as_uint(y), odd = (bits - ((bits ^ __float_as_uint(rest)) >> 31)) | 1u;
    return fabsf(rest) > 0.0f ? __uint_as_float(odd) : y;
}

// x / scale to F32, rounded to odd, from y = x times the scale's rounded reciprocal, which is up to 1.5 steps off: a step towards
// the quotient, then the remainder, whose sign is exact, says on which side of it that is.
__device__ __forceinline__ float quotient_to_odd(float x, float scale, float by) {
    const float first = x * by, y = fmaf(fmaf(-first, scale, x), by, first), rest = fmaf(-y, scale, x);
    const uint32_t bits = __float_as_uint(y), odd = (bits - ((bits ^ __float_as_uint(rest) ^ __float_as_uint(scale)) >> 31)) | 1u;
    return fabsf(rest) > 0.0f ? __uint_as_float(odd) : y == first ? first : y;      // (first: 0 with its sign)
}

// Four codes times a factor, each rounded once.
__device__ __forceinline__ uint32_t four_codes_times(uint32_t codes, float by) {
    const float2v a = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(codes, true);
    return four_codes(times_to_odd(a[0], by), times_to_odd(a[1], by), times_to_odd(b[0], by), times_to_odd(b[1], by));
}

// The new tokens of a block, one head of keys or values, by GROUP lanes that hold UNITS units each: entries token + j for
// the bits j of `members`, of which the first stands at sequence s and position pos.
template <typename T, bool HALVES, bool VEC, int GROUP, int UNITS>
__device__ __forceinline__ void store_block(const F8Args &a, int token, int s, int pos, uint64_t members, int hk, int lane,
                                            uint32_t (*tops)[kMostWaves], int &turn) {
    constexpr int kLanes = GROUP < kWave ? GROUP : kWave;                 // of the group that are in one wave
    const int units = a.units_per_head.d;
    const bool is_k = hk < a.pool.heads;
    const int h = is_k ? hk : hk - a.pool.heads;
    const int page_at = a.pool.per_page.div(pos), within = pos - page_at * a.pool.page_tokens;
    const int earlier = within & ((1 << a.block_log2) - 1);               // tokens of the block before these
    const int fresh = (kWave - __builtin_clzll(members)) * units;         // units up to the last one's end
    const int page = a.table[(int64_t)s * a.row_pages + page_at];         // asked about after the values are on their way
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
    if (!in_pool(a, page)) {
        if (hk == 0 && lane == 0) kk::report(a.status, kk::kBadPage);
        return;
    }
#pragma unroll
    for (int n = 0; n < UNITS; ++n) {
        const int number = lane + n * GROUP;
        if (number >= fresh) break;
        const int j = a.units_per_head.div(number);
        if (!(members >> j & 1)) continue;
        const Unit<T, HALVES, VEC> unit(number - j * units, rotary);
        const int64_t angles = (int64_t)(pos + j) * unit.half;
        unit.each_pair(a.cosine + angles, a.sine + angles, [&](int low, int high, float cs, float sn) {
            const double p = x[n][low], r = x[n][high], dc = cs, ds = sn;
            x[n][low] = to_odd(fma(p, dc, -(r * ds)));
            x[n][high] = to_odd(fma(p, ds, r * dc));
        });
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[n][i]) & 0x7fffffffu);
    }
#pragma unroll
    for (int offset = kLanes / 2; offset > 0; offset >>= 1)
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), offset, kWave)));
    if constexpr (GROUP > kWave) {
        // in turn, so that the next block's do not reach these before every wave has read them
        uint32_t *of_waves = tops[turn ^= 1];
        if (lane % kWave == 0) of_waves[lane / kWave] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < GROUP / kWave; ++w) top = max(top, of_waves[w]);
    }

    float *scale_at = (is_k ? a.k_scales : a.v_scales) + ((int64_t)page * a.pool.heads + h) * a.blocks + (within >> a.block_log2);
    uint8_t *block = (is_k ? a.k_pool : a.v_pool) + page * a.pool.page_stride + h * a.pool.head_stride +
                     (int64_t)(within - earlier) * a.pool.token_stride;
    float scale = least_scale(top);
    if (earlier > 0) {
        const float old = *scale_at;
        const bool grows = fabsf(old) < scale;                            // sizes: another producer's scale may be negative
        if (!grows && scale == scale) scale = old;                        // (one that is not a number stays)
        if (grows) {
            const float down = old / scale;
            for (int number = lane; number < earlier * units; number += GROUP) {
                const int j = a.units_per_head.div(number);
                uint2 *codes = reinterpret_cast<uint2 *>(block + j * a.pool.token_stride + (number - j * units) * 8);
                const uint2 old_codes = *codes;
                const uint32_t low = four_codes_times(old_codes.x, down);
                __builtin_amdgcn_sched_barrier(0);                        // (side by side they take 10 registers more)
                *codes = make_uint2(low, four_codes_times(old_codes.y, down));
            }
        }
        if constexpr (GROUP > kWave) __syncthreads();                     // every wave has read the old scale
    }
    if (lane == 0) *scale_at = scale;
    const float by = 1.0f / scale;
    const bool uneven = __any(__float_as_uint(scale) << 9 && scale == scale);   // a kept scale that is no power of two
#pragma unroll
    for (int n = 0; n < UNITS; ++n) {
        const int number = lane + n * GROUP;
        if (number >= fresh) break;
        const int j = a.units_per_head.div(number);
        if (!(members >> j & 1)) continue;
        const Unit<T, HALVES, VEC> unit(number - j * units, rotary);
        uint8_t *to = block + (earlier + j) * a.pool.token_stride;
        uint32_t low, high;
        if (uneven) {
            auto odd = [&](int i) { return quotient_to_odd(x[n][i], scale, by); };
            low = four_codes(odd(0), odd(1), odd(2), odd(3));
            __builtin_amdgcn_sched_barrier(0);
            high = four_codes(odd(4), odd(5), odd(6), odd(7));
        } else {
            low = four_codes(x[n][0] * by, x[n][1] * by, x[n][2] * by, x[n][3] * by);
            high = four_codes(x[n][4] * by, x[n][5] * by, x[n][6] * by, x[n][7] * by);
        }
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

// An entry, in terms that the tokens of one block share where they stand in consecutive entries of consecutive positions.
struct Entry {
    int s, lag, block;                   // sequence, position less number, block of the sequence; s -1: left out
    __device__ __forceinline__ bool same(const Entry &o) const { return s == o.s && lag == o.lag && block == o.block; }
};
__device__ __forceinline__ Entry entry_of(const F8Args &a, int i, bool &bad) {
    const bool there = i >= 0 && i < a.tokens;
    const Place at = place_of(a, there ? i : 0);
    bad = there && at.bad;
    return Entry{there && !at.out ? at.s : -1, at.pos - i, at.pos >> a.block_log2};
}

// The blocks that the entries of one window begin, one head of keys or values, by GROUP lanes. `little`: those whose
// new tokens fit the first kWave units, else the others.
template <typename T, bool HALVES, bool VEC, int GROUP, int UNITS>
__device__ __forceinline__ void store_window(const F8Args &a, uint32_t item, int size, bool little,
                                             uint32_t (*tops)[kMostWaves]) {
    constexpr int kLanes = GROUP < kWave ? GROUP : kWave;
    const int lane = threadIdx.x % GROUP, in_wave = threadIdx.x % kLanes, shift = static_cast<int>(threadIdx.x % kWave) - in_wave;
    const int window = a.heads_per_token.div(item), hk = item - window * a.heads_per_token.d, first = window * size;
    const uint64_t own = kLanes < kWave ? (uint64_t(1) << kLanes % kWave) - 1 : ~uint64_t(0);
    auto of_group = [&](bool what) { return (__ballot(what) >> shift) & own; };
    // the entries before the window, from its first on, and after those: a block's are less than kLanes apart
    bool bad, unused;
    const Entry none{-1, 0, 0}, here = entry_of(a, first + in_wave, bad);
    Entry before = none, after = none, last = none;
    if (a.block_log2 > 0) {
        before = entry_of(a, first + in_wave - kLanes, unused);
        after = entry_of(a, first + in_wave + kLanes, unused);
        last = entry_of(a, first + in_wave - 1, unused);
    }
    if (bad && in_wave < size && little && hk == 0) kk::report(a.status, kk::kBadIndex);
    int turn = 0;
    for (uint64_t left = of_group(in_wave < size && here.s >= 0 && !here.same(last)); left; left &= left - 1) {
        const int at = __builtin_ctzll(left);
        const Entry x{__shfl(here.s, shift + at, kWave), __shfl(here.lag, shift + at, kWave),
                      __shfl(here.block, shift + at, kWave)};
        const uint64_t window_has = of_group(x.same(here));
        // (it follows a left-out entry: an earlier one begins its block)
        if (of_group(x.same(before)) || window_has & ((uint64_t(1) << at) - 1)) continue;
        const uint64_t members = window_has >> at | (at ? of_group(x.same(after)) << (kLanes - at) : 0);
        if (((kWave - __builtin_clzll(members)) * static_cast<int>(a.units_per_head.d) <= kWave) != little) continue;
        const int token = first + at;
        store_block<T, HALVES, VEC, GROUP, UNITS>(a, token, x.s, x.lag + token, members, hk, lane, tops, turn);
    }
}

// Tokens of one block that stand apart in the list (k200.h forbids it) would each begin the block, and chance decides whose scale
// stays. Such a list is reported: workgroup `part` enters the first of every run of a block's tokens, where the hash of sequence
// and block gives it this part, in a table of LDS, and finds there a run of the same block that this one does not go on from.
// Half a table's places are for a part's share of the list; were all taken, the search would end without an answer. Beside the
// others' work: 32 sequences x 32 heads 5.63 -> 5.77 us a call, a prompt of 8000 tokens no change, of 100000 803 -> 818.
template <int THREADS>
__device__ __forceinline__ void check_list(const F8Args &a, uint32_t part, int *places) {
    for (int x = threadIdx.x; x < kPlaces; x += THREADS) places[x] = -1;
    __syncthreads();
    bool unused;
    for (int i0 = threadIdx.x; i0 < a.tokens; i0 += kCheckedAhead * THREADS) {
        Entry here[kCheckedAhead], last[kCheckedAhead];
#pragma unroll
        for (int n = 0; n < kCheckedAhead; ++n) {
            here[n] = entry_of(a, i0 + n * THREADS, unused);
            last[n] = entry_of(a, i0 + n * THREADS - 1, unused);
        }
#pragma unroll
        for (int n = 0; n < kCheckedAhead; ++n) {
            const Entry &x = here[n];
            if (x.s < 0 || x.same(last[n])) continue;
            // by the golden ratio: neighbouring sequences and blocks far apart
            const uint64_t hash = (static_cast<uint64_t>(x.s) << 32 | static_cast<uint32_t>(x.block)) * 0x9e3779b97f4a7c15u;
            if (__umulhi(static_cast<uint32_t>(hash >> 32), a.check_groups) != part) continue;
            uint32_t at = static_cast<uint32_t>(hash >> 32) % kPlaces;
            for (int tries = 0; tries < kPlaces; ++tries, at = (at + 1) % kPlaces) {
                const int other = atomicCAS(places + at, -1, i0 + n * THREADS);
                if (other < 0) break;
                const Entry y = entry_of(a, other, unused);
                if (x.s != y.s || x.block != y.block) continue;
                // (one place named twice is left to the caller, as kv_append leaves it)
                if (x.lag != y.lag && x.lag + i0 + n * THREADS != y.lag + other) kk::report(a.status, kk::kBadIndex);
                break;
            }
        }
    }
}

// The workgroups of the queries, which stream, lie evenly among those of keys and values, which wait for one another's
// results, so that a CU holds both (2047 tokens of 32 + 8 heads of 128: 20.3 us, one kind after the other 26). Of the
// latter first come those that check the list, then those that take many new tokens of a block together, then those of SMALL
// lanes for a block's few new tokens (all of them, where a whole block has no more units).
template <typename T, bool HALVES, bool VEC, int SMALL, int LARGE, int UNITS>
__global__ __launch_bounds__(LARGE ? LARGE : kThreads) void append_f8(F8Args a) {
    constexpr int kGroup = LARGE ? LARGE : kThreads;
    __shared__ uint32_t tops[2][kMostWaves];
    extern __shared__ int places[];      // kPlaces where workgroups check the list
    const uint32_t queries = __umulhi(blockIdx.x, a.q_step);    // of the workgroups before this one
    uint32_t number = blockIdx.x - queries;
    if (__umulhi(blockIdx.x + 1, a.q_step) != queries) {
        turn_queries<T, HALVES, VEC>(a, queries * kGroup + threadIdx.x);
        return;
    }
    if (number < a.check_groups) {
        check_list<kGroup>(a, number, places);
        return;
    }
    number -= a.check_groups;
    if (LARGE > 0 && number < a.large_groups) {
        if constexpr (LARGE > 0) store_window<T, HALVES, VEC, LARGE, UNITS>(a, number, 1 << a.block_log2, false, tops);
    } else {
        const uint32_t item = (number - a.large_groups) * (kGroup / SMALL) + threadIdx.x / SMALL;
        if (item < a.items) store_window<T, HALVES, VEC, SMALL, 1>(a, item, a.window, true, tops);
    }
}

template <typename T, bool HALVES, bool VEC, int SMALL, int LARGE, int UNITS>
int launch_groups(F8Args a, hipStream_t stream) {
    const int threads = LARGE ? LARGE : kThreads, units = a.units_per_head.d, pairs = a.heads_per_token.d;
    const uint32_t q_groups = (a.q_units + threads - 1) / threads;
    // one entry a group, or as many as leave few groups to look through a prompt's (2047 tokens of 8 heads without queries:
    // 2048 groups 12.0 us a call, 8192 14.6)
    const int64_t many = (int64_t)a.tokens * pairs / kMostGroups;
    a.window = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(1 << a.block_log2, many)));
    a.items = static_cast<uint32_t>((a.tokens + a.window - 1) / a.window * pairs);
    const uint32_t small_groups = (a.items * SMALL + threads - 1) / threads;
    const int windows = (a.tokens + (1 << a.block_log2) - 1) >> a.block_log2;
    a.large_groups = LARGE && (int64_t)a.tokens * units > kWave ? windows * pairs : 0;
    // (without positions each entry is a sequence of its own)
    a.check_groups = a.position && a.block_log2 > 0 && a.tokens > 1 ? (a.tokens + kPlaces / 2 - 1) / (kPlaces / 2) : 0;
    // 2^32 q_groups / groups rounded up: the queries' share of the first n is n q_step / 2^32, whole at the last
    const uint64_t groups = (uint64_t)a.check_groups + a.large_groups + small_groups + q_groups;
    a.q_step = static_cast<uint32_t>((((uint64_t)q_groups << 32) + groups - 1) / groups);
    hipLaunchKernelGGL((append_f8<T, HALVES, VEC, SMALL, LARGE, UNITS>), dim3(static_cast<unsigned>(groups)), dim3(threads),
                       a.check_groups ? kPlaces * sizeof(int) : 0, stream, a);
    return hipGetLastError();
}

template <typename T, bool HALVES, bool VEC>
int launch(const F8Args &a, hipStream_t stream) {
    const int units = a.units_per_head.d << a.block_log2;                 // of a whole block, up to 2048
    if (units <= 16) return launch_groups<T, HALVES, VEC, 16, 0, 1>(a, stream);
    if (units <= 32) return launch_groups<T, HALVES, VEC, 32, 0, 1>(a, stream);
    if (units <= 64) return launch_groups<T, HALVES, VEC, 64, 0, 1>(a, stream);
    if (units <= 256) return launch_groups<T, HALVES, VEC, 64, 256, 1>(a, stream);
    if (units <= 1024) return launch_groups<T, HALVES, VEC, 64, 512, 2>(a, stream);
    return launch_groups<T, HALVES, VEC, 64, 1024, 2>(a, stream);
}

// Tokens of the list: their keys' and values' codes times their scales, rounded once where rows are F16. A wave takes one
// token, or a part of its codes, kAhead pieces of N codes a lane with all loads ahead of the stores, which are whole 16-byte
// pieces side by side. Bound by the bytes: 35000 tokens of 8 heads to F32, 359 MB, 77 us (by 8 codes a thread, every thread
// with its own look-ups, 107).
constexpr int kAhead = 8;
constexpr uint32_t kLaunchItems = 1u << 25;          // of one launch, 2^31 threads: it has to stay below 2^32
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void read_f8(F8Args a, T *k_out, T *v_out) {
    constexpr int N = 16 / sizeof(T);
    const uint32_t item = a.first + blockIdx.x * (kThreads / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (item >= a.items) return;
    const int token = a.heads_per_token.div(item), part = item - token * a.heads_per_token.d, lane = threadIdx.x % kWave;
    const Place at = place_of(a, token);
    if (at.out) {
        if (at.bad && part == 0 && lane == 0) kk::report(a.status, kk::kBadIndex);
        return;
    }
    const int page = page_of(a, at);
    if (!in_pool(a, page)) {
        if (part == 0 && lane == 0) kk::report(a.status, kk::kBadPage);
        return;
    }
    const int within = at.pos - a.pool.per_page.div(at.pos) * a.pool.page_tokens;
    const int64_t row = page * a.pool.page_stride + within * a.pool.token_stride;
    const int64_t scales = (int64_t)page * a.pool.heads * a.blocks + (within >> a.block_log2);
    const int pieces = a.units_per_head.d, all = 2 * a.pool.heads * pieces;        // pieces of N codes of a head, of the token
    uint2 codes[kAhead];
    float scale[kAhead];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
        const int x = min((part * kAhead + n) * kWave + lane, all - 1);
        const int hk = a.units_per_head.div(x), piece = x - hk * pieces;
        const bool is_k = hk < a.pool.heads;
        const int h = is_k ? hk : hk - a.pool.heads;
        const uint8_t *from = (is_k ? a.k_pool : a.v_pool) + row + h * a.pool.head_stride + piece * N;
        if constexpr (N == 4) codes[n] = make_uint2(*reinterpret_cast<const uint32_t *>(from), 0);
        else codes[n] = *reinterpret_cast<const uint2 *>(from);
        scale[n] = (is_k ? a.k_scales : a.v_scales)[scales + (int64_t)h * a.blocks];
    }
    auto store = [&](int n, auto odd) {                                   // false: past the last piece
        const int x = (part * kAhead + n) * kWave + lane;
        if (x >= all) return false;
        const int hk = a.units_per_head.div(x), piece = x - hk * pieces;
        const bool is_k = hk < a.pool.heads;
        float y[8];
        if constexpr (odd) {
            eight_values(codes[n], 1.0f, y);
#pragma unroll
            for (int i = 0; i < N; ++i) y[i] = times_to_odd(y[i], scale[n]);
        } else {
            eight_values(codes[n], scale[n], y);
        }
        T *to = (is_k ? k_out + token * a.k_stride + hk * a.pool.width
                      : v_out + token * a.v_stride + (hk - a.pool.heads) * a.pool.width) + piece * N;
        if constexpr (VEC) {
            kk::store_values<T, N>(to, y, 0);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) to[i] = static_cast<T>(y[i]);
        }
        return true;
    };
    // F16 rows round once: products by powers of two are exact, others go to F16 by way of odd ones (always so, 500 tokens of
    // 32 heads take 6.1 us in place of 5.6)
    if constexpr (N == 8) {
        uint32_t uneven = 0;
#pragma unroll
        for (int n = 0; n < kAhead; ++n) uneven |= __float_as_uint(scale[n]) << 9;
        if (__any(uneven)) {
#pragma unroll
            for (int n = 0; n < kAhead; ++n)
                if (!store(n, std::true_type())) break;
            return;
        }
    }
#pragma unroll
    for (int n = 0; n < kAhead; ++n)
        if (!store(n, std::false_type())) break;
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
    const int64_t query_groups = (query_heads + kQueryHeads - 1) / kQueryHeads;
    a.q_units_per_token = kk::FastDiv(static_cast<uint32_t>(query_heads ? query_groups * per_head : 1));
    a.q_units = static_cast<uint32_t>(query_groups * per_head * p.tokens);
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
    if ((int64_t)p.tokens * 2 * c.heads * (c.width / 8) > INT32_MAX - 1024) return hipErrorInvalidValue;
    const bool f16 = p.type == kunlun::InputType::f16;
    const bool vec = ((uintptr_t)k_out | (uintptr_t)v_out) % 16 == 0 && (p.k_stride | p.v_stride) % (f16 ? 8 : 4) == 0;
    // pieces of 16 bytes of a row; parts of a token that a wave takes
    const int pieces = c.width / (f16 ? 8 : 4), parts = (2 * c.heads * pieces + kAhead * kWave - 1) / (kAhead * kWave);
    a.units_per_head = kk::FastDiv(pieces);
    a.heads_per_token = kk::FastDiv(parts);
    a.items = static_cast<uint32_t>(p.tokens * parts);
    _Float16 *kh = static_cast<_Float16 *>(k_out), *vh = static_cast<_Float16 *>(v_out);
    float *kf = static_cast<float *>(k_out), *vf = static_cast<float *>(v_out);
    for (a.first = 0; a.first < a.items; a.first += kLaunchItems) {
        const dim3 grid((std::min(a.items - a.first, kLaunchItems) + kThreads / kWave - 1) / (kThreads / kWave));
        if (f16 && vec) hipLaunchKernelGGL((read_f8<_Float16, true>), grid, dim3(kThreads), 0, stream, a, kh, vh);
        else if (f16) hipLaunchKernelGGL((read_f8<_Float16, false>), grid, dim3(kThreads), 0, stream, a, kh, vh);
        else if (vec) hipLaunchKernelGGL((read_f8<float, true>), grid, dim3(kThreads), 0, stream, a, kf, vf);
        else hipLaunchKernelGGL((read_f8<float, false>), grid, dim3(kThreads), 0, stream, a, kf, vf);
        if (const hipError_t rc = hipGetLastError()) return rc;
    }
    return hipSuccess;
}
