// Attention of one new token per sequence over a paged cache in 8 bits: e4m3 codes c with an F32 scale for every block of
// tokens and head, k_t = ks_t c, v_t = vs_t c.
//
// For query head h of sequence s, with key-value head h / group,
//   y = sum_t w_t vs_t c_t / sum_t w_t,   w_t = exp(scale * ks_t (q . c_t) - m),
// m the running maximum: one pass over keys and values, sums and statistics in F32, exponents in base 2. The scales
// stand outside both sums over a token's values: ks_t multiplies a score, vs_t a weight, and the products run
// on the codes alone, which v_cvt_scalef32_pk_f16_fp8 takes to F16 exactly, two an instruction.
//
// Workgroups, steps of 32 tokens, the 16 columns of 8 query heads in two F16 parts and the join are those of the F16
// cache's kernels. What differs:
//
// Rows. A lane's part of a K row is one run of bytes (piece G * D32 + d of 8 values in place of d * 4 + G: the sum over a
// row's values has no order), so that 16-byte loads fetch it; q is taken in the same order.
//
// What bounds it: reading codes (2 * width bytes per token and head, and 8 / block_tokens of scales). 32 sequences of 32768
// tokens x 8 heads 335 us, 6.4 TB/s, what a kernel that only reads reaches; below, a launch's chains of latencies (some 6 us), the
// beginnings of rows and the join's launch (4.5) stand beside it: 1 x 32768 15.7 us and 4.3 (the codes alone 10.2), 64 ragged
// to 2048 x 8 heads 39 (21). A second step's rows on their way changed nothing that paid: 335 -> 346, 39 -> 45 us.
//
// Weights. w_t vs_t has the scales' range, not that of [0, 1]: it is multiplied by a power of two (`lift`) that takes the
// largest one so far to [2^13, 2^14) before it is split into F16 parts, and the sums move along when that one grows, as
// they do with m. So a weight times its scale is held to 2^-22 of itself, 2^-38 of the largest or 2^-149, whichever is most: the
// low part ends at half of F16's least number, 2^-25 beside a largest of 2^13, and the power at 2^126.
#include "attention_common.h"
#include "launch.h"

#include <algorithm>
#include <type_traits>

namespace {

typedef uint32_t uint4a8 __attribute__((ext_vector_type(4), aligned(8)));   // rows begin on 8 bytes

constexpr int kWideWaves = 8;
constexpr int kMinChunk = kWaves * kStep;
constexpr int kMaxChunk = 512, kMaxChunkMany = 1024;
constexpr int kMostChunks = 65535;       // the grid's limit
constexpr int64_t kMostIds = 8000;       // page ids of a chunk in LDS, 32 KB
constexpr int kRowSteps = 2;             // what beginning a row counts in a share (64 ragged to 2048 x 8 38.7 us, 1: 41.1, 3: 38.6)
constexpr int kMostEven = 1024;          // sequences whose lengths a workgroup of attend_even_f8 goes through
constexpr int kLift = 13;                // exponent of the largest weight times its scale, as F16 parts
constexpr int kMostLift = 126;           // of the power that takes it there, whose reciprocal is a normal number too

struct AttendF8Args : AttendArgs {
    const float *k_scales, *v_scales;
    int blocks, block_log2;              // scales of a page and head; tokens of one are 2^block_log2
};

// How a lane finds the scales of its four neighbouring tokens: one for sixteen tokens or more, through the scalar cache;
// one for the four; one for each.
enum Scales { kSixteen, kFour, kEach };

// Two of a word's four codes in F16.
template <bool HIGH>
__device__ __forceinline__ uint32_t two_values(uint32_t codes) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, HIGH));
}
__device__ __forceinline__ half8 eight_values(uint2v codes) {
    const uint4v x{two_values<false>(codes[0]), two_values<true>(codes[0]), two_values<false>(codes[1]),
                   two_values<true>(codes[1])};
    return __builtin_bit_cast(half8, x);
}

// A step's scores to weights times their scales, in two parts as the second product's columns; maxima and sums so far
// move along. there(i): whether the lane's token i counts, asked where `masked`.
template <int VW, int NT, typename There>
__device__ __forceinline__ void weigh(const float4v (&scores)[NT][2], const float (&undo)[NT], const float (&ks)[8],
                                      float (&vs)[8], bool masked, There there, int c, float (&m)[NT], float (&l)[NT],
                                      float (&most)[NT], float (&lift)[NT], float4v (&acc)[NT][VW], half8 (&pf)[NT]) {
    if (masked) {                                    // what stands in a masked place may be anything
#pragma unroll
        for (int i = 0; i < 8; ++i) vs[i] = there(i) ? vs[i] : 0.0f;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float sc[8], p[8], top = -INFINITY, heaviest = 0.0f;
        // a factor above 1 (queries of a thousand and more) comes after the scale: no partial product is infinite where the
        // score is not, nor rounded to nothing but where that is next to nothing of a score
        whole_scores(scores[nt], fminf(undo[nt], 1.0f), c, sc);
        const float more = fmaxf(undo[nt], 1.0f);
#pragma unroll
        for (int i = 0; i < 8; ++i) sc[i] = sc[i] * ks[i] * more;
        if (masked) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sc[i] = there(i) ? sc[i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, sc[i]);
        top = fmaxf(m[nt], across_groups_max(top));
        const float from = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i] = __builtin_amdgcn_exp2f(sc[i] - from);
            sum += p[i];
            p[i] *= vs[i];
            heaviest = fmaxf(heaviest, fabsf(p[i]));
        }
        heaviest = across_groups_max(heaviest);
        if (__any(top > m[nt] || heaviest > most[nt])) {
            const float alpha = top > m[nt] ? __builtin_amdgcn_exp2f(m[nt] - top) : 1.0f;   // 0 from no token yet
            l[nt] *= alpha;
            m[nt] = top;
            most[nt] = fmaxf(most[nt] * alpha, heaviest);
            const int from_e = exponent_of(lift[nt]), to_e = min(kLift - exponent_of(most[nt]), kMostLift);
            const float change = ldexpf(alpha, to_e - from_e);
            lift[nt] = ldexpf(1.0f, to_e);
#pragma unroll
            for (int j = 0; j < VW; ++j) acc[nt][j] *= change;
        }
        l[nt] += sum;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = p[i] * lift[nt];
            const _Float16 high = static_cast<_Float16>(x);
            pf[nt][i] = c < 8 ? high : static_cast<_Float16>(x - static_cast<float>(high));
        }
    }
}

// The second product, four values of a lane's eight tokens at a time.
template <int VW, int NT>
__device__ __forceinline__ void add_codes(const uint32_t (&vr)[8][VW / 4], const half8 (&pf)[NT], float4v (&acc)[NT][VW]) {
#pragma unroll
    for (int w = 0; w < VW / 4; ++w) {
        uint32_t x[8][2];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i][0] = two_values<false>(vr[i][w]);
            x[i][1] = two_values<true>(vr[i][w]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            union { uint32_t u[4]; half8 h; } vf;
            const uint32_t pick = j & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
            for (int u = 0; u < 4; ++u) vf.u[u] = __builtin_amdgcn_perm(x[2 * u + 1][j / 2], x[2 * u][j / 2], pick);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                acc[nt][w * 4 + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf.h, pf[nt], acc[nt][w * 4 + j], 0, 0, 0);
        }
    }
}

// Where the two halves of a step stand: each in one page.
struct Halves {
    int64_t at[2], scales[2];            // of the rows; of the page's scales of the head
    int within[2];                       // the half's first token in its page
    bool ok[2];
};
__device__ __forceinline__ Halves find_halves(const AttendF8Args &a, const int *row, int kvh, int t0, int lo, int hi, int lane) {
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
        w.within[half] = t - p * a.pool.page_tokens;
        w.at[half] = (int64_t)id * a.pool.page_stride + (int64_t)w.within[half] * a.pool.token_stride;
        w.scales[half] = ((int64_t)id * a.pool.heads + kvh) * a.blocks;
    }
    return w;
}

// The scales of a lane's tokens: four of each half of a step.
template <Scales S>
struct TokenScales {
    static constexpr int kOf = S == kEach ? 8 : 2;
    float k[kOf], v[kOf];
    __device__ __forceinline__ void load(const AttendF8Args &a, const Halves &w, int G) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const float *ks = a.k_scales + w.scales[half], *vs = a.v_scales + w.scales[half];
            if constexpr (S == kSixteen) {
                k[half] = scalar_load(ks + (w.within[half] >> a.block_log2));
                v[half] = scalar_load(vs + (w.within[half] >> a.block_log2));
            } else {
#pragma unroll
                for (int i = 0; i < kOf / 2; ++i) {
                    const int at = (w.within[half] + G * 4 + i) >> a.block_log2;
                    k[half * (kOf / 2) + i] = ks[at];
                    v[half * (kOf / 2) + i] = vs[at];
                }
            }
        }
    }
    __device__ __forceinline__ void spread(float (&ks)[8], float (&vs)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) ks[i] = k[i * kOf / 8], vs[i] = v[i * kOf / 8];
    }
};

// A lane's part of a K row: D32 pieces of 8 codes on end, `pieces` of them within the width.
template <int D32, bool FULL, bool ONCE>
__device__ __forceinline__ void load_key(const uint8_t *p, int first, int pieces, uint2v (&k)[D32]) {
    if constexpr (FULL) {
        p += first * 8;
#pragma unroll
        for (int d = 0; d + 1 < D32; d += 2) {
            const uint4a8 x = load_row<uint4a8, ONCE>(p + d * 8);
            k[d] = uint2v{x[0], x[1]};
            k[d + 1] = uint2v{x[2], x[3]};
        }
        if constexpr (D32 % 2) k[D32 - 1] = load_row<uint2v, ONCE>(p + (D32 - 1) * 8);
    } else {
#pragma unroll
        for (int d = 0; d < D32; ++d) {
            const bool in = first + d < pieces;
            const uint2v x = load_row<uint2v, ONCE>(p + (in ? (first + d) * 8 : 0));
            k[d] = in ? x : uint2v{0, 0};
        }
    }
}
// A lane's part of a V row: VW codes from column c * VW on. A column past the width gives values that are not stored: any
// part of the row will do.
template <int VW, bool FULL, bool ONCE>
__device__ __forceinline__ void load_value(const uint8_t *p, int c, int width, uint32_t (&v)[VW / 4]) {
    const int col = c * VW;
    if constexpr (VW == 4) {
        v[0] = load_row<uint32_t, ONCE>(p + (col < width ? col : 0));
    } else if constexpr (VW == 8) {
        const uint2v x = load_row<uint2v, ONCE>(p + (col < width ? col : 0));
        v[0] = x[0], v[1] = x[1];
    } else if constexpr (FULL) {
        const uint4a8 x = load_row<uint4a8, ONCE>(p + (col < width ? col : 0));
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = x[u];
    } else {
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            const uint2v x = load_row<uint2v, ONCE>(p + (col + part * 8 < width ? col + part * 8 : 0));
            v[part * 2] = x[0], v[part * 2 + 1] = x[1];
        }
    }
}

// D32: 32-value pieces of a head (width <= 32 * D32; FULL: equal). VW: values a lane loads of a V row (16 lanes: width
// <= 16 * VW). NT: column tiles (8 query heads each). UNI: page_tokens % 16 == 0, so that a half step of 16 tokens lies in
// one page: its address is scalar, its page id a scalar load. Otherwise the chunk's page ids wait in LDS and each
// lane finds its rows and their scales there.
template <int D32, int VW, int NT, bool UNI, bool FULL, bool ONCE, Scales S, int WAVES>
__global__ __launch_bounds__(WAVES * kWave) void attend_f8(AttendF8Args a) {
    static_assert(UNI || S == kEach, "rows that are looked up one by one bring their scales");
    constexpr int DPad = 16 * VW;
    constexpr int kGroup = WAVES * kWave;
    extern __shared__ float lds[];
    const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int c = lane & 15, G = lane >> 4;
    const Part part = part_of(a);
    const int s = part.s, chunk = part.chunk, kvh = part.kvh, tile = part.tile;
    const int head0 = kvh * a.group + tile * 8 * NT;                        // first query head
    const int heads = min(8 * NT, a.group - tile * 8 * NT);
    const int width = FULL ? 32 * D32 : a.pool.width, pieces = width / 8;
    auto in = [&](int d) { return FULL || G * D32 + d < pieces; };

    // a part past the sequence's end, before it asks for anything
    if (chunk > 0 && a.window == 0 && chunk * a.chunk >= scalar_load(a.lengths + s)) return;
    // the queries' values are on their way while the sequence's length and pages are read
    float4v q[NT][D32][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int h = nt * 8 + (c & 7);
        const int64_t q_row = s * a.q_stride + (int64_t)(head0 + (h < heads ? h : 0)) * width;
#pragma unroll
        for (int d = 0; d < D32; ++d) load_query(a, q_row + (in(d) ? (G * D32 + d) * 8 : 0), q[nt][d]);
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

    const uint8_t *k_head = static_cast<const uint8_t *>(a.k) + (int64_t)kvh * a.pool.head_stride;
    const uint8_t *v_head = static_cast<const uint8_t *>(a.v) + (int64_t)kvh * a.pool.head_stride;

    // the registers of a step: its rows' codes as loaded, and their scales
    uint2v kr[2][D32];
    uint32_t vr[8][VW / 4];
    TokenScales<S> scales;
    // !UNI: the page, and the token in it, of token t, moved into the chunk
    struct Place {
        int id, within;
    };
    auto place_of = [&](int t) {
        t = min(max(t, lo), hi);
        const int p = a.pool.per_page.div(t);
        return Place{max(page_ids[p - page0], 0), t - p * a.pool.page_tokens};
    };
    auto row_of = [&](int t) {
        const Place x = place_of(t);
        return (int64_t)x.id * a.pool.page_stride + (int64_t)x.within * a.pool.token_stride;
    };
    // a lane's token of V register i, which is also the token of its score i
    auto token_of = [&](int t0, int i) { return t0 + (i < 4 ? 0 : 16) + G * 4 + (i & 3); };
    const uint32_t k_lane = static_cast<uint32_t>(c * a.pool.token_stride);
    const uint32_t v_lane = static_cast<uint32_t>(G * 4 * a.pool.token_stride);
    auto load_k = [&](int t0, const Halves &w) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
            load_key<D32, FULL, ONCE>(k_head + (UNI ? w.at[half] + k_lane : row_of(t0 + half * 16 + c)), G * D32, pieces,
                                      kr[half]);
    };
    auto load_v = [&](int t0, const Halves &w) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            load_value<VW, FULL, ONCE>(v_head + (UNI ? w.at[i / 4] + (i & 3) * a.pool.token_stride + v_lane
                                                     : row_of(token_of(t0, i))), c, width, vr[i]);
    };
    auto load_scales = [&](int t0, const Halves &w) {
        if constexpr (UNI) {
            scales.load(a, w, G);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const Place x = place_of(token_of(t0, i));
                const int64_t at = ((int64_t)x.id * a.pool.heads + kvh) * a.blocks + (x.within >> a.block_log2);
                scales.k[i] = a.k_scales[at];
                scales.v[i] = a.v_scales[at];
            }
        }
    };

    int t0 = begin + wave * kStep;
    Halves here{};
    half8 qf[NT][D32];
    float undo[NT];
    float4v acc[NT][VW];
    float m[NT], l[NT], most[NT], lift[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt] = -INFINITY;
        l[nt] = most[nt] = 0.0f;
        lift[nt] = 1.0f;
#pragma unroll
        for (int j = 0; j < VW; ++j) acc[nt][j] = float4v{0, 0, 0, 0};
    }

    // A step, with the loads of the next one or without. All loads stand in straight lines: where ways with and without
    // them meet, a wait for older loads has to wait for these too. (With that, and the first V rows asked for after the
    // queries are in parts, 200 ragged to 700 x 8 heads 46.5 -> 43 us, 64 to 1024 25.9 -> 23.5, 8 to 4096 19.6 -> 17.7.)
    auto step = [&](auto more) {
        constexpr bool kMore = decltype(more)::value;
        const int t1 = t0 + WAVES * kStep;
        Halves next{};
        if constexpr (UNI && kMore) next = find_halves(a, row, kvh, t1, lo, hi, lane);
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
        for (int nt = 0; nt < NT; ++nt) scores[nt][0] = scores[nt][1] = float4v{0, 0, 0, 0};
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int d = 0; d < D32; ++d) {
                const half8 kf = eight_values(kr[half][d]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    scores[nt][half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[nt][d], scores[nt][half], 0, 0, 0);
            }
        float ks[8], vs[8];
        scales.spread(ks, vs);
        // the next step's K rows are on their way during the weights and the second product, its V rows
        // during the next scores
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (kMore) {
            load_k(t1, next);
            load_scales(t1, next);
        }
        __builtin_amdgcn_sched_barrier(0);

        half8 pf[NT];
        weigh<VW, NT>(scores, undo, ks, vs, masked, there, c, m, l, most, lift, acc, pf);
        if (masked) {                                // 0 * NaN would reach the sums
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool ok = there(i);
#pragma unroll
                for (int u = 0; u < VW / 4; ++u) vr[i][u] = ok ? vr[i][u] : 0;
            }
        }
        add_codes<VW, NT>(vr, pf, acc);
        if constexpr (kMore) {
            __builtin_amdgcn_sched_barrier(0);
            load_v(t1, next);
            __builtin_amdgcn_sched_barrier(0);
            t0 = t1;
            here = next;
        }
    };
    if (t0 < end) {
        if constexpr (UNI) here = find_halves(a, row, kvh, t0, lo, hi, lane);
        load_k(t0, here);
        load_scales(t0, here);
        __builtin_amdgcn_sched_barrier(0);
        split_queries<D32, NT>(a.f16, a.scale_log2, heads, c, in, q, qf, undo);
        __builtin_amdgcn_sched_barrier(0);
        load_v(t0, here);
        __builtin_amdgcn_sched_barrier(0);
        while (t0 + WAVES * kStep < end) step(std::true_type());
        step(std::false_type());
    }
    if constexpr (!UNI) __syncthreads();             // page_ids are read; the sums go over them

    // the waves' sums side by side, then one sum per value
    float *wave_ml = lds, *wave_o = lds + WAVES * NT * 8 * 2;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const float total = across_groups_sum(l[nt]), lower = ldexpf(1.0f, -exponent_of(lift[nt]));
        const int h = nt * 8 + c;
        const bool mine = c < 8 && h < heads;
        if (mine && G == 0) {
            wave_ml[(wave * NT * 8 + h) * 2] = m[nt];
            wave_ml[(wave * NT * 8 + h) * 2 + 1] = total;
        }
        // row 4G + r of product j is value VW * (4G + r) + j
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < VW; j += 4) {
                float4v v;
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = both_parts(acc[nt][j + u][r]) * lower;
                if (mine) *reinterpret_cast<float4v *>(wave_o + (wave * heads + h) * DPad + (4 * G + r) * VW + j) = v;
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

// The same sums in equal shares of the steps of all rows, one or two workgroups to a CU (attend_even's scheme): four waves take
// four neighbouring key-value heads, a wave's sums are its head's.
template <int D32, int VW, Scales S>
__global__ __launch_bounds__(kThreads) void attend_even_f8(AttendF8Args a) {
    constexpr int width = 32 * D32;
    const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int c = lane & 15, G = lane >> 4;
    const int fours = a.pool.heads / kWaves, heads = a.group;
    const Share share = share_of<kRowSteps>(a, blockIdx.x, fours, lane,
                                            [&](int s) { return lane_length(a, s, blockIdx.x == 0 && wave == 0); });
    if (share.left == 0 || share.step + share.left <= kRowSteps) return;     // (or ends among a row's empty steps)

    // what a share has of one row
    struct Run {
        int s, four, step, steps, take;              // the row's steps, and this run's from `step` on, empty ones included
        int lo, hi, t0;                              // its tokens, and the first of its first step
    };
    auto run_at = [&](int s, int four, int step, int left) {
        Run r;
        const int len = length_of(a, s, false), base = base_of(a, len);
        r.s = s;
        r.four = four;
        r.step = step;
        r.steps = (len - base + kStep - 1) / kStep + kRowSteps;
        r.take = min(left, r.steps - step);
        r.t0 = base + max(0, step - kRowSteps) * kStep;
        r.lo = max(r.t0, a.window > 0 ? len - a.window : 0);
        r.hi = min(len, base + (step + r.take - kRowSteps) * kStep) - 1;
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
    auto find = [&](const Run &r, int t0) {
        Halves w = find_halves(a, a.table + (int64_t)r.s * a.row_pages, r.four * kWaves + wave, t0, r.lo, r.hi, lane);
#pragma unroll
        for (int half = 0; half < 2; ++half) w.at[half] += (int64_t)(r.four * kWaves + wave) * a.pool.head_stride;
        return w;
    };

    uint2v kr[2][D32];
    uint32_t vr[8][VW / 4];
    TokenScales<S> scales;
    const uint32_t k_lane = static_cast<uint32_t>(c * a.pool.token_stride);
    const uint32_t v_lane = static_cast<uint32_t>(G * 4 * a.pool.token_stride);
    auto load_k = [&](const Halves &w) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
            load_key<D32, true, true>(static_cast<const uint8_t *>(a.k) + w.at[half] + k_lane, G * D32, width / 8, kr[half]);
    };
    auto load_v = [&](const Halves &w) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            load_value<VW, true, true>(static_cast<const uint8_t *>(a.v) + w.at[i / 4] + (i & 3) * a.pool.token_stride + v_lane,
                                       c, width, vr[i]);
    };
    float4v q[1][D32][2];
    auto load_queries = [&](const Run &r) {
        const int64_t at = r.s * a.q_stride + (int64_t)((r.four * kWaves + wave) * a.group + (c & 7) % heads) * width;
#pragma unroll
        for (int d = 0; d < D32; ++d) load_query(a, at + (G * D32 + d) * 8, q[0][d]);
    };

    Run now = run_at(share.s, share.four, share.step, share.left);
    load_queries(now);
    Halves here = find(now, now.t0);
    load_k(here);
    scales.load(a, here, G);
    load_v(here);
    __builtin_amdgcn_sched_barrier(0);
    half8 qf[1][D32];
    float undo[1], m[1], l[1], most[1], lift[1];
    float4v acc[1][VW];
    auto start = [&] {
        split_queries<D32, 1>(a.f16, a.scale_log2, heads, c, [](int) { return true; }, q, qf, undo);
        m[0] = -INFINITY;
        l[0] = most[0] = 0.0f;
        lift[0] = 1.0f;
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
        const bool masked = t0 < now.lo || t0 + kStep > now.hi + 1 || !(here.ok[0] && here.ok[1]);
        auto there = [&](int i) {
            const int t = t0 + (i < 4 ? 0 : 16) + G * 4 + (i & 3);
            return t >= now.lo && t <= now.hi && here.ok[i / 4];
        };
        float4v scores[1][2] = {{float4v{0, 0, 0, 0}, float4v{0, 0, 0, 0}}};
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int d = 0; d < D32; ++d)
                scores[0][half] =
                    __builtin_amdgcn_mfma_f32_16x16x32_f16(eight_values(kr[half][d]), qf[0][d], scores[0][half], 0, 0, 0);
        float ks[8], vs[8];
        scales.spread(ks, vs);
        __builtin_amdgcn_sched_barrier(0);
        if (more) {
            load_k(next);
            scales.load(a, next, G);
        }
        if (last && more) load_queries(then);
        __builtin_amdgcn_sched_barrier(0);
        half8 pf[1];
        weigh<VW, 1>(scores, undo, ks, vs, masked, there, c, m, l, most, lift, acc, pf);
        if (masked) {                                // 0 * NaN would reach the sums
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool ok = there(i);
#pragma unroll
                for (int u = 0; u < VW / 4; ++u) vr[i][u] = ok ? vr[i][u] : 0;
            }
        }
        add_codes<VW, 1>(vr, pf, acc);
        __builtin_amdgcn_sched_barrier(0);
        if (more) load_v(next);
        __builtin_amdgcn_sched_barrier(0);
        if (last) {
            // sums to the output, or to place (workgroup + row): consecutive for the workgroups of one row
            const int row = now.s * fours + now.four, slot = blockIdx.x + row, head0 = (now.four * kWaves + wave) * a.group;
            const bool single = now.step <= kRowSteps && now.step + now.take == now.steps;
            if (now.step <= kRowSteps && tid == 0)
                a.spans[row] = int2{slot, share.holder(run_from - now.step + now.steps - 1) - static_cast<int>(blockIdx.x) + 1};
            const float total = across_groups_sum(l[0]), lower = ldexpf(1.0f, -exponent_of(lift[0]));
            const int64_t at = ((int64_t)slot * kWaves + wave) * a.group + c;
            const bool mine = c < heads;
            if (mine && G == 0 && !single) {
                a.part_ml[at * 2] = m[0];
                a.part_ml[at * 2 + 1] = total;
            }
            // row 4G + r of product j is value VW * (4G + r) + j
#pragma unroll
            for (int j = 0; j < VW; j += 4)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = (4 * G + r) * VW + j;
                    float4v v;
#pragma unroll
                    for (int u = 0; u < 4; ++u) v[u] = both_parts(acc[0][j + u][r]) * lower;
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

// Whether the 16 tokens of a half step are in one page; lane offsets within them are 32-bit.
bool in_halves(const kunlun::KVCacheLayout &c) { return c.page_tokens % 16 == 0 && c.token_stride < (1 << 26); }

struct Plan {
    int group, nt, tiles, chunk, chunks;
    bool halves, once, wide, narrow;
    int shares;                                      // attend_even_f8: workgroups, else 0
};

Plan plan_of(const kunlun::KVCacheLayout &c, const kunlun::PagedAttentionLayout &p, int cus) {
    Plan r;
    r.halves = in_halves(c);
    r.group = p.query_heads / c.heads;
    r.nt = r.group > 8 && c.width <= 128 ? 2 : 1;
    r.tiles = (r.group + 8 * r.nt - 1) / (8 * r.nt);
    const int longest = p.window > 0 ? std::min<int64_t>(p.longest, (int64_t)p.window + kStep - 1) : p.longest;
    const int64_t rows = (int64_t)p.sequences * c.heads * r.tiles;
    // The rules are the F16 cache's (rows whole on eight waves or four, parts of one size, equal shares), whose chains of
    // latencies they balance. Both sides of each for this cache, of one build (us a call; heads of 128, ragged where not full):
    // - eight waves to a whole row / parts: 8, 16 and 32 x 512 tokens x 8 heads 9.0 / 10.4, 9.3 / 11.9 and 9.6 / 13.6; 32 x 768
    //   11.3 / 15.4, 32 x 1024 13.1 / 17.1; 8 x 1024 12.3 / 12.0, windows of 1000 in 7 x 5 heads of 80 16.9 / 13.7. Fewer rows
    //   of 768 are parted, though 16 x 768 x 8 would take 11.3 whole and takes 13.6.
    // - four waves to a whole row / equal shares: 64 x 1024 x 8 23.0 / 26.6, full 26.3 / 34.5; 200 x 700 x 8 41.0 / 47.0 (on
    //   eight waves 55.8); token by token 49.2 / 47.3, 200 x 1000 67.4 / 59.2; 300 x 500 x 4 heads of 256 53.9 / 55.0.
    // - parts of 256, 512 and 1024 tokens: 1 x 32768 x 8 22.1, 20.1 and 19.6; 64 x 2048 x 2 in 512, 1024 and whole 16.7, 19.0 and
    //   23.8; 128 x 3000 x 5 in 512, 1024 and 1536 63.0, 60.3 and 59.7; 48 full rows of 544 x 8 whole 14.8, in 256 20.1.
    // - parts / equal shares: 64 x 2048 x 8 48.9 / 38.7; 32 x 4096 x 32 106.0 / 102.2; 64 x 2048 x 4 of 256 52.3 / 43.5.
    // - the non-temporal hint (`once`), without / with: 200 x 700 x 8 42.0 / 40.5; 96 x 900 x 8, whose 92 MB the 256 MiB
    //   cache holds from call to call, 25.3 / 26.3.
    const int whole = kMaxChunk + kStep;             // a window starts up to kStep - 1 tokens early
    r.wide = r.nt == 1 && c.width <= 128 && rows <= cus && longest > kMinChunk &&
             longest <= (rows > cus / 2 ? 2 * whole : whole);
    const int64_t least = r.wide ? longest : rows > cus && longest <= whole ? longest : kMinChunk;
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
    // One wave to a workgroup for many rows of up to four steps, or eight where the rows are very many or four waves' registers
    // leave a CU to one workgroup (us on four waves and on one, 250 tokens ragged: 512 sequences x 8 heads 46.6 / 44.5, of 120
    // tokens 36.3 / 25.8; 300 x 4 heads of 256 33.7 / 26.9; but 300 x 8 of 64 18.7 / 20.9, and 80 x 8, full rows, 14.0 / 15.3)
    const bool eight = c.width > 128 || (c.width > 64 && rows > 8 * cus);
    r.narrow = r.nt == 1 && rows > 2 * cus && longest <= (eight ? 8 : 4) * kStep;
    r.once = r.tiles == 1 && (int64_t)p.sequences * longest * c.heads * c.width * 2 > (64 << 20);
    const bool together = c.head_stride < c.token_stride;
    const bool share_whole = !r.wide && (c.width > 128 ? longest > kMaxChunk : together && longest > 6 * kMinChunk);
    r.shares = 0;
    if ((r.chunks > 1 || share_whole) && r.halves && r.once && r.nt == 1 && c.heads % kWaves == 0 &&
        (c.width % 64 == 0 || c.width == 96) && p.sequences <= kMostEven &&
        (p.sequences > 1 || (int64_t)longest * c.heads * c.width * 2 > (256 << 20)) &&
        (int64_t)p.sequences * c.heads * (longest / kStep + 3) < INT32_MAX)
        // two workgroups to a CU, whose registers allow it up to width 128 (64 sequences ragged to 2048 x 8 heads of 128 38.7 us
        // a call, one 48.3, three 48.6; 32 x 32768 347, 417 and 373; 4 heads of 256 one 43.5, two 49.4)
        r.shares = c.width <= 128 ? 2 * cus : cus;
    return r;
}

template <int D32, int VW, int NT, bool UNI, bool FULL, bool ONCE, Scales S, int WAVES>
hipError_t launch(const AttendF8Args &a, const Plan &p, int sequences, int heads, hipStream_t stream) {
    const size_t ids = UNI ? 0 : (p.chunk / a.pool.page_tokens + 2) * sizeof(int);
    const size_t sums = (size_t)WAVES * (NT * 8 * 2 + std::min(p.group, 8 * NT) * 16 * VW) * sizeof(float);
    const size_t lds = std::max(ids, sums);          // up to 33 KiB
    hipLaunchKernelGGL((attend_f8<D32, VW, NT, UNI, FULL, ONCE, S, WAVES>), dim3(heads * p.tiles, sequences, p.chunks),
                       dim3(WAVES * kWave), lds, stream, a);
    return hipGetLastError();
}

template <int D32, int VW, int NT, int WAVES>
hipError_t launch_tiles(const AttendF8Args &a, const Plan &p, int sequences, int heads, hipStream_t stream) {
    if (!p.halves) return launch<D32, VW, NT, false, false, false, kEach, WAVES>(a, p, sequences, heads, stream);
    if (a.pool.width != 32 * D32) return launch<D32, VW, NT, true, false, false, kEach, WAVES>(a, p, sequences, heads, stream);
    if constexpr (WAVES == kWaves) {
        if (p.once) {
            if (a.block_log2 >= 4) return launch<D32, VW, NT, true, true, true, kSixteen, WAVES>(a, p, sequences, heads, stream);
            if (a.block_log2 >= 2) return launch<D32, VW, NT, true, true, true, kFour, WAVES>(a, p, sequences, heads, stream);
            return launch<D32, VW, NT, true, true, true, kEach, WAVES>(a, p, sequences, heads, stream);
        }
    }
    if (a.block_log2 >= 4) return launch<D32, VW, NT, true, true, false, kSixteen, WAVES>(a, p, sequences, heads, stream);
    if (a.block_log2 >= 2) return launch<D32, VW, NT, true, true, false, kFour, WAVES>(a, p, sequences, heads, stream);
    return launch<D32, VW, NT, true, true, false, kEach, WAVES>(a, p, sequences, heads, stream);
}

template <int D32, int VW>
hipError_t launch_width(const AttendF8Args &a, const Plan &p, int sequences, int heads, hipStream_t stream) {
    if (p.shares) {                                  // before any other choice: the join reads what only this kernel writes
        if (a.pool.width != 32 * D32 || !p.halves || p.nt != 1) return hipErrorInvalidValue;
        const dim3 grid(p.shares), threads(kThreads);
        if (a.block_log2 >= 4) hipLaunchKernelGGL((attend_even_f8<D32, VW, kSixteen>), grid, threads, 0, stream, a);
        else if (a.block_log2 >= 2) hipLaunchKernelGGL((attend_even_f8<D32, VW, kFour>), grid, threads, 0, stream, a);
        else hipLaunchKernelGGL((attend_even_f8<D32, VW, kEach>), grid, threads, 0, stream, a);
        return hipGetLastError();
    }
    if (p.narrow) return launch_tiles<D32, VW, 1, 1>(a, p, sequences, heads, stream);
    if constexpr (VW <= 8) {
        if (p.nt == 2) return launch_tiles<D32, VW, 2, kWaves>(a, p, sequences, heads, stream);
        if (p.wide) return launch_tiles<D32, VW, 1, kWideWaves>(a, p, sequences, heads, stream);
    }
    return launch_tiles<D32, VW, 1, kWaves>(a, p, sequences, heads, stream);
}

// Places of attend_even_f8's sums: every workgroup begins one and every row, for each of its four heads' query heads.
size_t even_parts(const kunlun::KVCacheLayout &c, const kunlun::PagedAttentionLayout &p, const Plan &r) {
    return ((size_t)p.sequences * (c.heads / kWaves) + r.shares) * kWaves * r.group;
}

} // namespace

extern "C" size_t kk_paged_attention_f8_workspace_bytes(const kunlun::KVCacheLayout &c, const kunlun::PagedAttentionLayout &p,
                                                        int cus) {
    const Plan r = plan_of(c, p, cus);
    if (r.shares)
        return even_parts(c, p, r) * (c.width + 2) * sizeof(float) + (size_t)p.sequences * (c.heads / kWaves) * sizeof(int2);
    return r.chunks == 1 ? 0 : (size_t)p.sequences * p.query_heads * r.chunks * (c.width + 2) * sizeof(float);
}

extern "C" const char *kk_paged_attention_f8_route(const kunlun::KVCacheLayout &c, const kunlun::PagedAttentionLayout &p,
                                                   int cus) {
    const Plan r = plan_of(c, p, cus);
    return r.shares ? "paged_attention_f8_even" : r.chunks > 1 ? "paged_attention_f8_split" : "paged_attention_f8";
}

extern "C" int kk_paged_attention_f8(void *y, const void *q, const void *k, const void *v, const float *k_scales,
                                     const float *v_scales, const int *table, const int *lengths,
                                     const kunlun::KVCacheF8Layout &f8, const kunlun::PagedAttentionLayout &p, void *workspace,
                                     int *status, int cus, hipStream_t stream) {
    const kunlun::KVCacheLayout &c = f8.cache;
    const Plan r = plan_of(c, p, cus);
    if (c.width <= 0 || c.width > 256 || c.width % 8 || p.sequences > 65535 || r.chunks > kMostChunks ||
        f8.block_tokens <= 0 || ((r.chunks > 1 || r.shares) && !workspace))
        return hipErrorInvalidValue;
    AttendF8Args a;
    a.k = k;
    a.v = v;
    a.k_scales = k_scales;
    a.v_scales = v_scales;
    a.blocks = c.page_tokens / f8.block_tokens;
    a.block_log2 = __builtin_ctz(f8.block_tokens);
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
    const AttendArgs &joined = a;
    if (r.shares && little) hipLaunchKernelGGL((join_chunks<kWave, true>), grid, dim3(kWave), 0, stream, joined);
    else if (r.shares) hipLaunchKernelGGL((join_chunks<kThreads, true>), grid, dim3(kThreads), 0, stream, joined);
    else if (little) hipLaunchKernelGGL((join_chunks<kWave, false>), grid, dim3(kWave), 0, stream, joined);
    else hipLaunchKernelGGL((join_chunks<kThreads, false>), grid, dim3(kThreads), 0, stream, joined);
    return hipGetLastError();
}
