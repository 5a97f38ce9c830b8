// New tokens into a paged F16 key-value cache, their queries and keys turned by
// their position's angles on the way:
//   (a, b) -> (a cos - b sin, a sin + b cos)
// for pairs of a head's first `rotary` values, in F32, rounded once where it is
// stored as F16 (both products of a sum are rounded with it, by one fma). One launch
// reads the product's rows and writes q and both pools: bound by those bytes.
//
// A thread takes 8 values of one head of one token: 8 consecutive ones, or, of a
// head rotated in halves, 4 of the first half and their 4 partners. Where rows,
// strides or the tables' halves are off 4 values, every value is taken by itself.
#include "device_common.h"
#include "launch.h"
#include "paged.h"

namespace {

using kk::PoolView;

constexpr int kThreads = 256;

struct AppendArgs {
    _Float16 *k_pool, *v_pool;
    void *q_out;
    const void *q, *k, *v;
    const int *sequence, *position, *lengths, *table;
    const float *cosine, *sine;
    int *status;
    PoolView pool;
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    kk::FastDiv units_per_token, units_per_head;
    int tokens, sequences, row_pages, query_heads, rotary, positions;
    uint32_t units;                              // tokens x units of a token
};

template <typename T, int N>
struct alignas(N * sizeof(T)) Pack {
    T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_values(const T *from, float (&out)[8], int at) {
    const Pack<T, N> p = *reinterpret_cast<const Pack<T, N> *>(from);
#pragma unroll
    for (int i = 0; i < N; ++i) out[at + i] = static_cast<float>(p.v[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_values(T *to, const float (&x)[8], int at) {
    Pack<T, N> p;
#pragma unroll
    for (int i = 0; i < N; ++i) p.v[i] = static_cast<T>(x[at + i]);
    *reinterpret_cast<Pack<T, N> *>(to) = p;
}

template <typename T, bool HALVES, bool VEC>
__global__ __launch_bounds__(kThreads) void append(AppendArgs a) {
    const uint32_t unit = blockIdx.x * kThreads + threadIdx.x;
    if (unit >= a.units) return;
    const int token = a.units_per_token.div(unit);
    const int in_token = unit - token * a.units_per_token.d;
    const int head = a.units_per_head.div(in_token);
    const int u = in_token - head * a.units_per_head.d;      // which 8 values of the head

    const int s = a.sequence ? a.sequence[token] : token;
    if (s < 0) return;
    if (s >= a.sequences) {
        if (in_token == 0) kk::report(a.status, kk::kBadIndex);
        return;
    }
    const int pos = a.position ? a.position[token] : a.lengths[s] - 1;
    if (pos < 0) return;
    const int page_at = a.pool.per_page.div(pos);
    if (page_at >= a.row_pages || (a.rotary > 0 && pos >= a.positions)) {
        if (in_token == 0) kk::report(a.status, kk::kBadIndex);
        return;
    }
    const bool is_q = head < a.query_heads;
    const bool is_k = !is_q && head < a.query_heads + a.pool.heads;
    const int h = is_q ? head : head - a.query_heads - (is_k ? 0 : a.pool.heads);
    const T *from = (is_q ? static_cast<const T *>(a.q) + token * a.q_stride
                          : is_k ? static_cast<const T *>(a.k) + token * a.k_stride
                                 : static_cast<const T *>(a.v) + token * a.v_stride) + h * a.pool.width;
    // a token without a page is left out whole, its query too
    const int page = a.table[(int64_t)s * a.row_pages + page_at];
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.pool.pages)) {
        if (in_token == 0) kk::report(a.status, kk::kBadPage);
        return;
    }
    _Float16 *to = (is_k ? a.k_pool : a.v_pool) + page * a.pool.page_stride + h * a.pool.head_stride +
                   (pos - page_at * a.pool.page_tokens) * a.pool.token_stride;       // of a key or a value
    T *q_to = is_q ? static_cast<T *>(a.q_out) + token * a.q_out_stride + h * a.pool.width : nullptr;

    const int half = a.rotary / 2;
    const int64_t angles = (int64_t)pos * half;
    // in halves: unit u of the rotated part holds values 4u.. and half + 4u..
    const bool turned = (is_q || is_k) && u * 8 < a.rotary;
    float x[8];
    if constexpr (VEC) {
        const int e0 = HALVES && turned ? u * 4 : u * 8;
        const int e1 = HALVES && turned ? half + u * 4 : u * 8 + 4;
        load_values<T, 4>(from + e0, x, 0);
        load_values<T, 4>(from + e1, x, 4);
        if (turned) {
            float cs[8], sn[8];
            load_values<float, 4>(a.cosine + angles + u * 4, cs, 0);
            load_values<float, 4>(a.sine + angles + u * 4, sn, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i0 = HALVES ? j : 2 * j, i1 = HALVES ? j + 4 : 2 * j + 1;
                const float p = x[i0], r = x[i1];
                x[i0] = fmaf(p, cs[j], -(r * sn[j]));
                x[i1] = fmaf(p, sn[j], r * cs[j]);
            }
        }
        if (is_q) {
            store_values<T, 4>(q_to + e0, x, 0);
            store_values<T, 4>(q_to + e1, x, 4);
        } else {
            store_values<_Float16, 4>(to + e0, x, 0);
            store_values<_Float16, 4>(to + e1, x, 4);
        }
    } else {
        // pairs 4u..4u+3 of the rotated part (both of a pair read before either is written; q_out may be
        // q), then single values
        const int pairs = is_q || is_k ? min(4, max(0, half - u * 4)) : 0;
        for (int i = 0; i < pairs; ++i) {
            const int j = u * 4 + i, e0 = HALVES ? j : 2 * j, e1 = HALVES ? half + j : 2 * j + 1;
            const float p = static_cast<float>(from[e0]), r = static_cast<float>(from[e1]);
            const float cs = a.cosine[angles + j], sn = a.sine[angles + j];
            const float y0 = fmaf(p, cs, -(r * sn)), y1 = fmaf(p, sn, r * cs);
            if (is_q) {
                q_to[e0] = static_cast<T>(y0);
                q_to[e1] = static_cast<T>(y1);
            } else {
                to[e0] = static_cast<_Float16>(y0);
                to[e1] = static_cast<_Float16>(y1);
            }
        }
        for (int e = u * 8 + 2 * pairs; e < u * 8 + 8; ++e) {
            const float value = static_cast<float>(from[e]);
            if (is_q) q_to[e] = static_cast<T>(value);
            else to[e] = static_cast<_Float16>(value);
        }
    }
}

template <typename T, bool HALVES>
void launch(const AppendArgs &a, bool vec, hipStream_t stream) {
    const dim3 grid((a.units + kThreads - 1) / kThreads);
    if (vec) hipLaunchKernelGGL((append<T, HALVES, true>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((append<T, HALVES, false>), grid, dim3(kThreads), 0, stream, a);
}

} // namespace

extern "C" int kk_kv_append(void *k_pool, void *v_pool, void *q_out, const void *q, const void *k, const void *v,
                 const int *sequence, const int *position, const int *lengths, const int *table, const float *cosine,
                 const float *sine, const kunlun::KVCacheLayout &c, const kunlun::KVAppendLayout &p, int *status,
                 hipStream_t stream) {
    const int query_heads = q ? p.query_heads : 0;
    const int64_t per_head = c.width / 8, per_token = (query_heads + 2 * (int64_t)c.heads) * per_head;
    if (per_token * p.tokens > INT32_MAX - kThreads) return hipErrorInvalidValue;
    AppendArgs a;
    a.k_pool = static_cast<_Float16 *>(k_pool);
    a.v_pool = static_cast<_Float16 *>(v_pool);
    a.q_out = q_out;
    a.q = q;
    a.k = k;
    a.v = v;
    a.sequence = sequence;
    a.position = position;
    a.lengths = lengths;
    a.table = table;
    a.cosine = cosine;
    a.sine = sine;
    a.status = status;
    a.pool = PoolView(c);
    a.q_stride = p.q_stride;
    a.k_stride = p.k_stride;
    a.v_stride = p.v_stride;
    a.q_out_stride = p.q_out_stride;
    a.units_per_token = kk::FastDiv(static_cast<uint32_t>(per_token));
    a.units_per_head = kk::FastDiv(static_cast<uint32_t>(per_head));
    a.tokens = p.tokens;
    a.sequences = p.sequences;
    a.row_pages = p.row_pages;
    a.query_heads = query_heads;
    a.rotary = p.rotary;
    a.positions = p.positions;
    a.units = static_cast<uint32_t>(per_token * p.tokens);
    const bool f16 = p.type == kunlun::InputType::f16, halves = p.pairs == kunlun::RotaryPairs::halves;
    // loads and stores of 4 values: rows on 4 values, the rotated part whole units
    const int64_t strides = p.k_stride | p.v_stride | (q ? p.q_stride | p.q_out_stride : 0);
    const uintptr_t rows = (uintptr_t)k | (uintptr_t)v | (uintptr_t)q | (q ? (uintptr_t)q_out : 0);
    const bool vec = p.rotary % 8 == 0 && strides % 4 == 0 && rows % (f16 ? 8 : 16) == 0 &&
                     (p.rotary == 0 || ((uintptr_t)cosine | (uintptr_t)sine) % 16 == 0);
    if (f16) halves ? launch<_Float16, true>(a, vec, stream) : launch<_Float16, false>(a, vec, stream);
    else halves ? launch<float, true>(a, vec, stream) : launch<float, false>(a, vec, stream);
    return hipGetLastError();
}
