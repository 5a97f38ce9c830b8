// Logits before a token is chosen: penalties for repeated tokens, biases, a
// grammar's mask. One pass over the logits in F32; bound by reading and writing
// them (8 bytes a token).
//
// A workgroup takes a slice of one row, 4 * VPT logits a thread, which are on their
// way first. Meanwhile it counts the row's history and finds the last bias entry
// of each token in LDS words of its own slice, by integer atomics, whose order
// does not matter. Each slice reads the row's lists (from the L2 after the first)
// and tests every entry: of 200 rows x 32000 with 3000 history entries and 300 biases, 15.9 us, that is 2.7.
#include "device_common.h"
#include "launch.h"
#include "paged.h"

#include <kunlun/k200.h>

namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 8;                // history entries a thread reads ahead

struct LogitsArgs {
    float *y;
    const float *logits, *penalties;
    const int *history, *history_lengths, *bias_ids;
    const float *bias_values;
    const int *bias_lengths;
    const uint32_t *mask;
    int64_t logits_stride, y_stride, history_stride, bias_stride, mask_stride;
    int *status;
    int vocabulary;
};

constexpr int slice_of(int vpt) { return kThreads * 4 * vpt; }

// A word that no lane writes during the launch, read through the scalar cache.
template <typename T>
__device__ __forceinline__ T scalar_load(const T *p) {
    return *(const __attribute__((address_space(4))) T *)(p);
}

template <int VPT, bool VEC>
__global__ __launch_bounds__(kThreads) void process(LogitsArgs a) {
    constexpr int kSlice = slice_of(VPT);
    // counts, then bias entries: their place in the list + 1 above their value, so that the largest word is the last entry
    __shared__ uint4 words[3 * kSlice / 4];
    uint32_t *counts = reinterpret_cast<uint32_t *>(words);
    unsigned long long *entries = reinterpret_cast<unsigned long long *>(counts + kSlice);
    const int tid = threadIdx.x, row = blockIdx.y, first = blockIdx.x * kSlice;
    const int n = min(kSlice, a.vocabulary - first);
    const bool counted = a.history != nullptr, biased = a.bias_ids != nullptr;
    const float *in = a.logits + row * a.logits_stride + first;
    float *out = a.y + row * a.y_stride + first;
    const int *history = a.history + row * a.history_stride, *ids = a.bias_ids + row * a.bias_stride;
    const float *values = a.bias_values + row * a.bias_stride;

    // everything that is read is on its way at once: logits, mask, the first entries of both lists
    float4 z[VPT];
    uint32_t bits[VPT];
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
        const int i = (u * kThreads + tid) * 4;
        if (VEC && i + 4 <= n) {
            z[u] = *reinterpret_cast<const float4 *>(in + i);
        } else {
            // past the end the last logit again: it is not stored
            z[u] = make_float4(in[min(i, n - 1)], in[min(i + 1, n - 1)], in[min(i + 2, n - 1)], in[min(i + 3, n - 1)]);
        }
        const int at = min(i, n - 1);
        bits[u] = a.mask ? a.mask[row * a.mask_stride + (first + at) / 32] >> (at & 28) : ~0u;
    }
    // a list's length, cut to its room and reported where that is less
    auto length = [&](const int *lengths, int64_t room) {
        const int n = scalar_load(lengths + row);
        if ((n < 0 || n > room) && first == 0 && tid == 0) kk::report(a.status, kk::kBadIndex);
        return static_cast<int>(min<int64_t>(max(n, 0), room));
    };
    const int past = counted ? length(a.history_lengths, a.history_stride) : 0;
    const int given = biased ? length(a.bias_lengths, a.bias_stride) : 0;
    int seen[kAhead], id[2];
    float value[2];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) seen[u] = u * kThreads + tid < past ? history[u * kThreads + tid] : -1;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const bool in_list = u * kThreads + tid < given;
        id[u] = in_list ? ids[u * kThreads + tid] : -1;
        value[u] = in_list ? values[u * kThreads + tid] : 0.0f;
    }
    float r = 1.0f, f = 0.0f, p = 0.0f;
    if (counted) {
        r = scalar_load(a.penalties + row * 3);
        f = scalar_load(a.penalties + row * 3 + 1);
        p = scalar_load(a.penalties + row * 3 + 2);
    }
    // the slice's place of a token, or past its end
    auto place = [&](int token) { return token < 0 ? ~0u : static_cast<uint32_t>(token - first); };
    if (past > 0 || given > 0) {
#pragma unroll
        for (int u = 0; u < 3 * VPT; ++u) words[u * kThreads + tid] = make_uint4(0, 0, 0, 0);
        kk::lds_barrier();                           // the loads stay in flight
        auto count = [&](int token) {
            const uint32_t t = place(token);
            if (t < static_cast<uint32_t>(n)) atomicAdd(&counts[t], 1u);
        };
        auto enter = [&](int token, int i, float x) {
            const uint32_t t = place(token);
            if (t < static_cast<uint32_t>(n))
                atomicMax(&entries[t], static_cast<unsigned long long>(i + 1) << 32 | __float_as_uint(x));
        };
#pragma unroll
        for (int u = 0; u < kAhead; ++u) count(seen[u]);
        for (int i0 = kAhead * kThreads + tid; i0 < past; i0 += 4 * kThreads) {
            int token[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) token[u] = i0 + u * kThreads < past ? history[i0 + u * kThreads] : -1;
#pragma unroll
            for (int u = 0; u < 4; ++u) count(token[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) enter(id[u], u * kThreads + tid, value[u]);
        for (int i = 2 * kThreads + tid; i < given; i += kThreads) enter(ids[i], i, values[i]);
        kk::lds_barrier();
#pragma unroll
        for (int u = 0; u < VPT; ++u) {
            const uint4 met = reinterpret_cast<const uint4 *>(counts)[u * kThreads + tid];
            const uint4 b01 = reinterpret_cast<const uint4 *>(entries)[(u * kThreads + tid) * 2];
            const uint4 b23 = reinterpret_cast<const uint4 *>(entries)[(u * kThreads + tid) * 2 + 1];
            auto less = [&](float x, uint32_t times) {
                return times ? (x > 0.0f ? x / r : x * r) - static_cast<float>(times) * f - p : x;
            };
            if (met.x | met.y | met.z | met.w)       // few waves: a division is ten instructions
                z[u] = make_float4(less(z[u].x, met.x), less(z[u].y, met.y), less(z[u].z, met.z), less(z[u].w, met.w));
            z[u].x += __uint_as_float(b01.x);
            z[u].y += __uint_as_float(b01.z);
            z[u].z += __uint_as_float(b23.x);
            z[u].w += __uint_as_float(b23.z);
        }
    }
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
        const int i = (u * kThreads + tid) * 4;
        z[u].x = bits[u] & 1 ? z[u].x : -INFINITY;
        z[u].y = bits[u] & 2 ? z[u].y : -INFINITY;
        z[u].z = bits[u] & 4 ? z[u].z : -INFINITY;
        z[u].w = bits[u] & 8 ? z[u].w : -INFINITY;
        if (VEC && i + 4 <= n) {
            *reinterpret_cast<float4 *>(out + i) = z[u];
        } else {
            if (i < n) out[i] = z[u].x;
            if (i + 1 < n) out[i + 1] = z[u].y;
            if (i + 2 < n) out[i + 2] = z[u].z;
            if (i + 3 < n) out[i + 3] = z[u].w;
        }
    }
}

template <int VPT>
void launch(const LogitsArgs &a, int rows, bool vec, hipStream_t stream) {
    const dim3 grid((a.vocabulary + slice_of(VPT) - 1) / slice_of(VPT), rows);
    if (vec) hipLaunchKernelGGL((process<VPT, true>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((process<VPT, false>), grid, dim3(kThreads), 0, stream, a);
}

} // namespace

extern "C" int kk_process_logits(float *y, const float *logits, const float *penalties, const int *history,
                      const int *history_lengths, const int *bias_ids, const float *bias_values,
                      const int *bias_lengths, const uint32_t *mask, const kunlun::LogitsLayout &p,
                      int *status, int cus, hipStream_t stream) {
    if (p.rows <= 0 || p.rows > 65535 || p.vocabulary <= 0) return hipErrorInvalidValue;
    const LogitsArgs a{y, logits, penalties, history, history_lengths, bias_ids, bias_values, bias_lengths, mask,
                       p.logits_stride, p.y_stride, p.history_stride, p.bias_stride, p.mask_stride, status, p.vocabulary};
    const bool vec = ((uintptr_t)y | (uintptr_t)logits) % 16 == 0 && (p.logits_stride | p.y_stride) % 4 == 0;
    // larger slices read the lists less often, smaller ones leave no CU idle: 200 rows x 32000, history 3000: slices of
    // 4096 logits 20.3 us, 2048 15.9, 1024 16.6; up to 64 rows they are equal
    const int64_t logits_of_call = (int64_t)p.rows * p.vocabulary;
    if (logits_of_call >= (int64_t)slice_of(2) * 4 * cus) launch<2>(a, p.rows, vec, stream);
    else launch<1>(a, p.rows, vec, stream);
    return hipGetLastError();
}
