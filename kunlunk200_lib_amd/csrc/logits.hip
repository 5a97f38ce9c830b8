// Logits before a token is chosen: penalties for repeated tokens, biases, a
// grammar's mask. One pass over the logits in F32; bound by reading and writing
// them (8 bytes a token).
//
// A workgroup takes a slice of one row. It counts the row's history and finds the last
// bias entry of each token in LDS words of its own slice by integer atomics, whose order does not
// matter, then goes over the slice once. Each slice reads the row's lists (from
// the L2 after the first).
#include "device_common.h"
#include "launch.h"

#include <kunlun/k200.h>

namespace {

constexpr int kThreads = 256;
constexpr int kSlice = 4096;

struct LogitsArgs {
    float *y;
    const float *logits, *penalties;
    const int *history, *history_lengths, *bias_ids;
    const float *bias_values;
    const int *bias_lengths;
    const uint32_t *mask;
    int64_t logits_stride, y_stride, history_stride, bias_stride, mask_stride;
    int vocabulary;
};

template <bool VEC>
__global__ __launch_bounds__(kThreads) void process(LogitsArgs a) {
    __shared__ uint32_t counts[kSlice], entries[kSlice];
    const int tid = threadIdx.x, row = blockIdx.y, first = blockIdx.x * kSlice;
    const int n = min(kSlice, a.vocabulary - first);
    const bool counted = a.history != nullptr, biased = a.bias_ids != nullptr;
    for (int i = tid; i < kSlice; i += kThreads) counts[i] = entries[i] = 0;
    __syncthreads();
    if (counted) {
        const int *history = a.history + row * a.history_stride;
        const int length = static_cast<int>(min<int64_t>(a.history_lengths[row], a.history_stride));
        for (int i = tid; i < length; i += kThreads) {
            const unsigned t = static_cast<unsigned>(history[i] - first);
            if (history[i] >= 0 && t < static_cast<unsigned>(n)) atomicAdd(&counts[t], 1u);
        }
    }
    if (biased) {
        const int *ids = a.bias_ids + row * a.bias_stride;
        const int length = static_cast<int>(min<int64_t>(a.bias_lengths[row], a.bias_stride));
        for (int i = tid; i < length; i += kThreads) {
            const unsigned t = static_cast<unsigned>(ids[i] - first);
            if (ids[i] >= 0 && t < static_cast<unsigned>(n)) atomicMax(&entries[t], static_cast<uint32_t>(i) + 1);
        }
    }
    __syncthreads();
    float r = 1.0f, f = 0.0f, p = 0.0f;
    if (counted) {
        r = a.penalties[row * 3];
        f = a.penalties[row * 3 + 1];
        p = a.penalties[row * 3 + 2];
    }
    const float *in = a.logits + row * a.logits_stride + first;
    float *out = a.y + row * a.y_stride + first;
    const uint32_t *mask = a.mask ? a.mask + row * a.mask_stride + first / 32 : nullptr;
    const float *values = biased ? a.bias_values + row * a.bias_stride : nullptr;
    auto one = [&](int i, float z) {
        const uint32_t met = counts[i], entry = entries[i];
        if (met) {
            z = z > 0.0f ? z / r : z * r;
            z = z - static_cast<float>(met) * f - p;
        }
        if (entry) z += values[entry - 1];
        return z;
    };
    constexpr int N = VEC ? 4 : 1;
    for (int i = tid * N; i < n; i += kThreads * N) {
        float z[N];
        if constexpr (VEC) {
            // a row's last tokens past a multiple of 4 one by one
            if (i + 4 <= n) {
                const float4 x = *reinterpret_cast<const float4 *>(in + i);
                z[0] = x.x, z[1] = x.y, z[2] = x.z, z[3] = x.w;
            } else {
                for (int j = 0; j < 4; ++j) z[j] = i + j < n ? in[i + j] : 0.0f;
            }
        } else {
            z[0] = in[i];
        }
        const uint32_t bits = mask ? mask[i / 32] >> (i % 32) : ~0u;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            z[j] = one(i + j, z[j]);
            if (!(bits >> j & 1)) z[j] = -INFINITY;
        }
        if constexpr (VEC) {
            if (i + 4 <= n) *reinterpret_cast<float4 *>(out + i) = make_float4(z[0], z[1], z[2], z[3]);
            else
                for (int j = 0; j < 4; ++j)
                    if (i + j < n) out[i + j] = z[j];
        } else {
            out[i] = z[0];
        }
    }
}

} // namespace

extern "C" int kk_process_logits(float *y, const float *logits, const float *penalties, const int *history,
                      const int *history_lengths, const int *bias_ids, const float *bias_values,
                      const int *bias_lengths, const uint32_t *mask, const kunlun::LogitsLayout &p,
                      hipStream_t stream) {
    const int slices = (p.vocabulary + kSlice - 1) / kSlice;
    if (p.rows <= 0 || p.rows > 65535 || p.vocabulary <= 0) return hipErrorInvalidValue;
    const LogitsArgs a{y, logits, penalties, history, history_lengths, bias_ids, bias_values, bias_lengths, mask,
                       p.logits_stride, p.y_stride, p.history_stride, p.bias_stride, p.mask_stride, p.vocabulary};
    const bool vec = ((uintptr_t)y | (uintptr_t)logits) % 16 == 0 && (p.logits_stride | p.y_stride) % 4 == 0;
    if (vec) hipLaunchKernelGGL(process<true>, dim3(slices, p.rows), dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL(process<false>, dim3(slices, p.rows), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}
