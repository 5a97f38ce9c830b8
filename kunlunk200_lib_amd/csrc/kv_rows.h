// Runs of N values between a product's rows or a pool and registers.
#pragma once

#include <hip/hip_runtime.h>

namespace kk {

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

} // namespace kk
