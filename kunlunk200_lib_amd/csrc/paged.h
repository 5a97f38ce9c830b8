// What the kernels of the paged key-value cache share: addresses in a pool and
// the status word that they and the logits step report to.
#pragma once

#include <hip/hip_runtime.h>
#include <kunlun/k200.h>

#include <cstdint>

namespace kk {

// n / d for 0 <= n < 2^31 by a multiplication: with L = ceil(log2 d) and
// mul = ceil(2^(31+L) / d), n * mul / 2^(31+L) exceeds n / d by less than
// n / 2^31 / d, too little to reach the next integer.
struct FastDiv {
    uint32_t mul, shift, d;
    FastDiv() = default;
    __host__ explicit FastDiv(uint32_t divisor) : d(divisor) {
        uint32_t log = 0;
        while ((uint64_t(1) << log) < divisor) ++log;
        shift = 31 + log;
        mul = static_cast<uint32_t>(((uint64_t(1) << shift) + divisor - 1) / divisor);
    }
    __host__ __device__ __forceinline__ uint32_t div(uint32_t n) const {
        return static_cast<uint32_t>((static_cast<uint64_t>(n) * mul) >> shift);
    }
};

// Bits of the status word (kv_cache_status).
constexpr int kBadPage = 1, kBadIndex = 2, kNoPage = 4;

__device__ __forceinline__ void report(int *status, int bit) { atomicOr(status, bit); }

// One layout's addressing. Strides in elements.
struct PoolView {
    int64_t page_stride, head_stride, token_stride;
    int pages, page_tokens, heads, width;
    FastDiv per_page;
    PoolView() = default;
    __host__ explicit PoolView(const kunlun::KVCacheLayout &c)
        : page_stride(c.page_stride), head_stride(c.head_stride), token_stride(c.token_stride), pages(c.pages),
          page_tokens(c.page_tokens), heads(c.heads), width(c.width),
          per_page(static_cast<uint32_t>(c.page_tokens)) {}
};

} // namespace kk
