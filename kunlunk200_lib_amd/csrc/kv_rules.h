// What the entry points of the paged caches (F16 and 8-bit) and the logits step share on the host: argument rules, spans of
// memory, the Kernel's workspace. Not installed.
#pragma once

#include "runtime_internal.h"

#include <algorithm>
#include <cstdint>
#include <initializer_list>

namespace kunlun {
namespace rules {

constexpr int64_t kMostStride = int64_t(1) << 40;        // elements
constexpr int64_t kMostTokens = int64_t(1) << 27;        // of a sequence
constexpr int kMostCounted = 1 << 30;                    // pages and sequences that 32-bit loops count in steps

struct Span {
    uintptr_t at;
    size_t bytes;
    Span(const void * p, size_t n) : at((uintptr_t)p), bytes(p ? n : 0) {}
};

inline bool clash(const Span & a, const Span & b) {
    return a.bytes && b.bytes && a.at < b.at + b.bytes && b.at < a.at + a.bytes;
}
// Whether an output meets any of the others, or the others' list itself is out of range.
inline bool clash(const Span & out, std::initializer_list<Span> others) {
    for (const Span & s : others)
        if (clash(out, s)) return true;
    return false;
}
inline bool wraps(std::initializer_list<Span> spans) {
    for (const Span & s : spans)
        if (s.at + s.bytes < s.at) return true;
    return false;
}
inline bool aligned_to(size_t bytes, std::initializer_list<const void *> pointers) {
    for (const void * p : pointers)
        if ((uintptr_t)p % bytes) return false;
    return true;
}

inline int element_bytes(InputType type) { return type == InputType::f32 ? 4 : 2; }
inline bool known(InputType type) { return type == InputType::f32 || type == InputType::f16; }

// Elements from a pool's first value to its last, both included.
inline int64_t pool_elements(const KVCacheLayout & c) {
    return (c.pages - 1) * c.page_stride + (c.heads - 1) * c.head_stride + (c.page_tokens - 1) * c.token_stride + c.width;
}
// Rows of `width` values of `bytes` each.
inline Span rows_span(const void * first, int64_t rows, int64_t stride, int64_t width, int bytes) {
    return Span(first, (size_t)((rows - 1) * stride + width) * bytes);
}
inline Span ints(const void * p, int64_t n) { return Span(p, (size_t)n * 4); }

// The Kernel's device, or a visible one that the Kernel may be bound to.
template <typename Impl>
bool usable(const Impl & impl, int device) {
    return detail::device_visible(device) && (impl.id == -1 || impl.id == device);
}

// The Kernel's workspace of the cache operators; nullptr when there is no memory for it.
template <typename Impl>
void * workspace(Impl & impl, int device, detail::DeviceContext & ctx, size_t need) {
    if (impl.kv_workspace_size < need) {
        if (impl.kv_workspace) {
            detail::check_hip(hipStreamSynchronize(ctx.stream), "hipStreamSynchronize");
            release(device, impl.kv_workspace, impl.kv_workspace_size);
            impl.kv_workspace = nullptr;
            impl.kv_workspace_size = 0;
        }
        // at least 1 MiB, so that a decode loop's growing lengths seldom get here
        const size_t size = std::max<size_t>(need, size_t(1) << 20);
        impl.kv_workspace = allocate(device, size);
        if (!impl.kv_workspace) return nullptr;
        impl.kv_workspace_size = size;
    }
    return impl.kv_workspace;
}

template <typename Impl>
void note(Impl & impl, int device, const char * route) {
    impl.id = device;
    impl.route = route;
    detail::note_route(route);
}

// The memory of a cache: F16 pools, or 8-bit pools with their scales. Of layouts whose reasons are "".
struct Pools {
    Span part[4];                        // keys, values, their scales
    int parts;
    Pools(const void * k, const void * v, const KVCacheLayout & c)
        : part{Span(k, values(c) * 2), Span(v, values(c) * 2), Span(nullptr, 0), Span(nullptr, 0)}, parts(2) {}
    Pools(const void * k, const void * v, const KVCacheLayout & c, const KVPagesLayout & p)
        : part{Span(k, values(c, p) * 2), Span(v, values(c, p) * 2), Span(nullptr, 0), Span(nullptr, 0)}, parts(2) {}
    Pools(const void * k, const void * v, const float * k_scales, const float * v_scales, const KVCacheF8Layout & f)
        : part{Span(k, values(f.cache)), Span(v, values(f.cache)), Span(k_scales, scales(f) * 4),
               Span(v_scales, scales(f) * 4)}, parts(4) {}
    Pools(const void * k, const void * v, const float * k_scales, const float * v_scales, const KVCacheF8Layout & f,
          const KVPagesLayout & p)
        : part{Span(k, values(f.cache, p)), Span(v, values(f.cache, p)), Span(k_scales, scales(f) * p.layers * 4),
               Span(v_scales, scales(f) * p.layers * 4)}, parts(4) {}
    bool given() const {
        for (int i = 0; i < parts; ++i)
            if (!part[i].at) return false;
        return true;
    }
    bool aligned() const { return part[0].at % 16 == 0 && part[1].at % 16 == 0 && part[2].at % 4 == 0 && part[3].at % 4 == 0; }
    bool wrap() const { return wraps({part[0], part[1], part[2], part[3]}); }
    bool meet(const Span & other) const { return clash(other, {part[0], part[1], part[2], part[3]}); }
    bool meet(std::initializer_list<Span> others) const {
        for (const Span & s : others)
            if (meet(s)) return true;
        return false;
    }
    bool meet_each_other() const {
        return clash(part[0], {part[1], part[2], part[3]}) || clash(part[1], {part[2], part[3]}) || clash(part[2], part[3]);
    }
private:
    static size_t values(const KVCacheLayout & c) { return (size_t)pool_elements(c); }
    static size_t values(const KVCacheLayout & c, const KVPagesLayout & p) {
        return (size_t)(p.layers - 1) * p.layer_stride + pool_elements(c);
    }
    static size_t scales(const KVCacheF8Layout & f) {
        return (size_t)f.cache.pages * f.cache.heads * (f.cache.page_tokens / f.block_tokens);
    }
};

// The three arrays of a table, apart from each other and from `others`.
struct TableSpans {
    Span rows, lengths, references;
    TableSpans(const void * table, const void * lengths_, const void * references_, const KVCacheLayout & c,
               const KVPagesLayout & p)
        : rows(ints(table, (int64_t)p.sequences * p.row_pages)), lengths(ints(lengths_, p.sequences)),
          references(ints(references_, c.pages)) {}
    bool bad(std::initializer_list<Span> others) const {
        if (wraps({rows, lengths, references}) || wraps(others)) return true;
        return clash(rows, {lengths, references}) || clash(lengths, {references}) || clash(rows, others) ||
               clash(lengths, others) || clash(references, others);
    }
};

inline bool list_ok(int count, int most) { return count > 0 && count <= most; }

// Whether a call's layouts, pointers and memory are in order (the layouts' reasons are asked first).
bool attention_ok(const void * y, const void * q, const Pools & pools, const int * table, const int * lengths,
                  const KVCacheLayout & c, const PagedAttentionLayout & p);
bool append_ok(const Pools & pools, const void * q_out, const void * q, const void * k, const void * v,
               const int * sequence, const int * position, const int * lengths, const int * table, const float * cosine,
               const float * sine, const KVCacheLayout & c, const KVAppendLayout & p);
bool fork_ok(const Pools & pools, const int * table, const int * lengths, const int * references, const int * parents,
             const int * children, int count, const KVCacheLayout & c, const KVPagesLayout & p);
bool compact_ok(const Pools & pools, const int * table_out, const int * references_out, const int * used,
                const int * table, const int * lengths, const int * references, const KVCacheLayout & c,
                const KVPagesLayout & p);
bool copy_ok(const Pools & pools, const int * sources, const int * destinations, int count, const KVCacheLayout & c,
             const KVPagesLayout & p);

} // namespace rules
} // namespace kunlun
