// The paged key-value cache in 8 bits: argument rules and submission, in the manner of kv_cache.cpp, whose rules for
// tables, rows and calls hold here too.
#include "kv_rules.h"
#include "launch.h"

namespace kunlun {

using namespace rules;

const char * kv_cache_f8_reason(const KVCacheF8Layout & f) {
    const char * cache = kv_cache_reason(f.cache);
    if (*cache) return cache;
    if (f.block_tokens <= 0 || f.block_tokens > 64 || (f.block_tokens & (f.block_tokens - 1)) ||
        f.cache.page_tokens % f.block_tokens)
        return "block";
    return "";
}

const char * paged_attention_f8_reason(const KVCacheF8Layout & f, const PagedAttentionLayout & p) {
    const char * cache = kv_cache_f8_reason(f);
    return *cache ? cache : paged_attention_reason(f.cache, p);
}

bool paged_attention_f8(Kernel & kernel, int id, void * y, const void * q, const void * k, const void * v,
                        const float * k_scales, const float * v_scales, const int * table, const int * lengths,
                        const KVCacheF8Layout & f, const PagedAttentionLayout & p) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    if (*kv_cache_f8_reason(f) ||
        !attention_ok(y, q, Pools(k, v, k_scales, v_scales, f), table, lengths, f.cache, p))
        return false;
    Kernel::Impl & impl = *kernel.impl_;
    if (!usable(impl, id)) return false;
    detail::DeviceContext & ctx = detail::context(id);
    void * room = nullptr;
    if (const size_t need = kk_paged_attention_f8_workspace_bytes(f.cache, p, ctx.cus)) {
        room = workspace(impl, id, ctx, need);
        if (!room) return false;
    }
    detail::check_hip((hipError_t)kk_paged_attention_f8(y, q, k, v, k_scales, v_scales, table, lengths, f, p, room,
                                                        ctx.status + 1, ctx.cus, ctx.stream),
                      "kk_paged_attention_f8");
    note(impl, id, kk_paged_attention_f8_route(f.cache, p, ctx.cus));
    return true;
}

const char * kv_append_f8_reason(const KVCacheF8Layout & f, const KVAppendLayout & p) {
    const char * cache = kv_cache_f8_reason(f);
    if (*cache) return cache;
    const char * call = kv_append_reason(f.cache, p);
    if (*call) return call;
    // a bound that no launch comes near (a token's head takes up to 64 lanes and its part of a block's workgroup up to 128), so
    // that the launch's numbers stay within 32 bits whatever the widths and blocks
    if ((p.query_heads * (int64_t)(f.cache.width / 8) + 2 * (int64_t)f.cache.heads * 256) * p.tokens > INT32_MAX - 1024)
        return "shape";
    return "";
}

bool kv_append_f8(Kernel & kernel, int id, void * k_pool, void * v_pool, float * k_scales, float * v_scales, void * q_out,
                  const void * q, const void * k, const void * v, const int * sequence, const int * position,
                  const int * lengths, const int * table, const float * cosine, const float * sine,
                  const KVCacheF8Layout & f, const KVAppendLayout & given) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    KVAppendLayout p = given;
    if (!q) p.query_heads = 0;          // without queries their layout is ignored
    if (*kv_append_f8_reason(f, p) ||
        !append_ok(Pools(k_pool, v_pool, k_scales, v_scales, f), q_out, q, k, v, sequence, position, lengths, table, cosine,
                   sine, f.cache, p))
        return false;
    Kernel::Impl & impl = *kernel.impl_;
    if (!usable(impl, id)) return false;
    detail::DeviceContext & ctx = detail::context(id);
    detail::check_hip((hipError_t)kk_kv_append_f8(k_pool, v_pool, k_scales, v_scales, q_out, q, k, v, sequence, position,
                                                  lengths, table, cosine, sine, f, p, ctx.status + 1, ctx.stream),
                      "kk_kv_append_f8");
    note(impl, id, "kv_append_f8");
    return true;
}

const char * kv_read_f8_reason(const KVCacheF8Layout & f, const KVReadLayout & p) {
    const char * cache = kv_cache_f8_reason(f);
    if (*cache) return cache;
    if (!known(p.type)) return "type";
    if (p.tokens <= 0 || p.sequences <= 0 || p.row_pages <= 0) return "shape";
    if ((int64_t)p.row_pages * f.cache.page_tokens > kMostTokens) return "length";
    if (2 * (int64_t)f.cache.heads * (f.cache.width / 8) * p.tokens > INT32_MAX - 1024) return "shape";
    for (const int64_t s : {p.k_stride, p.v_stride})
        if (s < (int64_t)f.cache.heads * f.cache.width || s > kMostStride) return "stride";
    return "";
}

bool kv_read_f8(Kernel & kernel, int id, void * k, void * v, const void * k_pool, const void * v_pool,
                const float * k_scales, const float * v_scales, const int * sequence, const int * position,
                const int * lengths, const int * table, const KVCacheF8Layout & f, const KVReadLayout & p) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    if (*kv_read_f8_reason(f, p) || !k || !v || !table) return false;
    // a token's place: by position (with its sequence), or the newest of each sequence
    if (position ? !sequence : sequence || !lengths || p.tokens > p.sequences) return false;
    const Pools pools(k_pool, v_pool, k_scales, v_scales, f);
    const int bytes = element_bytes(p.type);
    if (!pools.given() || !pools.aligned() || !aligned_to(bytes, {k, v}) ||
        !aligned_to(4, {sequence, position, lengths, table}))
        return false;
    const int64_t row = (int64_t)f.cache.heads * f.cache.width;
    const Span k_out = rows_span(k, p.tokens, p.k_stride, row, bytes), v_out = rows_span(v, p.tokens, p.v_stride, row, bytes);
    const Span rows = ints(table, (int64_t)p.sequences * p.row_pages);
    const Span counts = ints(position ? nullptr : lengths, p.sequences);
    const Span at = ints(position, p.tokens), of = ints(sequence, p.tokens);
    if (wraps({k_out, v_out, rows, counts, at, of}) || pools.wrap() || pools.meet({k_out, v_out}) ||
        clash(k_out, {rows, counts, at, of}) || clash(v_out, {rows, counts, at, of}))
        return false;
    // rows of their own, or columns of common rows that lie side by side
    if (clash(k_out, v_out)) {
        const uintptr_t step = (uintptr_t)p.k_stride * bytes, width = (uintptr_t)row * bytes;
        const uintptr_t delta = (uintptr_t)k > (uintptr_t)v ? (uintptr_t)k - (uintptr_t)v : (uintptr_t)v - (uintptr_t)k;
        if (p.k_stride != p.v_stride || delta < width || delta + width > step) return false;
    }
    Kernel::Impl & impl = *kernel.impl_;
    if (!usable(impl, id)) return false;
    detail::DeviceContext & ctx = detail::context(id);
    detail::check_hip((hipError_t)kk_kv_read_f8(k, v, k_pool, v_pool, k_scales, v_scales, sequence, position, lengths, table,
                                                f, p, ctx.status + 1, ctx.stream),
                      "kk_kv_read_f8");
    note(impl, id, "kv_read_f8");
    return true;
}

const char * kv_pages_f8_reason(const KVCacheF8Layout & f, const KVPagesLayout & p) {
    const char * cache = kv_cache_f8_reason(f);
    return *cache ? cache : kv_pages_reason(f.cache, p);
}

bool kv_fork_f8(Kernel & kernel, int id, void * k, void * v, float * k_scales, float * v_scales, int * table, int * lengths,
                int * references, const int * parents, const int * children, int count, const KVCacheF8Layout & f,
                const KVPagesLayout & p) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    if (*kv_pages_f8_reason(f, p) || !fork_ok(Pools(k, v, k_scales, v_scales, f, p), table, lengths, references, parents,
                                              children, count, f.cache, p))
        return false;
    Kernel::Impl & impl = *kernel.impl_;
    if (!usable(impl, id)) return false;
    detail::DeviceContext & ctx = detail::context(id);
    void * room = workspace(impl, id, ctx, kk_kv_fork_workspace_bytes(p, count));
    if (!room) return false;
    detail::check_hip((hipError_t)kk_kv_fork_f8(k, v, k_scales, v_scales, table, lengths, references, parents, children,
                                                count, f, p, room, ctx.status + 1, ctx.stream),
                      "kk_kv_fork_f8");
    note(impl, id, "kv_fork_f8");
    return true;
}

bool kv_compact_f8(Kernel & kernel, int id, void * k, void * v, float * k_scales, float * v_scales, int * table_out,
                   int * references_out, int * used, const int * table, const int * lengths, const int * references,
                   const KVCacheF8Layout & f, const KVPagesLayout & p) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    if (*kv_pages_f8_reason(f, p) || !compact_ok(Pools(k, v, k_scales, v_scales, f, p), table_out, references_out, used,
                                                 table, lengths, references, f.cache, p))
        return false;
    Kernel::Impl & impl = *kernel.impl_;
    if (!usable(impl, id)) return false;
    detail::DeviceContext & ctx = detail::context(id);
    void * room = workspace(impl, id, ctx, kk_kv_compact_workspace_bytes(f.cache));
    if (!room) return false;
    detail::check_hip((hipError_t)kk_kv_compact_f8(k, v, k_scales, v_scales, table_out, references_out, used, table, lengths,
                                                   references, f, p, room, ctx.status + 1, ctx.cus, ctx.stream),
                      "kk_kv_compact_f8");
    note(impl, id, "kv_compact_f8");
    return true;
}

bool kv_copy_pages_f8(Kernel & kernel, int id, void * k, void * v, float * k_scales, float * v_scales, const int * sources,
                      const int * destinations, int count, const KVCacheF8Layout & f, const KVPagesLayout & p) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    if (*kv_pages_f8_reason(f, p) ||
        !copy_ok(Pools(k, v, k_scales, v_scales, f, p), sources, destinations, count, f.cache, p))
        return false;
    Kernel::Impl & impl = *kernel.impl_;
    if (!usable(impl, id)) return false;
    detail::DeviceContext & ctx = detail::context(id);
    detail::check_hip((hipError_t)kk_kv_copy_pages_f8(k, v, k_scales, v_scales, sources, destinations, count, f, p,
                                                      ctx.status + 1, ctx.cus, ctx.stream),
                      "kk_kv_copy_pages_f8");
    note(impl, id, "kv_copy_pages_f8");
    return true;
}

} // namespace kunlun
