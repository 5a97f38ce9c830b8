// The paged key-value cache and the logits step: argument rules, workspaces and
// submission. None of them has a counterpart in the part of the reference's
// header that this library keeps; they follow matmul in submitting without
// waiting and swiglu in refusing arguments by their return value.
#include "launch.h"
#include "runtime_internal.h"

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <initializer_list>

namespace kunlun {

namespace {

constexpr int64_t kMostStride = int64_t(1) << 40;        // elements
constexpr int64_t kMostTokens = int64_t(1) << 27;        // of a sequence
constexpr int kMostCounted = 1 << 30;                    // pages and sequences that 32-bit loops count in steps

struct Span {
    uintptr_t at;
    size_t bytes;
    Span(const void * p, size_t n) : at((uintptr_t)p), bytes(p ? n : 0) {}
};

bool clash(const Span & a, const Span & b) {
    return a.bytes && b.bytes && a.at < b.at + b.bytes && b.at < a.at + a.bytes;
}
// Whether an output meets any of the others, or the others' list itself is out of range.
bool clash(const Span & out, std::initializer_list<Span> others) {
    for (const Span & s : others)
        if (clash(out, s)) return true;
    return false;
}
bool wraps(std::initializer_list<Span> spans) {
    for (const Span & s : spans)
        if (s.at + s.bytes < s.at) return true;
    return false;
}
bool aligned_to(size_t bytes, std::initializer_list<const void *> pointers) {
    for (const void * p : pointers)
        if ((uintptr_t)p % bytes) return false;
    return true;
}

int element_bytes(InputType type) { return type == InputType::f32 ? 4 : 2; }
bool known(InputType type) { return type == InputType::f32 || type == InputType::f16; }

// Elements from a pool's first value to its last, both included.
int64_t pool_elements(const KVCacheLayout & c) {
    return (c.pages - 1) * c.page_stride + (c.heads - 1) * c.head_stride + (c.page_tokens - 1) * c.token_stride + c.width;
}
Span pool_span(const void * pool, const KVCacheLayout & c) { return Span(pool, (size_t)pool_elements(c) * 2); }
Span pool_span(const void * pool, const KVCacheLayout & c, const KVPagesLayout & p) {
    return Span(pool, ((size_t)(p.layers - 1) * p.layer_stride + pool_elements(c)) * 2);
}
// Rows of `width` values of `bytes` each.
Span rows_span(const void * first, int64_t rows, int64_t stride, int64_t width, int bytes) {
    return Span(first, (size_t)((rows - 1) * stride + width) * bytes);
}
Span ints(const void * p, int64_t n) { return Span(p, (size_t)n * 4); }

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

} // namespace

const char * kv_cache_reason(const KVCacheLayout & c) {
    if (c.pages <= 0 || c.page_tokens <= 0 || c.page_tokens > 65536 || c.heads <= 0 || c.heads > 1024 ||
        c.width <= 0 || c.width > 256 || c.width % 8)
        return "shape";
    for (const int64_t s : {c.page_stride, c.head_stride, c.token_stride})
        if (s < c.width || s > kMostStride || s % 8) return "stride";
    // one order within a page: a head's tokens together, or a token's heads
    const int64_t head_run = (c.page_tokens - 1) * c.token_stride + c.width;
    const int64_t token_run = (c.heads - 1) * c.head_stride + c.width;
    const bool heads = (c.heads == 1 || c.head_stride >= head_run) &&
                       c.page_stride >= (c.heads - 1) * c.head_stride + head_run;
    const bool tokens = (c.page_tokens == 1 || c.token_stride >= token_run) &&
                        c.page_stride >= (c.page_tokens - 1) * c.token_stride + token_run;
    if (!heads && !tokens) return "stride";
    if (c.page_stride > (INT64_MAX / 4) / c.pages) return "byte extent";
    return "";
}

const char * paged_attention_reason(const KVCacheLayout & c, const PagedAttentionLayout & p) {
    const char * cache = kv_cache_reason(c);
    if (*cache) return cache;
    if (!known(p.type)) return "type";
    if (p.sequences <= 0 || p.sequences > 65535 || p.row_pages <= 0 || p.window < 0) return "shape";
    if (p.query_heads <= 0 || p.query_heads > 1024 || p.query_heads % c.heads) return "heads";
    if (p.longest <= 0 || p.longest > kMostTokens - 4096 || p.longest > (int64_t)p.row_pages * c.page_tokens)
        return "length";
    if (!std::isfinite(p.scale * kLog2E)) return "scale";
    for (const int64_t s : {p.q_stride, p.y_stride})
        if (s < (int64_t)p.query_heads * c.width || s > kMostStride) return "stride";
    return "";
}

bool paged_attention(Kernel & kernel, int id, void * y, const void * q, const void * k, const void * v,
                     const int * table, const int * lengths, const KVCacheLayout & c,
                     const PagedAttentionLayout & p) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    if (*paged_attention_reason(c, p) || !y || !q || !k || !v || !table || !lengths) return false;
    const int bytes = element_bytes(p.type);
    if (!aligned_to(bytes, {y, q}) || !aligned_to(16, {k, v}) || !aligned_to(4, {table, lengths})) return false;
    const int64_t row = (int64_t)p.query_heads * c.width;
    const Span out = rows_span(y, p.sequences, p.y_stride, row, bytes);
    const Span in = rows_span(q, p.sequences, p.q_stride, row, bytes);
    const Span rows = ints(table, (int64_t)p.sequences * p.row_pages), counts = ints(lengths, p.sequences);
    const Span keys = pool_span(k, c), values = pool_span(v, c);
    if (wraps({out, in, rows, counts, keys, values}) || clash(out, {in, rows, counts, keys, values})) return false;
    Kernel::Impl & impl = *kernel.impl_;
    if (!usable(impl, id)) return false;
    detail::DeviceContext & ctx = detail::context(id);
    void * room = nullptr;
    if (const size_t need = kk_paged_attention_workspace_bytes(c, p, ctx.cus)) {
        room = workspace(impl, id, ctx, need);
        if (!room) return false;
    }
    detail::check_hip((hipError_t)kk_paged_attention(y, q, k, v, table, lengths, c, p, room, ctx.status + 1, ctx.cus,
                                                     ctx.stream),
                      "kk_paged_attention");
    note(impl, id, kk_paged_attention_route(c, p, ctx.cus));
    return true;
}

const char * kv_append_reason(const KVCacheLayout & c, const KVAppendLayout & p) {
    const char * cache = kv_cache_reason(c);
    if (*cache) return cache;
    if (!known(p.type) || (p.pairs != RotaryPairs::adjacent && p.pairs != RotaryPairs::halves)) return "type";
    if (p.tokens <= 0 || p.sequences <= 0 || p.row_pages <= 0) return "shape";
    if ((int64_t)p.row_pages * c.page_tokens > kMostTokens) return "length";
    if (p.query_heads < 0 || p.query_heads > 1024) return "heads";
    if ((p.query_heads + 2 * (int64_t)c.heads) * (c.width / 8) * p.tokens > INT32_MAX - 1024) return "shape";
    if (p.rotary < 0 || p.rotary > c.width || p.rotary % 2 || (p.rotary > 0 && p.positions <= 0)) return "rotary";
    const int64_t row = (int64_t)c.heads * c.width, q_row = (int64_t)p.query_heads * c.width;
    for (const int64_t s : {p.k_stride, p.v_stride})
        if (s < row || s > kMostStride) return "stride";
    for (const int64_t s : {p.q_stride, p.q_out_stride})
        if (p.query_heads > 0 && (s < q_row || s > kMostStride)) return "stride";
    return "";
}

bool kv_append(Kernel & kernel, int id, void * k_pool, void * v_pool, void * q_out, const void * q, const void * k,
               const void * v, const int * sequence, const int * position, const int * lengths, const int * table,
               const float * cosine, const float * sine, const KVCacheLayout & c, const KVAppendLayout & given) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    KVAppendLayout p = given;
    if (!q) p.query_heads = 0;          // without queries their layout is ignored
    if (*kv_append_reason(c, p) || !k_pool || !v_pool || !k || !v || !table) return false;
    const bool queries = q != nullptr;
    if (queries != (q_out != nullptr) || (queries && p.query_heads == 0)) return false;
    // a token's place: by position (with its sequence), or the newest of each sequence
    if (position ? !sequence : sequence || !lengths || p.tokens > p.sequences) return false;
    if (p.rotary > 0 && (!cosine || !sine)) return false;
    const int bytes = element_bytes(p.type);
    if (!aligned_to(16, {k_pool, v_pool}) || !aligned_to(bytes, {q, q_out, k, v}) ||
        !aligned_to(4, {sequence, position, lengths, table, cosine, sine}))
        return false;
    const int64_t row = (int64_t)c.heads * c.width, q_row = (int64_t)p.query_heads * c.width;
    const Span keys = pool_span(k_pool, c), values = pool_span(v_pool, c);
    const Span k_in = rows_span(k, p.tokens, p.k_stride, row, bytes), v_in = rows_span(v, p.tokens, p.v_stride, row, bytes);
    const Span q_in = rows_span(q, p.tokens, p.q_stride, q_row, bytes);
    const Span out = rows_span(q_out, p.tokens, p.q_out_stride, q_row, bytes);
    const Span rows = ints(table, (int64_t)p.sequences * p.row_pages);
    const Span counts = ints(position ? nullptr : lengths, p.sequences);
    const Span at = ints(position, p.tokens), of = ints(sequence, p.tokens);
    const int64_t angles = p.rotary > 0 ? (int64_t)p.positions * (p.rotary / 2) : 0;
    const Span cosines = ints(cosine, angles), sines = ints(sine, angles);
    if (wraps({keys, values, k_in, v_in, q_in, out, rows, counts, at, of, cosines, sines})) return false;
    if (clash(keys, {values, k_in, v_in, q_in, out, rows, counts, at, of, cosines, sines}) ||
        clash(values, {k_in, v_in, q_in, out, rows, counts, at, of, cosines, sines}) ||
        clash(out, {rows, counts, at, of, cosines, sines}))
        return false;
    // q_out: q itself, rows of its own, or the q columns of rows that hold k and v too
    const bool in_place = queries && q_out == q && p.q_out_stride == p.q_stride;
    if (!in_place && clash(out, {q_in})) return false;
    auto beside = [&](const void * rows_of, int64_t stride) {
        if (!clash(out, rows_span(rows_of, p.tokens, stride, row, bytes))) return true;
        if (!in_place || stride != p.q_stride) return false;
        const uintptr_t a = (uintptr_t)q_out, b = (uintptr_t)rows_of;
        const uintptr_t q_bytes = (uintptr_t)q_row * bytes, row_bytes = (uintptr_t)row * bytes;
        const uintptr_t step = (uintptr_t)stride * bytes, delta = a > b ? a - b : b - a;
        return a > b ? delta >= row_bytes && delta + q_bytes <= step : delta >= q_bytes && delta + row_bytes <= step;
    };
    if (queries && (!beside(k, p.k_stride) || !beside(v, p.v_stride))) return false;
    Kernel::Impl & impl = *kernel.impl_;
    if (!usable(impl, id)) return false;
    detail::DeviceContext & ctx = detail::context(id);
    detail::check_hip((hipError_t)kk_kv_append(k_pool, v_pool, q_out, q, k, v, sequence, position, lengths, table,
                                               cosine, sine, c, p, ctx.status + 1, ctx.stream),
                      "kk_kv_append");
    note(impl, id, "kv_append");
    return true;
}

const char * kv_pages_reason(const KVCacheLayout & c, const KVPagesLayout & p) {
    const char * cache = kv_cache_reason(c);
    if (*cache) return cache;
    if (p.sequences <= 0 || p.row_pages <= 0 || p.layers <= 0 || p.layers > 65535) return "shape";
    if (p.sequences > kMostCounted || c.pages > kMostCounted) return "shape";
    if ((int64_t)p.row_pages * c.page_tokens > kMostTokens) return "length";
    if (p.layers > 1 && (p.layer_stride < pool_elements(c) || p.layer_stride > (INT64_MAX / 4) / p.layers ||
                         p.layer_stride % 8))
        return "stride";
    return "";
}

namespace {

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

bool list_ok(int count, int most) { return count > 0 && count <= most; }

} // namespace

bool kv_reserve(Kernel & kernel, int id, int * table, int * lengths, int * references, const int * rows,
                const int * added, int count, const KVCacheLayout & c, const KVPagesLayout & p) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    if (*kv_pages_reason(c, p) || !table || !lengths || !references || !rows || !added || !list_ok(count, p.sequences))
        return false;
    if (!aligned_to(4, {table, lengths, references, rows, added})) return false;
    if (TableSpans(table, lengths, references, c, p).bad({ints(rows, count), ints(added, count)})) return false;
    Kernel::Impl & impl = *kernel.impl_;
    if (!usable(impl, id)) return false;
    detail::DeviceContext & ctx = detail::context(id);
    void * room = workspace(impl, id, ctx, kk_kv_reserve_workspace_bytes(c, p, count));
    if (!room) return false;
    detail::check_hip((hipError_t)kk_kv_reserve(table, lengths, references, rows, added, count, c, p, room,
                                                ctx.status + 1, ctx.stream),
                      "kk_kv_reserve");
    note(impl, id, "kv_reserve");
    return true;
}

bool kv_fork(Kernel & kernel, int id, void * k, void * v, int * table, int * lengths, int * references,
             const int * parents, const int * children, int count, const KVCacheLayout & c, const KVPagesLayout & p) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    if (*kv_pages_reason(c, p) || !k || !v || !table || !lengths || !references || !parents || !children ||
        !list_ok(count, std::min(p.sequences, 65535)))
        return false;
    if (!aligned_to(16, {k, v}) || !aligned_to(4, {table, lengths, references, parents, children})) return false;
    const Span keys = pool_span(k, c, p), values = pool_span(v, c, p), from = ints(parents, count),
               to = ints(children, count);
    if (TableSpans(table, lengths, references, c, p).bad({keys, values, from, to}) || clash(keys, {values, from, to}) ||
        clash(values, {from, to}))
        return false;
    Kernel::Impl & impl = *kernel.impl_;
    if (!usable(impl, id)) return false;
    detail::DeviceContext & ctx = detail::context(id);
    void * room = workspace(impl, id, ctx, kk_kv_fork_workspace_bytes(p, count));
    if (!room) return false;
    detail::check_hip((hipError_t)kk_kv_fork(k, v, table, lengths, references, parents, children, count, c, p, room,
                                             ctx.status + 1, ctx.stream),
                      "kk_kv_fork");
    note(impl, id, "kv_fork");
    return true;
}

bool kv_free(Kernel & kernel, int id, int * table, int * lengths, int * references, const int * rows, int count,
             const KVCacheLayout & c, const KVPagesLayout & p) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    if (*kv_pages_reason(c, p) || !table || !lengths || !references || !rows || !list_ok(count, p.sequences)) return false;
    if (!aligned_to(4, {table, lengths, references, rows})) return false;
    if (TableSpans(table, lengths, references, c, p).bad({ints(rows, count)})) return false;
    Kernel::Impl & impl = *kernel.impl_;
    if (!usable(impl, id)) return false;
    detail::DeviceContext & ctx = detail::context(id);
    detail::check_hip((hipError_t)kk_kv_free(table, lengths, references, rows, count, c, p, ctx.status + 1, ctx.stream),
                      "kk_kv_free");
    note(impl, id, "kv_free");
    return true;
}

bool kv_compact(Kernel & kernel, int id, void * k, void * v, int * table_out, int * references_out, int * used,
                const int * table, const int * lengths, const int * references, const KVCacheLayout & c,
                const KVPagesLayout & p) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    if (*kv_pages_reason(c, p) || !k || !v || !table_out || !references_out || !used || !table || !lengths || !references)
        return false;
    if (!aligned_to(16, {k, v}) || !aligned_to(4, {table_out, references_out, used, table, lengths, references}))
        return false;
    const Span keys = pool_span(k, c, p), values = pool_span(v, c, p), total = ints(used, 1);
    const TableSpans in(table, lengths, references, c, p);
    const Span rows = ints(table_out, (int64_t)p.sequences * p.row_pages), counts = ints(references_out, c.pages);
    if (in.bad({keys, values, total}) || wraps({rows, counts}) || clash(keys, {values, total}) || clash(values, {total}) ||
        clash(rows, {counts, keys, values, total, in.lengths, in.references}) ||
        clash(counts, {keys, values, total, in.lengths, in.rows}) || (table_out != table && clash(rows, {in.rows})) ||
        (references_out != references && clash(counts, {in.references})))
        return false;
    Kernel::Impl & impl = *kernel.impl_;
    if (!usable(impl, id)) return false;
    detail::DeviceContext & ctx = detail::context(id);
    void * room = workspace(impl, id, ctx, kk_kv_compact_workspace_bytes(c));
    if (!room) return false;
    detail::check_hip((hipError_t)kk_kv_compact(k, v, table_out, references_out, used, table, lengths, references, c, p,
                                                room, ctx.status + 1, ctx.cus, ctx.stream),
                      "kk_kv_compact");
    note(impl, id, "kv_compact");
    return true;
}

bool kv_copy_pages(Kernel & kernel, int id, void * k, void * v, const int * sources, const int * destinations,
                   int count, const KVCacheLayout & c, const KVPagesLayout & p) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    if (*kv_pages_reason(c, p) || !k || !v || !sources || !destinations || !list_ok(count, c.pages)) return false;
    if (!aligned_to(16, {k, v}) || !aligned_to(4, {sources, destinations})) return false;
    const Span keys = pool_span(k, c, p), values = pool_span(v, c, p), from = ints(sources, count),
               to = ints(destinations, count);
    if (wraps({keys, values, from, to}) || clash(keys, {values, from, to}) || clash(values, {from, to})) return false;
    Kernel::Impl & impl = *kernel.impl_;
    if (!usable(impl, id)) return false;
    detail::DeviceContext & ctx = detail::context(id);
    detail::check_hip((hipError_t)kk_kv_copy_pages(k, v, sources, destinations, count, c, p, ctx.status + 1, ctx.cus,
                                                   ctx.stream),
                      "kk_kv_copy_pages");
    note(impl, id, "kv_copy_pages");
    return true;
}

int kv_cache_status(int device) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    if (!detail::device_visible(device)) return -1;
    detail::DeviceContext & ctx = detail::context(device);
    int word = 0;
    detail::check_hip(hipMemcpyAsync(&word, ctx.status + 1, sizeof(word), hipMemcpyDeviceToHost, ctx.stream),
                      "hipMemcpyAsync");
    detail::check_hip(hipStreamSynchronize(ctx.stream), "hipStreamSynchronize");
    if (word) {
        const int zero = 0;
        detail::check_hip(hipMemcpyAsync(ctx.status + 1, &zero, sizeof(zero), hipMemcpyHostToDevice, ctx.stream),
                          "hipMemcpyAsync");
        detail::check_hip(hipStreamSynchronize(ctx.stream), "hipStreamSynchronize");
    }
    return word;
}

const char * logits_reason(const LogitsLayout & p) {
    if (p.rows <= 0 || p.rows > 65535 || p.vocabulary <= 0 || p.vocabulary > (1 << 24)) return "shape";
    for (const int64_t s : {p.logits_stride, p.y_stride})
        if (s < p.vocabulary || s > kMostStride) return "stride";
    for (const int64_t s : {p.history_stride, p.bias_stride})
        if (s < 0 || s > (1 << 24)) return "stride";
    if (p.mask_stride != 0 && (p.mask_stride < (p.vocabulary + 31) / 32 || p.mask_stride > kMostStride)) return "stride";
    return "";
}

bool process_logits(Kernel & kernel, int id, void * y, const void * logits, const float * penalties,
                    const int * history, const int * history_lengths, const int * bias_ids,
                    const float * bias_values, const int * bias_lengths, const uint32_t * mask,
                    const LogitsLayout & p) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    if (*logits_reason(p) || !y || !logits) return false;
    // a stride is a list's room too: 0 would pass over a list that is given
    if (history && (!history_lengths || !penalties || p.history_stride == 0)) return false;
    if (bias_ids && (!bias_values || !bias_lengths || p.bias_stride == 0)) return false;
    if (!aligned_to(4, {y, logits, penalties, history, history_lengths, bias_ids, bias_values, bias_lengths, mask}))
        return false;
    const Span out = rows_span(y, p.rows, p.y_stride, p.vocabulary, 4);
    const Span in = rows_span(logits, p.rows, p.logits_stride, p.vocabulary, 4);
    const Span past = ints(history, (int64_t)p.rows * p.history_stride);
    const Span pasts = ints(history ? history_lengths : nullptr, p.rows);
    const Span factors = ints(history ? penalties : nullptr, (int64_t)3 * p.rows);
    const Span ids = ints(bias_ids, (int64_t)p.rows * p.bias_stride);
    const Span biases = ints(bias_ids ? bias_values : nullptr, (int64_t)p.rows * p.bias_stride);
    const Span counts = ints(bias_ids ? bias_lengths : nullptr, p.rows);
    const Span words = rows_span(mask, p.rows, p.mask_stride, (p.vocabulary + 31) / 32, 4);
    const bool in_place = y == logits && p.y_stride == p.logits_stride;
    if (wraps({out, in, past, pasts, factors, ids, biases, counts, words}) ||
        clash(out, {past, pasts, factors, ids, biases, counts, words}) || (!in_place && clash(out, in)))
        return false;
    Kernel::Impl & impl = *kernel.impl_;
    if (!usable(impl, id)) return false;
    detail::DeviceContext & ctx = detail::context(id);
    detail::check_hip((hipError_t)kk_process_logits(static_cast<float *>(y), static_cast<const float *>(logits), penalties,
                                                    history, history_lengths, bias_ids, bias_values, bias_lengths, mask, p,
                                                    ctx.status + 1, ctx.cus, ctx.stream),
                      "kk_process_logits");
    note(impl, id, "process_logits");
    return true;
}

} // namespace kunlun
