// The paged key-value cache and the logits step: argument rules, workspaces and
// submission. None of them has a counterpart in the part of the reference's
// header that this library keeps; they follow matmul in submitting without
// waiting and swiglu in refusing arguments by their return value.
#include "kv_rules.h"
#include "launch.h"

#include <cmath>

namespace kunlun {

using namespace rules;

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

bool rules::attention_ok(const void * y, const void * q, const Pools & pools, const int * table, const int * lengths,
                         const KVCacheLayout & c, const PagedAttentionLayout & p) {
    if (*paged_attention_reason(c, p) || !y || !q || !pools.given() || !table || !lengths) return false;
    const int bytes = element_bytes(p.type);
    if (!aligned_to(bytes, {y, q}) || !pools.aligned() || !aligned_to(4, {table, lengths})) return false;
    const int64_t row = (int64_t)p.query_heads * c.width;
    const Span out = rows_span(y, p.sequences, p.y_stride, row, bytes);
    const Span in = rows_span(q, p.sequences, p.q_stride, row, bytes);
    const Span rows = ints(table, (int64_t)p.sequences * p.row_pages), counts = ints(lengths, p.sequences);
    return !wraps({out, in, rows, counts}) && !pools.wrap() && !clash(out, {in, rows, counts}) && !pools.meet(out);
}

bool paged_attention(Kernel & kernel, int id, void * y, const void * q, const void * k, const void * v,
                     const int * table, const int * lengths, const KVCacheLayout & c,
                     const PagedAttentionLayout & p) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    if (*kv_cache_reason(c) || !attention_ok(y, q, Pools(k, v, c), table, lengths, c, p)) return false;
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

bool rules::append_ok(const Pools & pools, const void * q_out, const void * q, const void * k, const void * v,
                      const int * sequence, const int * position, const int * lengths, const int * table,
                      const float * cosine, const float * sine, const KVCacheLayout & c, const KVAppendLayout & p) {
    if (*kv_append_reason(c, p) || !pools.given() || !k || !v || !table) return false;
    const bool queries = q != nullptr;
    if (queries != (q_out != nullptr) || (queries && p.query_heads == 0)) return false;
    // a token's place: by position (with its sequence), or the newest of each sequence
    if (position ? !sequence : sequence || !lengths || p.tokens > p.sequences) return false;
    if (p.rotary > 0 && (!cosine || !sine)) return false;
    const int bytes = element_bytes(p.type);
    if (!pools.aligned() || !aligned_to(bytes, {q, q_out, k, v}) ||
        !aligned_to(4, {sequence, position, lengths, table, cosine, sine}))
        return false;
    const int64_t row = (int64_t)c.heads * c.width, q_row = (int64_t)p.query_heads * c.width;
    const Span k_in = rows_span(k, p.tokens, p.k_stride, row, bytes), v_in = rows_span(v, p.tokens, p.v_stride, row, bytes);
    const Span q_in = rows_span(q, p.tokens, p.q_stride, q_row, bytes);
    const Span out = rows_span(q_out, p.tokens, p.q_out_stride, q_row, bytes);
    const Span rows = ints(table, (int64_t)p.sequences * p.row_pages);
    const Span counts = ints(position ? nullptr : lengths, p.sequences);
    const Span at = ints(position, p.tokens), of = ints(sequence, p.tokens);
    const int64_t angles = p.rotary > 0 ? (int64_t)p.positions * (p.rotary / 2) : 0;
    const Span cosines = ints(cosine, angles), sines = ints(sine, angles);
    if (wraps({k_in, v_in, q_in, out, rows, counts, at, of, cosines, sines}) || pools.wrap()) return false;
    if (pools.meet_each_other() || pools.meet({k_in, v_in, q_in, out, rows, counts, at, of, cosines, sines}) ||
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
    return !queries || (beside(k, p.k_stride) && beside(v, p.v_stride));
}

bool kv_append(Kernel & kernel, int id, void * k_pool, void * v_pool, void * q_out, const void * q, const void * k,
               const void * v, const int * sequence, const int * position, const int * lengths, const int * table,
               const float * cosine, const float * sine, const KVCacheLayout & c, const KVAppendLayout & given) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    KVAppendLayout p = given;
    if (!q) p.query_heads = 0;          // without queries their layout is ignored
    if (*kv_cache_reason(c) || !append_ok(Pools(k_pool, v_pool, c), q_out, q, k, v, sequence, position, lengths, table,
                                          cosine, sine, c, p))
        return false;
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

bool rules::fork_ok(const Pools & pools, const int * table, const int * lengths, const int * references,
                    const int * parents, const int * children, int count, const KVCacheLayout & c, const KVPagesLayout & p) {
    if (*kv_pages_reason(c, p) || !pools.given() || !table || !lengths || !references || !parents || !children ||
        !list_ok(count, std::min(p.sequences, 65535)))
        return false;
    if (!pools.aligned() || !aligned_to(4, {table, lengths, references, parents, children})) return false;
    const Span from = ints(parents, count), to = ints(children, count);
    const TableSpans tables(table, lengths, references, c, p);
    return !tables.bad({from, to}) && !pools.wrap() && !pools.meet_each_other() &&
           !pools.meet({tables.rows, tables.lengths, tables.references, from, to});
}

bool kv_fork(Kernel & kernel, int id, void * k, void * v, int * table, int * lengths, int * references,
             const int * parents, const int * children, int count, const KVCacheLayout & c, const KVPagesLayout & p) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    if (*kv_pages_reason(c, p) || !fork_ok(Pools(k, v, c, p), table, lengths, references, parents, children, count, c, p))
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

bool rules::compact_ok(const Pools & pools, const int * table_out, const int * references_out, const int * used,
                       const int * table, const int * lengths, const int * references, const KVCacheLayout & c,
                       const KVPagesLayout & p) {
    if (*kv_pages_reason(c, p) || !pools.given() || !table_out || !references_out || !used || !table || !lengths ||
        !references)
        return false;
    if (!pools.aligned() || !aligned_to(4, {table_out, references_out, used, table, lengths, references})) return false;
    const Span total = ints(used, 1);
    const TableSpans in(table, lengths, references, c, p);
    const Span rows = ints(table_out, (int64_t)p.sequences * p.row_pages), counts = ints(references_out, c.pages);
    return !in.bad({total}) && !wraps({rows, counts}) && !pools.wrap() && !pools.meet_each_other() &&
           !pools.meet({in.rows, in.lengths, in.references, rows, counts, total}) &&
           !clash(rows, {counts, total, in.lengths, in.references}) && !clash(counts, {total, in.lengths, in.rows}) &&
           (table_out == table || !clash(rows, {in.rows})) &&
           (references_out == references || !clash(counts, {in.references}));
}

bool kv_compact(Kernel & kernel, int id, void * k, void * v, int * table_out, int * references_out, int * used,
                const int * table, const int * lengths, const int * references, const KVCacheLayout & c,
                const KVPagesLayout & p) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    if (*kv_pages_reason(c, p) ||
        !compact_ok(Pools(k, v, c, p), table_out, references_out, used, table, lengths, references, c, p))
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

bool rules::copy_ok(const Pools & pools, const int * sources, const int * destinations, int count,
                    const KVCacheLayout & c, const KVPagesLayout & p) {
    if (*kv_pages_reason(c, p) || !pools.given() || !sources || !destinations || !list_ok(count, c.pages)) return false;
    if (!pools.aligned() || !aligned_to(4, {sources, destinations})) return false;
    const Span from = ints(sources, count), to = ints(destinations, count);
    return !wraps({from, to}) && !pools.wrap() && !pools.meet_each_other() && !pools.meet({from, to});
}

bool kv_copy_pages(Kernel & kernel, int id, void * k, void * v, const int * sources, const int * destinations,
                   int count, const KVCacheLayout & c, const KVPagesLayout & p) {
    std::lock_guard<std::recursive_mutex> lock(detail::mutex());
    if (*kv_pages_reason(c, p) || !copy_ok(Pools(k, v, c, p), sources, destinations, count, c, p)) return false;
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
