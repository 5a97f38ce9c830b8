// Pages of a paged key-value cache: taken, shared, copied, moved and given back
// by reference counts.
//
// What has to be decided in order (which free page goes to which sequence, which page
// moves where, which of two entries that name one sequence counts) is decided by prefix sums over the reference
// counts and by the lowest place in the caller's list, in the order of page numbers and of that list, so that the
// same calls give the same tables every time: one workgroup for reservations and forks, one a tile of pages for the
// compaction. Counts themselves change by integer atomics. What moves data (rows, pages) follows in a second launch over
// the whole card and is bound by the bytes it copies.
#include "device_common.h"
#include "launch.h"
#include "paged.h"

#include <algorithm>
#include <climits>

namespace {

using kk::kWave;
using kk::PoolView;

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / kWave;
constexpr int kCopyThreads = 256;

struct PagesArgs {
    _Float16 *k, *v;
    int *table, *lengths, *references;
    int *status;
    PoolView pool;
    kk::FastDiv per_row;                 // 16-byte vectors of a token's head
    int64_t layer_stride;
    int sequences, row_pages, layers;
};

// Sum of `v` over the threads before this one; `total` over all of them. Ends
// with a barrier, so it may be called again at once.
template <typename T>
__device__ __forceinline__ T prefix(T v, T &total, T *scratch) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    T sum = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const T other = __shfl_up(sum, o, kWave);
        if (lane >= o) sum += other;
    }
    if (lane == kWave - 1) scratch[wave] = sum;
    __syncthreads();
    T before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        const T x = scratch[w];
        before += w < wave ? x : 0;
        total += x;
    }
    __syncthreads();
    return before + sum - v;
}

// A thread's counts of a tile of N * kPlanThreads pages, in order: -1 past the last page.
template <int N>
struct Counts {
    int r[N];
    int first;
    __device__ __forceinline__ Counts(const int *references, int pages, int p0) : first(p0 + threadIdx.x * N) {
#pragma unroll
        for (int u = 0; u < N; ++u) r[u] = first + u < pages ? references[first + u] : -1;
    }
};
constexpr int kPerThread = 8, kTile = kPerThread * kPlanThreads;

// Writes the free pages of a tile to found[have..wanted) in order; returns how many are had.
template <int N>
__device__ __forceinline__ int free_in_tile(const int *references, int pages, int p0, int have, int wanted, int *found,
                                            int *scratch) {
    const Counts<N> c(references, pages, p0);
    int mine = 0, total;
#pragma unroll
    for (int u = 0; u < N; ++u) mine += c.r[u] == 0;
    int at = have + prefix<int>(mine, total, scratch);
#pragma unroll
    for (int u = 0; u < N; ++u)
        if (c.r[u] == 0) {
            if (at < wanted) found[at] = c.first + u;
            ++at;
        }
    return have + total;
}

// Writes the lowest `wanted` free pages to found[] in order; returns how many there are. A small first tile
// mostly has them (of 4096 pages 100: 4.3 us the launch, in a large tile 6.3); a full pool is
// gone through in large ones.
__device__ __forceinline__ int free_pages(const int *references, int pages, int wanted, int *found, int *scratch) {
    int have = wanted > 0 ? free_in_tile<1>(references, pages, 0, 0, wanted, found, scratch) : 0;
    for (int p0 = kPlanThreads; p0 < pages && have < wanted; p0 += kTile)
        have = free_in_tile<kPerThread>(references, pages, p0, have, wanted, found, scratch);
    __syncthreads();
    return min(have, wanted);
}

__device__ __forceinline__ int pages_of(const PagesArgs &a, int tokens) {
    return a.pool.per_page.div(tokens + a.pool.page_tokens - 1);
}
// A length as it can be: within the row.
__device__ __forceinline__ int length_in_row(const PagesArgs &a, int len) {
    const int64_t most = (int64_t)a.row_pages * a.pool.page_tokens;
    if (len < 0 || len > most) {
        kk::report(a.status, kk::kBadIndex);
        return len < 0 ? 0 : static_cast<int>(most);
    }
    return len;
}
__device__ __forceinline__ int length_of(const PagesArgs &a, int s) { return length_in_row(a, a.lengths[s]); }
__device__ __forceinline__ bool sequence_ok(const PagesArgs &a, int s) {
    if (static_cast<unsigned>(s) < static_cast<unsigned>(a.sequences)) return true;
    kk::report(a.status, kk::kBadIndex);
    return false;
}
// Gives back the first n pages of a row.
__device__ __forceinline__ void release_row(const PagesArgs &a, const int *row, int n) {
    for (int j = threadIdx.x; j < n; j += blockDim.x) {
        const int page = row[j];
        if (static_cast<unsigned>(page) < static_cast<unsigned>(a.pool.pages)) atomicSub(&a.references[page], 1);
        else kk::report(a.status, kk::kBadPage);
    }
}

// Which entry of a list counts for the sequence it names: the first of those that claim it. Claims stand in LDS
// where the table has few sequences, else in the workspace (by LDS instructions instead of flat ones they take as long).
constexpr int kNearClaims = 4096;

__device__ __forceinline__ int *cleared_claims(int *near, int *far, int sequences, const int *list, int count) {
    if (sequences <= kNearClaims) {
        for (int s = threadIdx.x; s < sequences; s += kPlanThreads) near[s] = INT_MAX;
    } else {
        for (int i = threadIdx.x; i < count; i += kPlanThreads)
            if (static_cast<unsigned>(list[i]) < static_cast<unsigned>(sequences)) far[list[i]] = INT_MAX;
    }
    __syncthreads();
    return sequences <= kNearClaims ? near : far;
}
__device__ __forceinline__ void claim(int *claims, int s, int i) { atomicMin(&claims[s], i); }
// After a barrier; past the vector cache, which may hold the word from before the claims.
__device__ __forceinline__ bool claimed(const int *claims, int s, int i) {
    return __hip_atomic_load(&claims[s], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == i;
}

// ---- kv_reserve ----------------------------------------------------------------------------

constexpr int kLeftOut = -1, kRefused = -2;

// For lists that ask for more pages than there are: in list order, whatever still fits is granted; what does not
// takes nothing from those after it. One prefix sum finds the first entry that does not fit, then every later one
// that needs more than is left there goes with it, so the next sum grants at least one more.
__device__ __forceinline__ void refuse_what_does_not_fit(int *need_of, int *first_of, int count, int have, long long *sums,
                                                         int *room) {
    int taken = 0;
    for (int i0 = 0; i0 < count; i0 += kPlanThreads) {
        const int i = i0 + threadIdx.x, left = have - taken, asked = i < count ? need_of[i] : kLeftOut;
        long long need = max(asked, 0), total;
        if (need > left) need = 0;
        for (;;) {
            const long long at = prefix<long long>(need, total, sums);
            if (total <= left) {
                if (i < count) first_of[i] = taken + static_cast<int>(at);
                break;
            }
            const bool first = at <= left && at + need > left;
            if (first) *room = left - static_cast<int>(at);
            __syncthreads();
            if (first || (at > left && need > *room)) need = 0;
        }
        if (asked > 0 && need == 0) need_of[i] = kRefused;
        taken += static_cast<int>(total);
    }
}

__global__ __launch_bounds__(kPlanThreads) void reserve(PagesArgs a, const int *rows, const int *added, int count,
                                                        int *need_of, int *first_of, int *end_of, int *found,
                                                        int *far_claims) {
    __shared__ int scratch[kPlanWaves], near_claims[kNearClaims], room;
    __shared__ long long sums[kPlanWaves];
    int *claims = cleared_claims(near_claims, far_claims, a.sequences, rows, count);
    int64_t wanted = 0;
    for (int i0 = 0; i0 < count; i0 += kPlanThreads) {
        const int i = i0 + threadIdx.x;
        int need = kLeftOut;
        if (i < count && sequence_ok(a, rows[i])) {
            const int64_t len = length_of(a, rows[i]), more = added[i];
            if (more >= 0 && len + more <= (int64_t)a.row_pages * a.pool.page_tokens) {
                end_of[i] = static_cast<int>(len + more);
                need = pages_of(a, end_of[i]) - pages_of(a, static_cast<int>(len));
                claim(claims, rows[i], i);
            } else {
                kk::report(a.status, kk::kBadIndex);
            }
        }
        __syncthreads();
        // a claim of this step never takes a sequence from an earlier one: entries come in order
        if (need >= 0 && !claimed(claims, rows[i], i)) {
            kk::report(a.status, kk::kBadIndex);
            need = kLeftOut;
        }
        long long total;
        const int64_t at = wanted + prefix<long long>(max(need, 0), total, sums);
        if (i < count) {
            need_of[i] = need;
            first_of[i] = static_cast<int>(min<int64_t>(at, a.pool.pages));      // as it is where all are granted
        }
        wanted += total;
    }
    const int have = free_pages(a.references, a.pool.pages, static_cast<int>(min<int64_t>(wanted, a.pool.pages)),
                                found, scratch);
    if (have < wanted) refuse_what_does_not_fit(need_of, first_of, count, have, sums, &room);
    // lengths first, a thread for each listed sequence: 64 sequences in turn 3.9 us the launch, one wave each 4.7
    for (int i = threadIdx.x; i < count; i += kPlanThreads) {
        const int need = need_of[i];
        if (need == kRefused) kk::report(a.status, kk::kNoPage);
        if (need >= 0) a.lengths[rows[i]] = end_of[i];
    }
    __syncthreads();
    // a wave for each listed sequence
    for (int i = threadIdx.x / kWave; i < count; i += kPlanWaves) {
        const int need = need_of[i], first = first_of[i];
        if (need <= 0) continue;
        int *row = a.table + (int64_t)rows[i] * a.row_pages + pages_of(a, end_of[i]) - need;
        for (int j = threadIdx.x % kWave; j < need; j += kWave) {
            const int page = found[first + j];
            row[j] = page;
            a.references[page] = 1;
        }
    }
}

// ---- kv_fork -------------------------------------------------------------------------------

// What the first launch finds out of fork i: the parent's length (-1: left out), and the page that
// its last, not full page is copied to (-1: there is none, -2: no page was free).
struct ForkNote {
    int length, page;
};

// Workgroup 0 finds the pages; workgroup 1 + i copies the parent's row aside (a
// parent may be a child whose row the second launch overwrites).
__global__ __launch_bounds__(kPlanThreads) void fork_plan(PagesArgs a, const int *parents, const int *children,
                                                          int count, ForkNote *notes, int *found, int *rows, int *far_claims) {
    if (blockIdx.x > 0) {
        const int i = blockIdx.x - 1, s = parents[i];
        if (static_cast<unsigned>(s) >= static_cast<unsigned>(a.sequences)) return;
        const int n = pages_of(a, length_of(a, s));
        for (int j = threadIdx.x; j < n; j += kPlanThreads)
            rows[(int64_t)i * a.row_pages + j] = a.table[(int64_t)s * a.row_pages + j];
        return;
    }
    __shared__ int scratch[kPlanWaves], near_claims[kNearClaims];
    int *claims = cleared_claims(near_claims, far_claims, a.sequences, children, count);
    int wanted = 0;
    for (int i0 = 0; i0 < count; i0 += kPlanThreads) {
        const int i = i0 + threadIdx.x;
        int length = -1;
        if (i < count && sequence_ok(a, parents[i]) && sequence_ok(a, children[i])) {
            length = length_of(a, parents[i]);
            claim(claims, children[i], i);
        }
        __syncthreads();
        if (length >= 0 && !claimed(claims, children[i], i)) {
            kk::report(a.status, kk::kBadIndex);
            length = -1;
        }
        const bool part = length > 0 && length % a.pool.page_tokens != 0;
        int total;
        const int at = wanted + prefix<int>(part, total, scratch);
        if (i < count) notes[i] = ForkNote{length, part ? at : -1};
        wanted += total;
    }
    const int have = free_pages(a.references, a.pool.pages, min(wanted, a.pool.pages), found, scratch);
    for (int i = threadIdx.x; i < count; i += kPlanThreads) {
        const int at = notes[i].page;
        if (at < 0) continue;
        notes[i].page = at < have ? found[at] : -2;
        if (at >= have) kk::report(a.status, kk::kNoPage);
    }
}

// Fork i: its first workgroup releases the child's pages and writes the child's row,
// the others copy the tokens of the parent's last page.
__global__ __launch_bounds__(kCopyThreads) void fork_apply(PagesArgs a, const int *children, const ForkNote *notes,
                                                           const int *rows) {
    const int i = blockIdx.y;
    const ForkNote note = notes[i];
    if (note.length < 0) return;
    const int full = a.pool.per_page.div(note.length), rest = note.length - full * a.pool.page_tokens;
    const int *from = rows + (int64_t)i * a.row_pages;
    if (blockIdx.x == 0) {
        const int s = children[i];
        int *row = a.table + (int64_t)s * a.row_pages;
        const int old = pages_of(a, length_of(a, s));
        release_row(a, row, old);
        __syncthreads();
        const int kept = note.page == -2 ? 0 : full;
        for (int j = threadIdx.x; j < a.row_pages; j += kCopyThreads) {
            int page = -1;
            if (j < kept) {
                page = from[j];
                if (static_cast<unsigned>(page) < static_cast<unsigned>(a.pool.pages)) atomicAdd(&a.references[page], 1);
                else kk::report(a.status, kk::kBadPage);
            } else if (j == full && note.page >= 0) {
                page = note.page;
                atomicAdd(&a.references[page], 1);
            }
            row[j] = page;
        }
        if (threadIdx.x == 0) a.lengths[s] = note.page == -2 ? 0 : note.length;
        return;
    }
    if (note.page < 0) return;
    const int page = from[full];
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.pool.pages)) {
        if (blockIdx.x == 1 && threadIdx.x == 0) kk::report(a.status, kk::kBadPage);
        return;
    }
    // 16 bytes a thread: a (layer, pool, head) at a time, its rows of `rest` tokens
    const int row_vectors = a.pool.width / 8, vectors = rest * row_vectors;
    const int blocks = a.layers * 2 * a.pool.heads;
    for (int b = blockIdx.x - 1; b < blocks; b += gridDim.x - 1) {
        const int head = b % a.pool.heads, pool = b / a.pool.heads % 2, layer = b / a.pool.heads / 2;
        _Float16 *base = (pool ? a.v : a.k) + layer * a.layer_stride + head * a.pool.head_stride;
        const _Float16 *src = base + page * a.pool.page_stride;
        _Float16 *dst = base + note.page * a.pool.page_stride;
        for (int x = threadIdx.x; x < vectors; x += kCopyThreads) {
            const int token = a.per_row.div(x), at = x - token * row_vectors;
            const int64_t off = token * a.pool.token_stride + at * 8;
            *reinterpret_cast<uint4 *>(dst + off) = *reinterpret_cast<const uint4 *>(src + off);
        }
    }
}

// ---- kv_free -------------------------------------------------------------------------------

constexpr int kMostFreeGroups = 65536;           // a launch has fewer than 2^32 threads

__global__ __launch_bounds__(kCopyThreads) void free_rows(PagesArgs a, const int *list, int count) {
    __shared__ int length;
    const int64_t most = (int64_t)a.row_pages * a.pool.page_tokens;
    for (int i = blockIdx.x; i < count; i += gridDim.x) {
        const int s = list[i];
        if (static_cast<unsigned>(s) >= static_cast<unsigned>(a.sequences)) {
            if (threadIdx.x == 0) kk::report(a.status, kk::kBadIndex);
            continue;
        }
        // of two entries that name one sequence only one finds its length
        if (threadIdx.x == 0) length = atomicExch(&a.lengths[s], 0);
        __syncthreads();
        const int len = length;
        __syncthreads();
        if (len < 0 || len > most) {
            if (threadIdx.x == 0) kk::report(a.status, kk::kBadIndex);
        }
        const int n = pages_of(a, len < 0 ? 0 : static_cast<int>(min<int64_t>(len, most)));
        int *row = a.table + (int64_t)s * a.row_pages;
        release_row(a, row, n);
        for (int j = threadIdx.x; j < n; j += kCopyThreads) row[j] = -1;
    }
}

// ---- kv_compact ----------------------------------------------------------------------------

// Used pages among the first n, by the whole workgroup.
__device__ __forceinline__ int used_among(const int *references, int n, int *scratch) {
    int mine = 0, total;
    int p = threadIdx.x;
    for (; p + 7 * kPlanThreads < n; p += 8 * kPlanThreads) {
        int r[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) r[u] = references[p + u * kPlanThreads];
#pragma unroll
        for (int u = 0; u < 8; ++u) mine += r[u] > 0;
    }
    for (; p < n; p += kPlanThreads) mine += references[p] > 0;
    prefix<int>(mine, total, scratch);
    return total;
}

// What becomes of a page: a used page below U stays, a hole takes another page's values, a free page above U and a used
// one, whose rank among those is the place of its hole in the list.
constexpr int kStays = -1, kHole = -2;

// U and, one workgroup a tile of pages, the lists of holes below U and of used pages from U up. Each workgroup
// counts all pages for itself, from the L2 (the call on 128 Ki pages of 16 bytes: 226 us where one workgroup goes through
// them in turn, 59 so; 1 Mi pages 1990 and 416).
__global__ __launch_bounds__(kPlanThreads) void compact_plan(const int *references, int pages, int *used_out, int *moves,
                                                             int *holes, int *movers, int *fate) {
    __shared__ int scratch[kPlanWaves];
    __shared__ long long sums[kPlanWaves];
    // a pool of one tile is read once: its counts stay in registers
    const bool one = pages <= kTile;
    const Counts<kPerThread> all(references, one ? pages : 0, 0);
    auto used_here = [&](int n) {
        int mine = 0, total;
#pragma unroll
        for (int u = 0; u < kPerThread; ++u) mine += all.r[u] > 0 && all.first + u < n;
        prefix<int>(mine, total, scratch);
        return total;
    };
    const int used = one ? used_here(pages) : used_among(references, pages, scratch);
    const int used_below = one ? used_here(used) : used_among(references, used, scratch);      // of the first U pages
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *used_out = used;
        *moves = used - used_below;
    }
    for (int p0 = blockIdx.x * kTile; p0 < pages; p0 += gridDim.x * kTile) {
        // holes before a tile are its pages below U less the used ones; used pages from U up likewise
        const int before = p0 > 0 ? used_among(references, p0, scratch) : 0;
        const int n_holes = p0 <= used ? p0 - before : 0, n_movers = p0 <= used ? 0 : before - used_below;
        const Counts<kPerThread> c = one ? all : Counts<kPerThread>(references, pages, p0);
        // both in one prefix: holes in the low half of a word, movers in the high half
        long long mine = 0, total;
#pragma unroll
        for (int u = 0; u < kPerThread; ++u) {
            if (c.first + u < used) mine += c.r[u] <= 0;
            else if (c.r[u] > 0) mine += 1ll << 32;
        }
        const long long prior = prefix<long long>(mine, total, sums);
        int h = n_holes + static_cast<int>(prior), m = n_movers + static_cast<int>(prior >> 32);
#pragma unroll
        for (int u = 0; u < kPerThread; ++u) {
            const int p = c.first + u;
            if (p >= pages) break;
            const bool taken = c.r[u] > 0;
            int what = kStays;
            if (p < used && !taken) {
                holes[h++] = p;
                what = kHole;
            } else if (p >= used && taken) {
                what = m;
                movers[m++] = p;
            }
            fate[p] = what;
        }
    }
}

// Copies page src to dst in one layer's pool; the workgroup takes part `part` of
// `parts`. DENSE: a page is one run of values.
template <bool DENSE>
__device__ __forceinline__ void copy_page(const PagesArgs &a, _Float16 *pool, int src, int dst, int part, int parts) {
    const _Float16 *from = pool + src * a.pool.page_stride;
    _Float16 *to = pool + dst * a.pool.page_stride;
    const int row_vectors = a.pool.width / 8;
    // up to 1024 x 65536 x 32 vectors
    const uint32_t vectors = static_cast<uint32_t>(a.pool.heads) * a.pool.page_tokens * row_vectors;
    for (uint32_t x = part * kCopyThreads + threadIdx.x; x < vectors; x += parts * kCopyThreads) {
        int64_t off = (int64_t)x * 8;
        if constexpr (!DENSE) {
            const uint32_t row = a.per_row.div(x), head = a.pool.per_page.div(row), token = row - head * a.pool.page_tokens;
            off = head * a.pool.head_stride + token * a.pool.token_stride + (x - row * row_vectors) * 8;
        }
        *reinterpret_cast<uint4 *>(to + off) = *reinterpret_cast<const uint4 *>(from + off);
    }
}

// Pages sources[i] -> destinations[i], i < *count: work items are (pair, layer, pool, part).
template <bool DENSE>
__device__ __forceinline__ void copy_pairs(const PagesArgs &a, const int *sources, const int *destinations, int count,
                                           int parts, int item, int step) {
    const int per_pair = a.layers * 2 * parts;
    const int64_t items = (int64_t)count * per_pair;
    for (int64_t x = item; x < items; x += step) {
        const int i = static_cast<int>(x / per_pair), rest = static_cast<int>(x - (int64_t)i * per_pair);
        const int part = rest % parts, pool = rest / parts % 2, layer = rest / parts / 2;
        const int src = sources[i], dst = destinations[i];
        if (src < 0 || dst < 0) continue;
        if (src >= a.pool.pages || dst >= a.pool.pages) {
            if (rest == 0 && threadIdx.x == 0) kk::report(a.status, kk::kBadPage);
            continue;
        }
        copy_page<DENSE>(a, (pool ? a.v : a.k) + layer * a.layer_stride, src, dst, part, parts);
    }
}

template <bool DENSE>
__global__ __launch_bounds__(kCopyThreads) void copy_pages(PagesArgs a, const int *sources, const int *destinations,
                                                           int count, int parts) {
    copy_pairs<DENSE>(a, sources, destinations, count, parts, blockIdx.x, gridDim.x);
}

// The first `groups` workgroups rewrite the table and the counts, the others move the pages.
template <bool DENSE>
__global__ __launch_bounds__(kCopyThreads) void compact_apply(PagesArgs a, const int *table, const int *references,
                                                              int *references_out, const int *used, const int *moves,
                                                              const int *holes, const int *movers, const int *fate,
                                                              int parts, int groups) {
    if (static_cast<int>(blockIdx.x) >= groups) {
        copy_pairs<DENSE>(a, movers, holes, *moves, parts, blockIdx.x - groups, gridDim.x - groups);
        return;
    }
    const int u = *used;
    for (int s = blockIdx.x; s < a.sequences; s += groups) {
        const int n = pages_of(a, length_of(a, s));
        for (int j = threadIdx.x; j < a.row_pages; j += kCopyThreads) {
            const int64_t at = (int64_t)s * a.row_pages + j;
            int page = table[at];
            if (j < n) {
                if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.pool.pages)) {
                    kk::report(a.status, kk::kBadPage);
                } else if (page >= u) {              // a row that names a free page keeps it
                    const int rank = fate[page];
                    page = rank >= 0 ? holes[rank] : page;
                }
            }
            a.table[at] = page;
        }
    }
    // each page's thread writes its own count, a mover's its hole's too; holes' threads touch none
    for (int p = blockIdx.x * kCopyThreads + threadIdx.x; p < a.pool.pages; p += groups * kCopyThreads) {
        const int what = fate[p];
        if (p < u) {
            if (what == kStays && references_out != references) references_out[p] = references[p];
        } else {
            if (what >= 0) references_out[holes[what]] = references[p];
            references_out[p] = 0;
        }
    }
}

PagesArgs args_of(void *k, void *v, int *table, int *lengths, int *references, const kunlun::KVCacheLayout &c,
                  const kunlun::KVPagesLayout &p, int *status) {
    PagesArgs a;
    a.k = static_cast<_Float16 *>(k);
    a.v = static_cast<_Float16 *>(v);
    a.table = table;
    a.lengths = lengths;
    a.references = references;
    a.status = status;
    a.pool = PoolView(c);
    a.per_row = kk::FastDiv(static_cast<uint32_t>(c.width / 8));
    a.layer_stride = p.layer_stride;
    a.sequences = p.sequences;
    a.row_pages = p.row_pages;
    a.layers = p.layers;
    return a;
}

// A page is one run of values, in either order.
bool dense(const kunlun::KVCacheLayout &c) {
    const int64_t w = c.width;
    const bool heads = (c.page_tokens == 1 || c.token_stride == w) && (c.heads == 1 || c.head_stride == w * c.page_tokens);
    const bool tokens = (c.heads == 1 || c.head_stride == w) && (c.page_tokens == 1 || c.token_stride == w * c.heads);
    return heads || tokens;
}

// Workgroups that share a page's values in one pool: 16 KiB each.
int parts_of(const kunlun::KVCacheLayout &c) {
    const int64_t bytes = (int64_t)c.heads * c.page_tokens * c.width * 2;
    return static_cast<int>(std::min<int64_t>(64, (bytes + 16383) / 16384));
}

} // namespace

extern "C" size_t kk_kv_reserve_workspace_bytes(const kunlun::KVCacheLayout &c, const kunlun::KVPagesLayout &p, int count) {
    return ((size_t)3 * count + c.pages + (p.sequences > kNearClaims ? p.sequences : 0)) * sizeof(int);
}
extern "C" int kk_kv_reserve(int *table, int *lengths, int *references, const int *rows, const int *added, int count,
                  const kunlun::KVCacheLayout &c, const kunlun::KVPagesLayout &p, void *workspace, int *status,
                  hipStream_t stream) {
    int *need = static_cast<int *>(workspace), *found = need + 3 * (size_t)count;
    hipLaunchKernelGGL(reserve, dim3(1), dim3(kPlanThreads), 0, stream,
                       args_of(nullptr, nullptr, table, lengths, references, c, p, status), rows, added, count, need,
                       need + count, need + 2 * (size_t)count, found, found + c.pages);
    return hipGetLastError();
}

extern "C" size_t kk_kv_fork_workspace_bytes(const kunlun::KVPagesLayout &p, int count) {
    return (size_t)count * (sizeof(ForkNote) + sizeof(int) + (size_t)p.row_pages * sizeof(int)) +
           (size_t)(p.sequences > kNearClaims ? p.sequences : 0) * sizeof(int);
}
extern "C" int kk_kv_fork(void *k, void *v, int *table, int *lengths, int *references, const int *parents, const int *children,
               int count, const kunlun::KVCacheLayout &c, const kunlun::KVPagesLayout &p, void *workspace, int *status,
               hipStream_t stream) {
    const PagesArgs a = args_of(k, v, table, lengths, references, c, p, status);
    ForkNote *notes = static_cast<ForkNote *>(workspace);
    int *found = reinterpret_cast<int *>(notes + count), *rows = found + count;
    int *far_claims = rows + (size_t)count * p.row_pages;
    hipLaunchKernelGGL(fork_plan, dim3(1 + count), dim3(kPlanThreads), 0, stream, a, parents, children, count, notes,
                       found, rows, far_claims);
    // at most eight (layer, pool, head) blocks of the last page per workgroup
    const int blocks = p.layers * 2 * c.heads, copiers = std::max(1, std::min(blocks, 4096 / count));
    hipLaunchKernelGGL(fork_apply, dim3(1 + copiers, count), dim3(kCopyThreads), 0, stream, a, children, notes, rows);
    return hipGetLastError();
}

extern "C" int kk_kv_free(int *table, int *lengths, int *references, const int *rows, int count, const kunlun::KVCacheLayout &c,
               const kunlun::KVPagesLayout &p, int *status, hipStream_t stream) {
    hipLaunchKernelGGL(free_rows, dim3(std::min(count, kMostFreeGroups)), dim3(kCopyThreads), 0, stream,
                       args_of(nullptr, nullptr, table, lengths, references, c, p, status), rows, count);
    return hipGetLastError();
}

extern "C" size_t kk_kv_compact_workspace_bytes(const kunlun::KVCacheLayout &c) {
    return ((size_t)3 * c.pages + 64) * sizeof(int);
}
extern "C" int kk_kv_compact(void *k, void *v, int *table_out, int *references_out, int *used, const int *table,
                  const int *lengths, const int *references, const kunlun::KVCacheLayout &c,
                  const kunlun::KVPagesLayout &p, void *workspace, int *status, int cus, hipStream_t stream) {
    int *moves = static_cast<int *>(workspace), *holes = moves + 64, *movers = holes + c.pages, *fate = movers + c.pages;
    const int tiles = (c.pages + kTile - 1) / kTile;
    hipLaunchKernelGGL(compact_plan, dim3(std::min(tiles, cus)), dim3(kPlanThreads), 0, stream, references, c.pages, used,
                       moves, holes, movers, fate);
    const PagesArgs a = args_of(k, v, table_out, const_cast<int *>(lengths), nullptr, c, p, status);
    const int groups = std::min(std::max(p.sequences, (c.pages + 4 * kCopyThreads - 1) / (4 * kCopyThreads)), 256);
    const int parts = parts_of(c);
    const dim3 grid(groups + 8 * cus);
    if (dense(c))
        hipLaunchKernelGGL(compact_apply<true>, grid, dim3(kCopyThreads), 0, stream, a, table, references, references_out,
                           used, moves, holes, movers, fate, parts, groups);
    else
        hipLaunchKernelGGL(compact_apply<false>, grid, dim3(kCopyThreads), 0, stream, a, table, references, references_out,
                           used, moves, holes, movers, fate, parts, groups);
    return hipGetLastError();
}

extern "C" int kk_kv_copy_pages(void *k, void *v, const int *sources, const int *destinations, int count,
                     const kunlun::KVCacheLayout &c, const kunlun::KVPagesLayout &p, int *status, int cus,
                     hipStream_t stream) {
    const PagesArgs a = args_of(k, v, nullptr, nullptr, nullptr, c, p, status);
    const int parts = parts_of(c);
    const int64_t items = (int64_t)count * p.layers * 2 * parts;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(items, 8 * cus)));
    if (dense(c))
        hipLaunchKernelGGL(copy_pages<true>, grid, dim3(kCopyThreads), 0, stream, a, sources, destinations, count, parts);
    else
        hipLaunchKernelGGL(copy_pages<false>, grid, dim3(kCopyThreads), 0, stream, a, sources, destinations, count, parts);
    return hipGetLastError();
}
