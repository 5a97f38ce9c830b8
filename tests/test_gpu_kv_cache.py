"""The paged key-value cache and the logits step on the GPU against plain
computations in 64 bits, at the sizes, layouts and masks where they can go wrong.

Attention's tolerance, per output value: a score's error is at most
e_s = a (2^-21 + width 2^-24) with a = max_t sum_d |scale q_d k_td| (two fp16 parts
hold a factor to 2^-22, sums are F32), a weight's relative error e_w = e_s + 2^-20 (exponential
and its own parts), so numerator and denominator differ by at most e_w + n 2^-24
relative to sum_t w_t |v_t|. F16 outputs are rounded once more (2^-11 relative, 2^-25).
"""
import numpy as np
import pytest

import kunlunk200_lib_amd as kl

pytestmark = pytest.mark.gpu

F32, F16 = kl.InputType.f32, kl.InputType.f16
GUARD = -12345.0


def upload(array):
    array = np.ascontiguousarray(array)
    buffer = kl.Buffer(0, max(array.nbytes, 16))
    if array.nbytes:
        buffer.upload(array)
    return buffer


def finish():
    with kl.runtime_mutex():
        kl.select(0)
        kl.check(kl.wait())


class Cache:
    """Pools in either order with optional padding, kept as [layer][page][head][token][value] float16 views."""

    def __init__(self, rng, pages, page_tokens, heads, width, order="heads", pad=0, layers=1, fill=None):
        w = width + 8 * pad
        if order == "heads":
            strides = (page_tokens * w * heads + 16 * pad, page_tokens * w, w)
        else:
            strides = (page_tokens * w * heads + 16 * pad, w, w * heads)
        self.layout = kl.KVCacheLayout(pages, page_tokens, heads, width, *strides)
        self.layers, self.layer = layers, strides[0] * pages
        assert kl.kv_cache_reason(self.layout) == ""
        self.flat = []
        for _ in range(2):
            x = rng.standard_normal(self.layer * layers).astype(np.float16)
            if fill is not None:
                x[:] = fill
            self.flat.append(x)
        self.k, self.v = (self.view(x) for x in self.flat)
        self.buffers = None

    def view(self, flat):
        c = self.layout
        return np.lib.stride_tricks.as_strided(
            flat, (self.layers, c.pages, c.heads, c.page_tokens, c.width),
            (2 * self.layer, 2 * c.page_stride, 2 * c.head_stride, 2 * c.token_stride, 2))

    def upload(self):
        self.buffers = [upload(x) for x in self.flat]
        return [b.data for b in self.buffers]

    def download(self):
        flat = [b.download(x.shape, np.float16) for b, x in zip(self.buffers, self.flat)]
        return flat, [self.view(x) for x in flat]


def table_of(rng, lengths, page_tokens, pages, row_pages, rest=-1):
    ids = list(rng.permutation(pages))
    table = np.full((len(lengths), row_pages), rest, np.int32)
    for s, n in enumerate(lengths):
        for j in range(-(-n // page_tokens)):
            table[s, j] = ids.pop()
    return table


def gold_attention(cache, table, lengths, q, window, scale, skip=()):
    """(y, tolerance without the output's rounding); `skip`: page ids whose tokens are left out."""
    c = cache.layout
    n, query_heads, width = q.shape
    group = query_heads // c.heads
    y, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s, length in enumerate(lengths):
        t = np.arange(max(0, length - window) if window else 0, length)
        page = table[s, t // c.page_tokens]
        keep = ~np.isin(page, list(skip))
        t, page = t[keep], page[keep]
        if not len(t):
            continue
        for h in range(query_heads):
            k = cache.k[0, page, h // group, t % c.page_tokens].astype(np.float64)
            v = cache.v[0, page, h // group, t % c.page_tokens].astype(np.float64)
            qh = q[s, h].astype(np.float64)
            with np.errstate(invalid="ignore"):
                score = (k @ qh) * scale
            if np.all(score == -np.inf):
                continue
            p = np.exp(score - score.max())
            y[s, h] = p @ v / p.sum()
            finite = np.isfinite(score)
            a = np.abs(k[finite] * qh).sum(1).max(initial=0.0) * abs(scale)
            e_w = a * (2.0 ** -21 + width * 2.0 ** -24) + 2.0 ** -20
            tol[s, h] = (2 * e_w + 2 * len(t) * 2.0 ** -24) * (p @ np.abs(v)) / p.sum()
    return y, tol


def run_attention(cache, table, lengths, q, window=0, scale=None, longest=None, pad=0, kernel=None):
    n, query_heads, width = q.shape
    scale = width ** -0.5 if scale is None else scale
    longest = max(1, max(lengths)) if longest is None else longest
    kind = F16 if q.dtype == np.float16 else F32
    row = query_heads * width
    rows = np.full((n, row + pad), GUARD, q.dtype)
    rows[:, :row] = q.reshape(n, row)
    out = np.full((n, row + pad), GUARD, q.dtype)
    k, v = cache.upload()
    bufs = [upload(x) for x in (out, rows, np.asarray(table, np.int32), np.asarray(lengths, np.int32))]
    call = kl.PagedAttentionLayout(n, query_heads, longest, window, table.shape[1], row + pad, row + pad, scale, kind)
    assert kl.paged_attention_reason(cache.layout, call) == ""
    kernel = kernel or kl.Kernel()
    assert kl.paged_attention(kernel, 0, bufs[0].data, bufs[1].data, k, v, bufs[2].data, bufs[3].data, cache.layout, call)
    finish()
    y = bufs[0].download(out.shape, q.dtype)
    assert np.all(y[:, row:] == np.array(GUARD, q.dtype)), "wrote between rows"
    flat, _ = cache.download()
    assert all(np.array_equal(a.view(np.uint16), b.view(np.uint16)) for a, b in zip(flat, cache.flat)), "cache changed"
    return y[:, :row].reshape(q.shape), kernel.route


def check(y, gold, tol):
    if y.dtype == np.float16:
        tol = tol + 2.0 ** -11 * np.abs(gold) * 1.01 + 2.0 ** -25
    err = np.abs(y.astype(np.float64) - gold)
    assert np.all(np.isfinite(y))
    assert np.all(err <= tol + 1e-37), f"worst {np.max(err / (tol + 1e-37)):.3g} of the tolerance"


# lengths, heads, query heads, width, tokens of a page, window, F16, order, padding
ATTENTION = [
    ([1], 1, 1, 8, 1, 0, False, "heads", 0),
    ([1, 0, 2], 2, 2, 64, 16, 0, False, "heads", 0),
    ([31, 32, 33, 0, 16, 17], 4, 4, 128, 16, 0, False, "heads", 0),
    ([127, 128, 129, 255, 256, 257, 5, 1], 8, 32, 128, 32, 0, True, "tokens", 0),
    ([300, 77], 5, 15, 80, 20, 0, False, "heads", 1),
    ([300, 77], 5, 15, 80, 20, 100, True, "tokens", 1),
    ([513], 2, 18, 96, 3, 0, False, "heads", 0),            # 9 query heads a key-value head: two column tiles
    ([700, 3], 1, 16, 128, 64, 0, True, "heads", 0),
    ([640], 1, 71, 64, 16, 0, False, "tokens", 0),          # three launches' worth of tiles of 16 heads
    ([260, 261], 2, 2, 256, 16, 0, False, "heads", 0),
    ([130], 3, 27, 192, 100, 0, True, "heads", 1),          # two tiles of 8 heads at two halves of 128 values
    ([90], 1, 1, 24, 7, 0, False, "tokens", 1),
    ([90], 2, 4, 40, 4, 0, True, "heads", 0),
    ([90], 2, 4, 72, 12, 33, False, "heads", 0),
    ([90], 2, 4, 104, 1, 0, False, "heads", 0),
    ([90, 12], 2, 2, 136, 8, 0, False, "heads", 0),
    ([150], 1, 9, 200, 16, 64, False, "tokens", 0),
    ([5000, 4999, 10], 1, 4, 128, 2048, 0, False, "heads", 0),
    ([9001, 1, 4096, 0], 2, 8, 64, 16, 0, False, "heads", 0),
    ([9001, 700, 64], 2, 8, 128, 16, 1, False, "heads", 0),  # the newest token alone
    ([3000, 65], 2, 8, 128, 16, 64, True, "heads", 0),
    ([20000], 8, 8, 128, 128, 0, True, "heads", 0),
    ([70, 16], 2, 8, 96, 16, 0, False, "heads", 0),
    ([70, 16], 2, 2, 192, 32, 40, False, "tokens", 0),
    ([70, 16], 1, 12, 56, 16, 0, True, "heads", 0),
    ([2100, 300], 1, 20, 128, 48, 500, False, "heads", 1),
]


@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention(gpu, case):
    lengths, heads, query_heads, width, page_tokens, window, half, order, pad = ATTENTION[case]
    rng = np.random.default_rng(1000 + case)
    row_pages = -(-max(lengths) // page_tokens) + 2
    pages = sum(-(-n // page_tokens) for n in lengths) + 2
    cache = Cache(rng, pages, page_tokens, heads, width, order, pad)
    # entries past a sequence's pages are not read, whatever they hold
    table = table_of(rng, lengths, page_tokens, pages, row_pages, rest=2 ** 30)
    q = (rng.standard_normal((len(lengths), query_heads, width)) * 2).astype(np.float16 if half else np.float32)
    # what no token owns may be anything: NaN and Inf past each end and in free pages
    owned = np.zeros((pages, page_tokens), bool)
    for s, n in enumerate(lengths):
        t = np.arange(n)
        owned[table[s, t // page_tokens], t % page_tokens] = True
    for pool in (cache.k, cache.v):
        pool[0].transpose(0, 2, 1, 3)[~owned] = np.nan
    cache.v[0].transpose(0, 2, 1, 3)[~owned, :, ::2] = np.inf
    y, route = run_attention(cache, table, lengths, q, window, pad=3 * pad)
    gold, tol = gold_attention(cache, table, lengths, q, window, width ** -0.5)
    check(y, gold, tol)
    again, _ = run_attention(cache, table, lengths, q, window, pad=3 * pad)
    assert np.array_equal(y, again), "the same call gives other bits"
    assert gpu.kv_cache_status(0) == 0
    # a looser bound on the lengths splits otherwise and gives the same within the tolerance
    y, _ = run_attention(cache, table, lengths, q, window, longest=row_pages * page_tokens)
    check(y, gold, tol)


def test_attention_splits(gpu):
    rng = np.random.default_rng(5)
    cache = Cache(rng, 600, 16, 1, 64)
    lengths = [9000]
    table = table_of(rng, lengths, 16, 600, 563)
    q = rng.standard_normal((1, 1, 64)).astype(np.float32)
    _, route = run_attention(cache, table, lengths, q)
    assert route == "paged_attention_split"
    table = table_of(rng, [64], 16, 600, 563)
    _, route = run_attention(cache, table, [64], q)
    assert route == "paged_attention"


@pytest.mark.parametrize("scale", [0.0, -0.5, 1e-20, 30.0])
@pytest.mark.parametrize("size", [1e-30, 1.0, 1e4])
def test_attention_scales(gpu, scale, size):
    rng = np.random.default_rng(6)
    cache = Cache(rng, 20, 16, 2, 64)
    table = table_of(rng, [200], 16, 20, 13)
    q = (rng.standard_normal((1, 4, 64)) * size).astype(np.float32)
    y, _ = run_attention(cache, table, [200], q, scale=scale)
    gold, tol = gold_attention(cache, table, [200], q, 0, float(np.float32(scale)))
    # scores of several thousand: their error makes the tolerance more than the values
    check(y, gold, np.minimum(tol, 20.0))


@pytest.mark.parametrize("half", [False, True])
def test_attention_infinite_keys(gpu, half):
    """-Inf scores weigh nothing, wherever they stand; a row of nothing else gives zeros."""
    rng = np.random.default_rng(7)
    lengths = [150, 40, 1]
    cache = Cache(rng, 20, 16, 2, 64)
    table = table_of(rng, lengths, 16, 20, 12)
    q = np.abs(rng.standard_normal((3, 4, 64)) + 0.1).astype(np.float16 if half else np.float32)
    for s, t in ((0, 0), (0, 31), (0, 100), (0, 149)):
        cache.k[0, table[s, t // 16], :, t % 16, 5] = -np.inf
    for s in (1, 2):
        for t in range(lengths[s]):
            cache.k[0, table[s, t // 16], 1, t % 16, 7] = -np.inf       # all keys of head 1
    y, _ = run_attention(cache, table, lengths, q)
    gold, tol = gold_attention(cache, table, lengths, q, 0, 0.125)
    assert np.all(gold[1:, 2:] == 0)
    check(y, gold, tol)


@pytest.mark.parametrize("width,longest", [(64, 150), (128, 2816)])
def test_attention_infinite_values(gpu, width, longest):
    """An infinite value gives its infinity to the output's column, two of both signs what is not a number."""
    rng = np.random.default_rng(11)
    lengths = [150, 40, 1, 0, 70, 33, 1, 2]
    cache = Cache(rng, 30, 16, 8, width)
    table = table_of(rng, lengths, 16, 30, 176)
    q = rng.standard_normal((8, 8, width)).astype(np.float32)
    for t, d, x in ((0, 3, np.inf), (77, 4, -np.inf), (5, 5, np.inf), (149, 5, -np.inf)):
        cache.v[0, table[0, t // 16], 1, t % 16, d] = x
    cache.v[0, table[2, 0], 6, 0, 9] = -np.inf
    y, _ = run_attention(cache, table, lengths, q, longest=longest)
    with np.errstate(invalid="ignore"):
        gold, tol = gold_attention(cache, table, lengths, q, 0, width ** -0.5)
    assert gold[0, 1, 3] == np.inf and gold[0, 1, 4] == -np.inf and np.isnan(gold[0, 1, 5]) and gold[2, 6, 9] == -np.inf
    odd = ~np.isfinite(gold)
    assert np.array_equal(y[odd], gold[odd].astype(np.float32), equal_nan=True)
    check(np.where(odd, 0, y), np.where(odd, 0, gold), np.where(odd, 0, tol))


def test_attention_not_a_number(gpu):
    """NaN among the keys or the query reaches the heads that read it and no others."""
    rng = np.random.default_rng(8)
    cache = Cache(rng, 20, 16, 2, 64)
    table = table_of(rng, [150, 150], 16, 20, 10)
    q = rng.standard_normal((2, 4, 64)).astype(np.float32)
    cache.k[0, table[0, 3], 1, 4, 9] = np.nan
    q[1, 0, 3] = np.nan
    y, _ = run_attention(cache, table, [150, 150], q)
    assert np.all(np.isnan(y[0, 2:])) and np.all(np.isnan(y[1, 0]))
    gold, tol = gold_attention(cache, table, [150, 150], q, 0, 0.125)
    check(y[0, :2], gold[0, :2], tol[0, :2])
    check(y[1, 1:], gold[1, 1:], tol[1, 1:])


def test_attention_reports(gpu):
    """Pages outside the pool are left out, lengths past the bound cut, and both reported once."""
    rng = np.random.default_rng(9)
    lengths = [150, 400]
    cache = Cache(rng, 40, 16, 2, 64)
    table = table_of(rng, lengths, 16, 40, 26)
    q = rng.standard_normal((2, 4, 64)).astype(np.float32)
    assert gpu.kv_cache_status(0) == 0
    bad = table.copy()
    bad[0, 2], bad[1, 7] = 40, -1
    y, _ = run_attention(cache, bad, lengths, q)
    assert gpu.kv_cache_status(0) == kl.KV_BAD_PAGE
    assert gpu.kv_cache_status(0) == 0
    safe = bad.copy()
    safe[0, 2] = -1
    gold, tol = gold_attention(cache, safe, lengths, q, 0, 0.125, skip=(-1,))
    check(y, gold, tol)
    y, _ = run_attention(cache, table, [150, 400], q, longest=300)
    assert gpu.kv_cache_status(0) == kl.KV_BAD_INDEX
    gold, tol = gold_attention(cache, table, [150, 300], q, 0, 0.125)
    check(y, gold, tol)
    y, _ = run_attention(cache, table, [150, -3], q)
    assert gpu.kv_cache_status(0) == kl.KV_BAD_INDEX
    assert np.all(y[1] == 0)


def test_window_pages_given_back(gpu):
    """Pages before the window may be gone from the row."""
    rng = np.random.default_rng(10)
    cache = Cache(rng, 40, 16, 2, 64)
    table = table_of(rng, [500], 16, 40, 32)
    q = rng.standard_normal((1, 4, 64)).astype(np.float32)
    gold, tol = gold_attention(cache, table, [500], q, 90, 0.125)
    table[0, :(500 - 90) // 16] = -1
    y, _ = run_attention(cache, table, [500], q, window=90)
    check(y, gold, tol)
    assert gpu.kv_cache_status(0) == 0


def test_offsets_past_32_bits(gpu):
    """Pages more than 4 GiB apart: attention, append and copies reach them."""
    rng = np.random.default_rng(11)
    pages, pt, heads, width = 3, 16, 2, 64
    stride = (1 << 31) + 1024                                     # elements
    layout = kl.KVCacheLayout(pages, pt, heads, width, stride, pt * width, width)
    small = Cache(rng, pages, pt, heads, width)
    n = heads * pt * width
    size = ((pages - 1) * stride + n) * 2
    with kl.Buffer(0, size) as kb, kl.Buffer(0, size) as vb:
        for p in range(pages):
            kb.upload(small.flat[0][p * n:(p + 1) * n], offset=2 * p * stride)
            vb.upload(small.flat[1][p * n:(p + 1) * n], offset=2 * p * stride)
        table = np.array([[2, 0, 1]], np.int32)
        lengths = [41]
        q = rng.standard_normal((1, 4, width)).astype(np.float32)
        bufs = [upload(x) for x in (q, q, table, np.array(lengths, np.int32))]
        call = kl.PagedAttentionLayout(1, 4, 41, 0, 3, 256, 256, 0.125, F32)
        kernel = kl.Kernel()
        assert kl.paged_attention(kernel, 0, bufs[0].data, bufs[1].data, kb.data, vb.data, bufs[2].data,
                                  bufs[3].data, layout, call)
        finish()
        y = bufs[0].download(q.shape, np.float32)
        gold, tol = gold_attention(small, table, lengths, q, 0, 0.125)
        check(y, gold, tol)
        new = rng.standard_normal((1, 2 * heads * width)).astype(np.float32)
        place = [upload(x) for x in (new, np.array([0], np.int32), np.array([3], np.int32))]
        append = kl.KVAppendLayout(1, 1, 3, 0, 0, 256, 256, 0, 0, 0, kl.RotaryPairs.adjacent, F32)
        assert kl.kv_append(kernel, 0, kb.data, vb.data, None, None, place[0].data, place[0].data + 512, place[1].data,
                            place[2].data, None, bufs[2].data, None, None, layout, append)
        pair = [upload(np.array([x], np.int32)) for x in (2, 1)]
        assert kl.kv_copy_pages(kernel, 0, kb.data, vb.data, pair[0].data, pair[1].data, 1, layout,
                                kl.KVPagesLayout(1, 3, 1, 0))
        finish()
        for p in (2, 1):
            k = kb.download((heads, pt, width), np.float16, offset=2 * p * stride)
            want = small.k[0, 2].copy()
            want[:, 3] = new[0, :128].reshape(2, 64).astype(np.float16)
            assert np.array_equal(k, want)


# --- kv_append --------------------------------------------------------------------------

def turned(x, cosine, sine, pairs):
    """x [tokens, heads, width] in 64 bits, its first values turned."""
    y, half = x.astype(np.float64), cosine.shape[1]
    c, s = cosine.astype(np.float64)[:, None], sine.astype(np.float64)[:, None]
    first = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if pairs == kl.RotaryPairs.adjacent else \
        (slice(0, half), slice(half, 2 * half))
    a, b = y[..., first[0]].copy(), y[..., first[1]].copy()
    y[..., first[0]], y[..., first[1]] = a * c - b * s, a * s + b * c
    return y


# tokens of each sequence (from each past), heads, query heads, width, page tokens, rotary, pairs, F16, order, pad, offset
APPEND = [
    ([1], 1, 1, 8, 1, 8, 0, False, "heads", 0, 0),
    ([1, 1, 1, 1], 8, 32, 128, 16, 128, 0, False, "heads", 0, 0),
    ([33, 1, 70], 4, 8, 128, 16, 128, 1, False, "heads", 0, 0),
    ([33, 1, 70], 4, 8, 128, 16, 64, 1, True, "tokens", 1, 0),
    ([200], 5, 15, 80, 20, 80, 0, True, "heads", 0, 0),
    ([17], 2, 2, 64, 3, 6, 0, False, "heads", 0, 0),           # a part that ends inside a thread's values
    ([17], 2, 2, 64, 3, 20, 1, False, "tokens", 1, 0),
    ([17], 2, 2, 64, 3, 64, 1, False, "heads", 0, 1),          # rows off 16 bytes
    ([17], 2, 2, 64, 3, 64, 0, True, "heads", 0, 1),
    ([40, 3], 2, 4, 64, 16, 0, 0, False, "heads", 0, 0),       # not turned
    ([9], 1, 3, 256, 16, 256, 1, False, "heads", 0, 0),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(gpu, case, in_place):
    each, heads, query_heads, width, pt, rotary, pairs, half, order, pad, offset = APPEND[case]
    pairs = kl.RotaryPairs(pairs)
    rng = np.random.default_rng(2000 + case)
    n, tokens = len(each), sum(each)
    past = rng.integers(0, 50, n)
    lengths = past + np.array(each)
    row_pages = -(-int(lengths.max()) // pt) + 1
    pages = int(sum(-(-lengths // pt))) + 2
    cache = Cache(rng, pages, pt, heads, width, order, pad)
    table = table_of(rng, lengths, pt, pages, row_pages)
    sequence = np.repeat(np.arange(n), each).astype(np.int32)
    position = np.concatenate([np.arange(p, p + e) for p, e in zip(past, each)]).astype(np.int32)
    mix = rng.permutation(tokens)
    sequence, position = sequence[mix], position[mix]
    dtype = np.float16 if half else np.float32
    row = (query_heads + 2 * heads) * width
    stride = row + (offset or 0)
    rows = (rng.standard_normal((tokens, stride)) * 3).astype(dtype)
    positions = int(lengths.max())
    angle = np.arange(positions)[:, None] / 10000.0 ** (np.arange(rotary // 2) / max(1, rotary // 2))[None, :]
    cosine, sine = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    k_pool, v_pool = cache.upload()
    size = rows.itemsize
    flat = np.concatenate([np.zeros(offset, dtype), rows.ravel()])
    rows_b = upload(flat)
    at = rows_b.data + offset * size
    out = np.full(tokens * (query_heads * width + 8), GUARD, dtype)
    out_b = upload(out)
    bufs = [upload(x) for x in (sequence, position, table, cosine, sine)]
    q_stride = stride if in_place else query_heads * width + 8
    call = kl.KVAppendLayout(tokens, n, row_pages, query_heads, stride, stride, stride, q_stride, rotary, positions,
                             pairs, F16 if half else F32)
    assert kl.kv_append_reason(cache.layout, call) == ""
    kernel = kl.Kernel()
    k_at, v_at = at + query_heads * width * size, at + (query_heads + heads) * width * size
    assert kl.kv_append(kernel, 0, k_pool, v_pool, at if in_place else out_b.data, at, k_at, v_at, bufs[0].data,
                        bufs[1].data, None, bufs[2].data, bufs[3].data if rotary else None,
                        bufs[4].data if rotary else None, cache.layout, call)
    finish()
    assert kernel.route == "kv_append" and gpu.kv_cache_status(0) == 0
    x = rows[:, :row].reshape(tokens, -1, width)
    x = [x[:, :query_heads], x[:, query_heads:query_heads + heads], x[:, query_heads + heads:]]
    gold_q, gold_k = (turned(a, cosine[position], sine[position], pairs) for a in x[:2])
    # a sum of two products, one rounding in F32 each: 2^-23 of their sizes
    room = 2.0 ** -23 * 2 * np.abs(rows[:, :row].astype(np.float64)).max()
    rows_after = rows_b.download(flat.shape, dtype)[offset:].reshape(rows.shape)
    if in_place:
        q = rows_after[:, :query_heads * width]
        assert np.array_equal(rows_after[:, query_heads * width:], rows[:, query_heads * width:]), "k or v changed"
    else:
        q = out_b.download((tokens, query_heads * width + 8), dtype)
        assert np.all(q[:, -8:] == np.array(GUARD, dtype)) and np.array_equal(rows_after, rows)
        q = q[:, :-8]
    q = q.reshape(tokens, query_heads, width).astype(np.float64)
    step = 2.0 ** -11 if half else 2.0 ** -24
    assert np.all(np.abs(q - gold_q) <= room + step * np.abs(gold_q) + 2.0 ** -25)
    before = [y.copy() for y in (cache.k, cache.v)]
    flats, (k, v) = cache.download()
    page, slot = table[sequence, position // pt], position % pt
    assert np.all(np.abs(k[0, page, :, slot].astype(np.float64) - gold_k) <= room + 2.0 ** -11 * np.abs(gold_k) + 2.0 ** -25)
    assert np.array_equal(v[0, page, :, slot], x[2].astype(np.float16))
    before[0][0, page, :, slot], before[1][0, page, :, slot] = k[0, page, :, slot], v[0, page, :, slot]
    assert np.array_equal(before[0], k) and np.array_equal(before[1], v), "other tokens changed"
    for flat_after, flat_before, view in zip(flats, cache.flat, (k, v)):
        flat_before = flat_before.copy()
        cache.view(flat_before)[:] = view
        assert np.array_equal(flat_after, flat_before), "wrote into the padding"


def test_append_newest_and_left_out(gpu):
    """Without positions: token i is the newest of sequence i. Negative places are left out, impossible ones reported."""
    rng = np.random.default_rng(21)
    cache = Cache(rng, 12, 4, 2, 64)
    lengths = np.array([5, 0, 9, 1], np.int32)
    table = table_of(rng, lengths, 4, 12, 4)
    rows = rng.standard_normal((4, 256)).astype(np.float32)
    k_pool, v_pool = cache.upload()
    r, t, l = upload(rows), upload(table), upload(lengths)
    call = kl.KVAppendLayout(4, 4, 4, 0, 0, 256, 256, 0, 0, 0, kl.RotaryPairs.adjacent, F32)
    kernel = kl.Kernel()
    assert kl.kv_append(kernel, 0, k_pool, v_pool, None, None, r.data, r.data + 512, None, None, l.data, t.data, None,
                        None, cache.layout, call)
    _, (k, v) = cache.download()
    want = cache.k.copy()
    for s in (0, 2, 3):
        at = lengths[s] - 1
        want[0, table[s, at // 4], :, at % 4] = rows[s, :128].reshape(2, 64).astype(np.float16)
    assert np.array_equal(k, want) and gpu.kv_cache_status(0) == 0
    sequence, position = np.array([-1, 4, 0, 2], np.int32), np.array([0, 0, 16, -7], np.int32)
    s, p = upload(sequence), upload(position)
    cache.upload()
    k_pool, v_pool = (b.data for b in cache.buffers)
    assert kl.kv_append(kernel, 0, k_pool, v_pool, None, None, r.data, r.data + 512, s.data, p.data, None, t.data, None,
                        None, cache.layout, call)
    assert gpu.kv_cache_status(0) == kl.KV_BAD_INDEX
    flat, _ = cache.download()
    assert all(np.array_equal(a, b) for a, b in zip(flat, cache.flat))
    table[0, 0], table[2, 2] = 12, -1
    t.upload(table)
    sequence, position = np.array([0, 2, 0, 3], np.int32), np.array([3, 8, 4, 0], np.int32)
    s.upload(sequence)
    p.upload(position)
    assert kl.kv_append(kernel, 0, k_pool, v_pool, None, None, r.data, r.data + 512, s.data, p.data, None, t.data, None,
                        None, cache.layout, call)
    assert gpu.kv_cache_status(0) == kl.KV_BAD_PAGE
    _, (k, _) = cache.download()
    want = cache.k.copy()
    for i in (2, 3):
        want[0, table[sequence[i], position[i] // 4], :, position[i] % 4] = rows[i, :128].reshape(2, 64).astype(np.float16)
    assert np.array_equal(k, want)


# --- pages ------------------------------------------------------------------------------

class Book:
    """The page operations' rules, plainly: tables, lengths, counts and pools on the host."""

    def __init__(self, rng, sequences, row_pages, pages, pt, heads=2, width=16, layers=2, order="heads", pad=0):
        self.cache = Cache(rng, pages, pt, heads, width, order, pad, layers)
        self.table = np.full((sequences, row_pages), -1, np.int32)
        self.lengths = np.zeros(sequences, np.int32)
        self.references = np.zeros(pages, np.int32)
        self.pages = kl.KVPagesLayout(sequences, row_pages, layers, self.cache.layer)
        self.pt = pt

    def upload(self):
        self.pools = self.cache.upload()
        self.b = [upload(x) for x in (self.table, self.lengths, self.references)]
        self.p = [b.data for b in self.b]
        self.kernel = kl.Kernel()
        self.want = [x.copy() for x in (self.cache.k, self.cache.v)]

    def held(self, n):
        return -(-int(n) // self.pt)

    def reserve(self, rows, added):
        free, taken, used = list(np.flatnonzero(self.references == 0)), 0, 0
        for r, a in zip(rows, added):
            held, need = self.held(self.lengths[r]), self.held(self.lengths[r] + a)
            first, taken = taken, taken + need - held
            if need > self.table.shape[1]:
                taken = first
                continue
            if need > held and taken > len(free):
                continue
            for j in range(held, need):
                page = free[first + j - held]
                self.table[r, j], self.references[page] = page, 1
            self.lengths[r] += a

    def fork(self, parents, children):
        free = list(np.flatnonzero(self.references == 0))
        rows, lengths = self.table[parents].copy(), self.lengths[parents].copy()
        for c in children:
            for j in range(self.held(self.lengths[c])):
                self.references[self.table[c, j]] -= 1
        before = [x.copy() for x in self.want]
        for i, c in enumerate(children):
            full, rest = divmod(int(lengths[i]), self.pt)
            self.table[c], self.lengths[c] = -1, 0
            if rest and not free:
                continue
            self.table[c, :full], self.lengths[c] = rows[i, :full], lengths[i]
            np.add.at(self.references, rows[i, :full], 1)
            if rest:
                page = free.pop(0)
                self.table[c, full], self.references[page] = page, 1
                for pool, old in zip(self.want, before):
                    pool[:, page, :, :rest] = old[:, rows[i, full], :, :rest]

    def free(self, rows):
        for r in rows:
            for j in range(self.held(self.lengths[r])):
                self.references[self.table[r, j]] -= 1
            self.table[r], self.lengths[r] = -1, 0

    def compact(self):
        used = int((self.references > 0).sum())
        to = np.arange(len(self.references))
        holes = [p for p in range(used) if self.references[p] == 0]
        movers = [p for p in range(used, len(to)) if self.references[p] > 0]
        for h, m in zip(holes, movers):
            to[m] = h
            for pool in self.want:
                pool[:, h] = pool[:, m]
            self.references[h], self.references[m] = self.references[m], 0
        for s, n in enumerate(self.lengths):
            held = self.held(n)
            self.table[s, :held] = to[self.table[s, :held]]
        return used

    def check(self, status=0):
        finish()
        assert kl.kv_cache_status(0) == status
        got = [b.download(x.shape, np.int32) for b, x in zip(self.b, (self.table, self.lengths, self.references))]
        assert np.array_equal(got[1], self.lengths)
        assert np.array_equal(got[0], self.table)
        assert np.array_equal(got[2], self.references)
        flats, views = self.cache.download()
        for flat, before, view, want in zip(flats, self.cache.flat, views, self.want):
            assert np.array_equal(view, want)
            before = before.copy()
            self.cache.view(before)[:] = want
            assert np.array_equal(flat, before), "wrote into the padding"


def lists(*values):
    return [upload(np.array(v, np.int32)) for v in values]


PAGES = [  # sequences, entries of a row, pages, tokens of a page, order, padding
    (3, 4, 7, 4, "heads", 0),
    (9, 6, 40, 16, "tokens", 1),
    (9, 6, 40, 1, "heads", 0),
    (40, 30, 2500, 20, "heads", 1),
    (1500, 3, 5000, 8, "heads", 0),
]


@pytest.mark.parametrize("case", range(len(PAGES)))
def test_pages_life(gpu, case):
    """Random reservations, forks, releases and compactions, each compared whole."""
    sequences, row_pages, pages, pt, order, pad = PAGES[case]
    rng = np.random.default_rng(3000 + case)
    book = Book(rng, sequences, row_pages, pages, pt, order=order, pad=pad)
    book.upload()
    args = (book.cache.layout, book.pages)
    k, v = book.pools
    for turn in range(6):
        n = int(rng.integers(1, sequences + 1))
        rows = rng.permutation(sequences)[:n]
        room = row_pages * pt - book.lengths[rows]
        added = np.minimum(rng.integers(0, max(2, pages * pt // sequences // 2), n), room)
        full = book.lengths.copy()
        r, a = lists(rows, added)
        book.reserve(rows, added)
        assert kl.kv_reserve(book.kernel, 0, *book.p, r.data, a.data, n, *args)
        short = np.any((book.lengths - full)[rows] != added)
        book.check(kl.KV_NO_PAGE if short else 0)
        n = int(rng.integers(1, max(2, sequences // 2)))
        children = rng.permutation(sequences)[:n]
        parents = rng.integers(0, sequences, n)
        p, c = lists(parents, children)
        wanted = book.lengths[parents].copy()
        book.fork(parents, children)
        assert kl.kv_fork(book.kernel, 0, k, v, *book.p, p.data, c.data, n, *args)
        book.check(kl.KV_NO_PAGE if np.any(book.lengths[children] != wanted) else 0)
        rows = rng.permutation(sequences)[: max(1, sequences // 3)]
        r, = lists(rows)
        book.free(rows)
        assert kl.kv_free(book.kernel, 0, *book.p, r.data, len(rows), *args)
        book.check()
        used, = lists([0])
        if turn % 2:
            total = book.compact()
            assert kl.kv_compact(book.kernel, 0, k, v, book.p[0], book.p[2], used.data, *book.p, *args)
            book.check()
            assert used.download(1, np.int32)[0] == total
        else:                                      # the same into other arrays
            t, c = upload(np.zeros_like(book.table)), upload(np.zeros_like(book.references))
            total = book.compact()
            assert kl.kv_compact(book.kernel, 0, k, v, t.data, c.data, used.data, *book.p, *args)
            finish()
            book.b[0], book.b[2] = t, c
            book.p = [b.data for b in book.b]
            book.check()
            assert used.download(1, np.int32)[0] == total
        assert np.all(book.references[total:] == 0) and np.all(book.references[:total] > 0)


def test_beams_change_places(gpu):
    """Every sequence of a beam search continues another one, and each is overwritten."""
    rng = np.random.default_rng(31)
    book = Book(rng, 4, 5, 64, 8)
    book.upload()
    args = (book.cache.layout, book.pages)
    r, a = lists([0, 1, 2, 3], [30, 17, 8, 5])
    book.reserve([0, 1, 2, 3], [30, 17, 8, 5])
    assert kl.kv_reserve(book.kernel, 0, *book.p, r.data, a.data, 4, *args)
    for parents in ([1, 0, 3, 2], [0, 0, 0, 1], [3, 3, 3, 3], [2, 1, 0, 3]):
        p, c = lists(parents, [0, 1, 2, 3])
        book.fork(np.array(parents), np.arange(4))
        assert kl.kv_fork(book.kernel, 0, *book.pools, *book.p, p.data, c.data, 4, *args)
        book.check()


def test_pages_report(gpu):
    """Sequences and pages that cannot be are left out and reported; nothing else changes."""
    rng = np.random.default_rng(32)
    book = Book(rng, 4, 5, 12, 8)
    book.upload()
    args = (book.cache.layout, book.pages)
    r, a = lists([0, 4, 1, -1], [10, 5, 41, 5])
    book.reserve([0], [10])
    assert kl.kv_reserve(book.kernel, 0, *book.p, r.data, a.data, 4, *args)
    book.check(kl.KV_BAD_INDEX)
    p, c = lists([0, 9, 0], [1, 2, -4])
    book.fork(np.array([0]), np.array([1]))
    assert kl.kv_fork(book.kernel, 0, *book.pools, *book.p, p.data, c.data, 3, *args)
    book.check(kl.KV_BAD_INDEX)
    r, = lists([17, 1, 1])
    book.free([1])
    assert kl.kv_free(book.kernel, 0, *book.p, r.data, 3, *args)
    book.check(kl.KV_BAD_INDEX)
    s, d = lists([0, 12, -1], [11, 1, 2])
    for pool in book.want:
        pool[:, 11] = pool[:, 0]
    assert kl.kv_copy_pages(book.kernel, 0, *book.pools, s.data, d.data, 3, *args)
    book.check(kl.KV_BAD_PAGE)


def test_reserve_named_twice(gpu):
    """Of two reservations for one sequence one counts; the other, which would end past the row, is reported."""
    rng = np.random.default_rng(33)
    book = Book(rng, 3, 5, 24, 8)
    book.upload()
    args = (book.cache.layout, book.pages)
    r, a = lists([1, 0, 1], [30, 9, 30])
    assert kl.kv_reserve(book.kernel, 0, *book.p, r.data, a.data, 3, *args)
    finish()
    assert kl.kv_cache_status(0) == kl.KV_BAD_INDEX
    table, lengths, references = (b.download(x.shape, np.int32)
                                  for b, x in zip(book.b, (book.table, book.lengths, book.references)))
    assert lengths.tolist() == [9, 30, 0]
    assert table[0].tolist() == [4, 5, -1, -1, -1] and table[2].tolist() == [-1] * 5
    assert table[1].tolist() in ([0, 1, 2, 3, -1], [6, 7, 8, 9, -1])
    held = np.bincount(table[table >= 0], minlength=24)
    assert np.array_equal(references, held)


def test_fork_named_twice(gpu):
    """Of two forks to one child one is made; the other is reported, and every count is its page's rows."""
    rng = np.random.default_rng(34)
    book = Book(rng, 4, 5, 24, 8)
    book.upload()
    args = (book.cache.layout, book.pages)
    r, a = lists([0, 1, 2], [30, 17, 9])
    book.reserve([0, 1, 2], [30, 17, 9])
    assert kl.kv_reserve(book.kernel, 0, *book.p, r.data, a.data, 3, *args)
    p, c = lists([0, 1, 0], [2, 2, 3])
    assert kl.kv_fork(book.kernel, 0, *book.pools, *book.p, p.data, c.data, 3, *args)
    finish()
    assert kl.kv_cache_status(0) == kl.KV_BAD_INDEX
    table, lengths, references = (b.download(x.shape, np.int32)
                                  for b, x in zip(book.b, (book.table, book.lengths, book.references)))
    assert lengths[[0, 1, 3]].tolist() == [30, 17, 30] and lengths[2] in (30, 17)
    assert np.array_equal(table[:2], book.table[:2])
    parent = 0 if lengths[2] == 30 else 1
    for child, of in ((2, parent), (3, 0)):
        full = int(lengths[of]) // 8
        assert np.array_equal(table[child, :full], book.table[of, :full])
        assert np.all(table[child, full + 1:] == -1)
        for view, pool in zip(book.cache.download()[1], book.want):
            rest = int(lengths[of]) % 8
            assert np.array_equal(view[:, table[child, full], :, :rest], pool[:, book.table[of, full], :, :rest])
    assert np.array_equal(references, np.bincount(table[table >= 0], minlength=24))


@pytest.mark.parametrize("order,pad,count", [("heads", 0, 1), ("tokens", 0, 40), ("heads", 1, 40), ("tokens", 1, 3)])
def test_copy_pages(gpu, order, pad, count):
    rng = np.random.default_rng(33)
    book = Book(rng, 2, 5, 100, 24, heads=5, width=72, layers=3, order=order, pad=pad)
    book.upload()
    ids = rng.permutation(100)
    src, dst = ids[:count], ids[count:2 * count]
    for pool in book.want:
        pool[:, dst] = pool[:, src]
    s, d = lists(src, dst)
    assert kl.kv_copy_pages(book.kernel, 0, *book.pools, s.data, d.data, count, book.cache.layout, book.pages)
    book.check()


# --- logits -----------------------------------------------------------------------------

def gold_logits(z, penalties, history, history_lengths, ids, values, bias_lengths, mask):
    y = z.astype(np.float64)
    rows, vocabulary = y.shape
    for i in range(rows):
        if history is not None:
            h = history[i, :history_lengths[i]]
            n = np.bincount(h[(h >= 0) & (h < vocabulary)], minlength=vocabulary).astype(np.float64)
            r, f, p = penalties[i].astype(np.float64)
            met = n > 0
            y[i] = np.where(met, np.where(y[i] > 0, y[i] / r, y[i] * r) - n * f - p, y[i])
        if ids is not None:
            last = {t: x for t, x in zip(ids[i, :bias_lengths[i]], values[i, :bias_lengths[i]])
                    if 0 <= t < vocabulary}
            for t, x in last.items():
                y[i, t] += np.float64(x)
        if mask is not None:
            words = mask[i if len(mask) > 1 else 0]
            bits = (words[:, None] >> np.arange(32, dtype=np.uint32)) & 1
            y[i, bits.ravel()[:vocabulary] == 0] = -np.inf
    return y


# rows, vocabulary, history, biases, mask (0 none, 1 shared, 2 each row), pad, offset, in place
LOGITS = [
    (1, 1, 1, 1, 0, 0, 0, False),
    (1, 31, 5, 2, 2, 0, 0, False),
    (3, 4096, 100, 10, 2, 0, 0, True),
    (3, 4097, 300, 10, 1, 0, 0, False),
    (5, 32000, 3000, 300, 2, 0, 0, False),
    (2, 32000, 0, 0, 0, 4, 0, True),
    (4, 8193, 70, 400, 2, 3, 1, False),
    (2, 151937, 9000, 64, 1, 7, 0, True),
]


@pytest.mark.parametrize("case", range(len(LOGITS)))
def test_logits(gpu, case):
    rows, vocabulary, past, biases, masks, pad, offset, in_place = LOGITS[case]
    rng = np.random.default_rng(4000 + case)
    z = (rng.standard_normal((rows, vocabulary)) * 4).astype(np.float32)
    z.flat[:: 97] = np.inf
    z.flat[1:: 101] = -np.inf
    z.flat[2:: 103] = 0.0
    penalties = np.stack([1 + rng.random(rows), rng.random(rows), rng.random(rows)], 1).astype(np.float32)
    # some tokens many times, some outside the vocabulary
    history = rng.integers(-3, min(vocabulary, 40) + 3, (rows, past)).astype(np.int32) if past else None
    if past:
        history[:, ::2] = rng.integers(0, vocabulary, history[:, ::2].shape)
    history_lengths = rng.integers(0, past + 1, rows).astype(np.int32)
    history_lengths[0] = past
    ids = rng.integers(-2, vocabulary + 2, (rows, biases)).astype(np.int32) if biases else None
    values = (rng.standard_normal((rows, biases)) * 5).astype(np.float32)
    if biases > 3:
        ids[:, 3] = ids[:, 0]                          # named twice: the later one counts
        values[:, 2] = -np.inf
    bias_lengths = rng.integers(0, biases + 1, rows).astype(np.int32)
    bias_lengths[0] = biases
    mask = None
    if masks:
        mask = rng.integers(0, 2 ** 32, (1 if masks == 1 else rows, -(-vocabulary // 32)), dtype=np.uint32)
        mask[-1] = 0                                   # a grammar that allows nothing
    stride = vocabulary + pad
    flat = np.full(offset + rows * stride, GUARD, np.float32)
    flat[offset:].reshape(rows, stride)[:, :vocabulary] = z
    zb = upload(flat)
    yb = zb if in_place else upload(np.full_like(flat, GUARD))
    b = [upload(x) if x is not None else None
         for x in (penalties, history, history_lengths, ids, values, bias_lengths, mask)]
    call = kl.LogitsLayout(rows, vocabulary, stride, stride, past, biases, 0 if masks < 2 else mask.shape[1])
    assert kl.logits_reason(call) == ""
    kernel = kl.Kernel()
    assert kl.process_logits(kernel, 0, yb.data + 4 * offset, zb.data + 4 * offset, *b, call)
    finish()
    assert kernel.route == "process_logits"
    got = yb.download(flat.shape, np.float32)
    assert np.all(got[:offset] == GUARD) and np.all(got[offset:].reshape(rows, stride)[:, vocabulary:] == GUARD)
    y = got[offset:].reshape(rows, stride)[:, :vocabulary].astype(np.float64)
    with np.errstate(invalid="ignore"):
        gold = gold_logits(z, penalties, history, history_lengths, ids, values, bias_lengths, mask)
        same = (y == gold) | (np.isnan(y) & np.isnan(gold))
        # up to four F32 roundings of values up to |z| r + n f + p + |bias|
        size = np.abs(z) * 2 + 2 + past + 30
        assert np.all(same | (np.abs(y - gold) <= 4 * 2.0 ** -24 * size))
    assert not np.any(np.isposinf(gold) ^ np.isposinf(y))


def test_compact_large_pool(gpu):
    """Lists over several workgroups: more pages than one takes, holes and used pages anywhere, counts in place and apart."""
    rng = np.random.default_rng(51)
    for pages, share in ((20000, 0.5), (20000, 0.97), (30001, 0.05), (8192, 1.0), (8193, 0.0)):
        book = Book(rng, 50, pages // 50 + 1, pages, 1, heads=1, width=8, layers=1)
        ids = rng.permutation(pages)[: int(pages * share)]
        for s, part in enumerate(np.array_split(ids, 50)):
            book.table[s, :len(part)], book.lengths[s] = part, len(part)
        book.references[ids] = rng.integers(1, 4, len(ids))
        book.upload()
        used, = lists([-1])
        args = (book.cache.layout, book.pages)
        t, c = upload(np.zeros_like(book.table)), upload(np.full_like(book.references, 77))
        total = book.compact()
        assert kl.kv_compact(book.kernel, 0, *book.pools, t.data, c.data, used.data, *book.p, *args)
        finish()
        assert used.download(1, np.int32)[0] == total == len(ids)
        assert np.array_equal(t.download(book.table.shape, np.int32), book.table)
        assert np.array_equal(c.download(book.references.shape, np.int32), book.references)
        assert kl.kv_compact(book.kernel, 0, *book.pools, book.p[0], book.p[2], used.data, *book.p, *args)
        book.check()


@pytest.mark.parametrize("page_tokens", [1, 3, 16])
@pytest.mark.parametrize("sequences,heads", [(1, 1), (70, 8)])
def test_attention_loose_bound(gpu, page_tokens, sequences, heads):
    """`longest` far above the lengths: rows of many entries, most of which are never read."""
    rng = np.random.default_rng(61)
    longest = 1 << 20 if sequences == 1 else 150000
    lengths = [int(n) for n in rng.integers(1, 40, sequences)]
    lengths[-1] = 700
    pages = sum(-(-n // page_tokens) for n in lengths) + 1
    cache = Cache(rng, pages, page_tokens, heads, 64)
    table = table_of(rng, lengths, page_tokens, pages, -(-longest // page_tokens), rest=-7)
    q = rng.standard_normal((sequences, heads, 64)).astype(np.float32)
    y, _ = run_attention(cache, table, lengths, q, longest=longest)
    gold, tol = gold_attention(cache, table, lengths, q, 0, 0.125)
    check(y, gold, tol)
    assert gpu.kv_cache_status(0) == 0


def test_attention_subnormal_values(gpu):
    """F16 values below 2^-14 count in full, as keys and as values."""
    rng = np.random.default_rng(62)
    lengths = [100, 33]
    cache = Cache(rng, 20, 16, 2, 64)
    cache.flat[1][:] = (rng.integers(-1023, 1024, cache.flat[1].size) * 2.0 ** -24).astype(np.float16)
    cache.flat[0][:] = (rng.integers(-1023, 1024, cache.flat[0].size) * 2.0 ** -24).astype(np.float16)
    table = table_of(rng, lengths, 16, 20, 7)
    q = rng.standard_normal((2, 4, 64)).astype(np.float32)
    y, _ = run_attention(cache, table, lengths, q, scale=4096.0)
    gold, tol = gold_attention(cache, table, lengths, q, 0, 4096.0)
    assert np.abs(gold).max() < 2.0 ** -14 and np.abs(gold).max() > 2.0 ** -18
    check(y, gold, tol)


def test_attention_many_rows(gpu):
    """More rows than the card holds at once, short and ragged: one wave to a workgroup and whole rows."""
    rng = np.random.default_rng(63)
    for most, width in ((3, 64), (97, 72), (128, 128), (129, 64), (500, 64)):
        lengths = [int(n) for n in rng.integers(0, most + 1, 140)]
        lengths[7] = most
        pages = sum(-(-n // 16) for n in lengths) + 1
        cache = Cache(rng, pages, 16, 8, width)
        table = table_of(rng, lengths, 16, pages, -(-most // 16), rest=99999999)
        q = rng.standard_normal((140, 8, width)).astype(np.float32)
        y, route = run_attention(cache, table, lengths, q)
        assert route == "paged_attention"
        gold, tol = gold_attention(cache, table, lengths, q, 0, width ** -0.5)
        check(y, gold, tol)


# lengths, heads, query heads, width, tokens of a page, window, F16, order, `longest`
EVEN = [
    ([0, 1, 33, 0, 0, 700, 32, 31, 2500, 64, 5, 0], 4, 4, 128, 16, 0, False, "heads", 2816),
    ([0] * 12, 4, 8, 128, 16, 0, False, "heads", 2816),
    ([1] * 12, 4, 8, 128, 16, 0, True, "tokens", 2816),
    ([2816, 1, 1, 2815, 16, 17, 129, 0], 8, 32, 128, 32, 0, True, "tokens", 2816),
    ([40, 41, 1500, 3, 1301, 999, 0, 7, 8, 9, 10, 11] * 2, 4, 28, 64, 48, 0, False, "tokens", 2816),
    ([300, 2100, 33, 70], 8, 8, 256, 16, 0, False, "heads", 2560),
    ([7000, 5033, 10, 4999], 4, 16, 256, 16, 5000, True, "tokens", 7008),
    ([4000, 1501, 1500, 1499, 0, 20, 3000, 2000], 8, 24, 192, 32, 1500, False, "heads", 4000),
    ([1800, 90, 0, 1, 640, 33, 34, 35], 12, 12, 96, 16, 0, True, "tokens", 2000),
    ([3000], 4, 32, 256, 64, 0, False, "tokens", 66048),
    ([i * 37 % 61 for i in range(130)], 4, 8, 64, 16, 0, False, "heads", 1104),
    ([i * 53 % 101 if i > 99 else 0 for i in range(200)], 4, 4, 128, 16, 0, False, "tokens", 1104),
    ([i * 71 % 601 for i in range(40)], 4, 8, 256, 16, 0, False, "heads", 608),
    ([i * 71 % 901 for i in range(70)], 8, 8, 64, 32, 0, True, "tokens", 928),
]


@pytest.mark.parametrize("case", range(len(EVEN)))
def test_attention_even(gpu, case):
    """Equal shares of all sequences' tokens: parts that begin and end anywhere, in rows of any length and of none."""
    lengths, heads, query_heads, width, page_tokens, window, half, order, longest = EVEN[case]
    rng = np.random.default_rng(1500 + case)
    row_pages = -(-longest // page_tokens)
    pages = sum(-(-n // page_tokens) for n in lengths) + 2
    cache = Cache(rng, pages, page_tokens, heads, width, order, case % 2)
    table = table_of(rng, lengths, page_tokens, pages, row_pages, rest=2 ** 30)
    q = (rng.standard_normal((len(lengths), query_heads, width)) * 2).astype(np.float16 if half else np.float32)
    owned = np.zeros((pages, page_tokens), bool)
    for s, n in enumerate(lengths):
        t = np.arange(n)
        owned[table[s, t // page_tokens], t % page_tokens] = True
    for pool in (cache.k, cache.v):
        pool[0].transpose(0, 2, 1, 3)[~owned] = np.nan
    y, route = run_attention(cache, table, lengths, q, window, longest=longest, pad=3)
    assert route == "paged_attention_even"
    gold, tol = gold_attention(cache, table, lengths, q, window, width ** -0.5)
    check(y, gold, tol)
    again, _ = run_attention(cache, table, lengths, q, window, longest=longest, pad=3)
    assert np.array_equal(y, again), "the same call gives other bits"
    assert gpu.kv_cache_status(0) == 0


@pytest.mark.parametrize("sequences,heads,width,page_tokens,order,longest", [
    (1000, 8, 256, 32, "heads", 64),            # one wave a workgroup
    (1000, 4, 128, 16, "tokens", 128),
    (32, 8, 128, 16, "tokens", 1024),           # eight waves
    (600, 4, 256, 16, "heads", 512),            # whole rows
    (64, 8, 160, 16, "tokens", 2048),           # a width between
    (64, 6, 128, 16, "tokens", 2048),           # heads that are not fours
    (64, 8, 128, 24, "heads", 2048),            # pages that are not whole half steps
    (1100, 4, 128, 16, "heads", 1040),          # more sequences than are shared out
])
def test_attention_not_even(gpu, sequences, heads, width, page_tokens, order, longest):
    """Large calls beside those that are shared out."""
    rng = np.random.default_rng(72)
    lengths = [int(n) for n in rng.integers(0, 40, sequences)]
    lengths[sequences // 3] = longest
    pages = sum(-(-n // page_tokens) for n in lengths) + 1
    cache = Cache(rng, pages, page_tokens, heads, width, order)
    table = table_of(rng, lengths, page_tokens, pages, -(-longest // page_tokens), rest=-7)
    q = rng.standard_normal((sequences, heads, width)).astype(np.float32)
    y, route = run_attention(cache, table, lengths, q, longest=longest)
    assert route != "paged_attention_even"
    gold, tol = gold_attention(cache, table, lengths, q, 0, width ** -0.5)
    check(y, gold, tol)


def test_attention_even_reports(gpu):
    """Bad pages and lengths among even shares; what is not a number stays in its sequence and heads."""
    rng = np.random.default_rng(71)
    lengths = [500, 40, 0, 900, 33, 1, 320, 1200]
    cache = Cache(rng, 260, 16, 8, 128)
    table = table_of(rng, lengths, 16, 260, 176)
    q = rng.standard_normal((8, 8, 128)).astype(np.float32)
    gold, tol = gold_attention(cache, table, lengths, q, 0, 128 ** -0.5)
    bad = table.copy()
    bad[0, 3], bad[3, 20], bad[4, 0] = 260, -1, 2 ** 31 - 1
    y, route = run_attention(cache, bad, lengths, q, longest=2816)
    assert route == "paged_attention_even"
    assert gpu.kv_cache_status(0) == kl.KV_BAD_PAGE
    safe = bad.copy()
    safe[0, 3] = safe[4, 0] = -1
    check(y, *gold_attention(cache, safe, lengths, q, 0, 128 ** -0.5, skip=(-1,)))
    wrong = [500, 40, -5, 900, 33, 1, 320, 2 ** 30]
    table[7] = np.resize(table[7, :75], 176)
    y, _ = run_attention(cache, table, wrong, q, longest=2816)
    assert gpu.kv_cache_status(0) == kl.KV_BAD_INDEX
    check(y[:7], gold[:7], tol[:7])
    gold_cut, tol_cut = gold_attention(cache, table, [0] * 7 + [2816], q, 0, 128 ** -0.5)
    check(y[7], gold_cut[7], tol_cut[7])
    cache.k[0, table[3, 30], 5, 2, 9] = np.nan
    cache.v[0, table[6, 1], 2, 2, 9] = np.inf
    q[1, 6, 77] = np.nan
    y, _ = run_attention(cache, table, lengths, q, longest=2816)
    odd = np.zeros(y.shape, bool)
    odd[3, 5] = odd[1, 6] = odd[6, 2, 9] = True
    assert np.array_equal(~np.isfinite(y), odd)
    gold, tol = gold_attention(cache, table, lengths, q, 0, 128 ** -0.5)
    check(np.where(odd, 0, y), np.where(odd, 0, gold), np.where(odd, 0, tol))
