"""The 8-bit key-value cache on the GPU against plain models (kv_f8.py) in 64 bits: codes and scales bit for bit, attention
within the tolerance derived there."""
import numpy as np
import pytest

import kunlunk200_lib_amd as kl
from kv_f8 import (GUARD, VALUES, CacheF8, check, encode, finish, gold_attention, model_append, model_read, run_append,
                   run_attention, run_read, table_of, turned, upload)

pytestmark = pytest.mark.gpu
ADJACENT, HALVES = kl.RotaryPairs.adjacent, kl.RotaryPairs.halves

# lengths, heads, query heads, width, tokens of a page, of a block, window, F16, order, padding
ATTENTION = [
    ([1], 1, 1, 8, 1, 1, 0, False, "heads", 0),
    ([1, 0, 2], 2, 2, 64, 16, 16, 0, False, "heads", 0),
    ([31, 32, 33, 0, 16, 17], 4, 4, 128, 16, 8, 0, False, "heads", 0),
    ([127, 128, 129, 255, 256, 257, 5, 1], 8, 32, 128, 32, 1, 0, True, "tokens", 0),
    ([300, 77], 5, 15, 80, 20, 4, 0, False, "heads", 1),
    ([300, 77], 5, 15, 80, 20, 1, 100, True, "tokens", 1),
    ([300, 77], 5, 15, 80, 48, 16, 100, True, "heads", 1),
    ([513], 2, 18, 96, 3, 1, 0, False, "heads", 0),             # 9 query heads a key-value head: two column tiles
    ([700, 3], 1, 16, 128, 64, 64, 0, True, "heads", 0),
    ([640], 1, 71, 64, 16, 2, 0, False, "tokens", 0),
    ([260, 261], 2, 2, 256, 16, 4, 0, False, "heads", 0),
    ([260, 61], 2, 2, 256, 32, 32, 0, True, "tokens", 1),
    ([130], 3, 27, 192, 100, 2, 0, True, "heads", 1),
    ([90], 1, 1, 24, 7, 1, 0, False, "tokens", 1),
    ([90], 2, 4, 40, 4, 4, 0, True, "heads", 0),
    ([90], 2, 4, 72, 12, 2, 33, False, "heads", 0),
    ([90], 2, 4, 104, 1, 1, 0, False, "heads", 0),
    ([90, 12], 2, 2, 136, 8, 8, 0, False, "heads", 0),
    ([90, 12], 2, 2, 136, 16, 1, 0, False, "tokens", 0),
    ([150], 1, 9, 200, 16, 16, 64, False, "tokens", 0),
    ([5000, 4999, 10], 1, 4, 128, 2048, 32, 0, False, "heads", 0),
    ([9001, 1, 4096, 0], 2, 8, 64, 16, 2, 0, False, "heads", 0),
    ([9001, 700, 64], 2, 8, 128, 16, 16, 1, False, "heads", 0),   # the newest token alone
    ([3000, 65], 2, 8, 128, 16, 4, 64, True, "heads", 0),
    ([20000], 8, 8, 128, 128, 64, 0, True, "heads", 0),
    ([70, 16], 2, 8, 96, 16, 8, 0, False, "heads", 0),
    ([70, 16], 2, 2, 192, 32, 16, 40, False, "tokens", 0),
    ([70, 16], 1, 12, 56, 16, 1, 0, True, "heads", 0),
    ([2100, 300], 1, 20, 128, 48, 4, 500, False, "heads", 1),
]


def spoil(cache, table, lengths, window=0):
    """What no token owns may be anything: codes that are no numbers past each end, before each window and in free pages,
    and scales of blocks without a token."""
    c, block = cache.layout.cache, cache.layout.block_tokens
    owned = np.zeros((c.pages, c.page_tokens), bool)
    for s, n in enumerate(lengths):
        t = np.arange(max(0, n - window) if window else 0, n)
        owned[table[s, t // c.page_tokens], t % c.page_tokens] = True
    for pool in (cache.k, cache.v):
        pool[0].transpose(0, 2, 1, 3)[~owned] = 0x7f
    cache.v[0].transpose(0, 2, 1, 3)[~owned, :, ::2] = 0xff
    of_block = owned.reshape(c.pages, -1, block).any(2)
    for scales, bad in ((cache.ks, np.nan), (cache.vs, np.inf)):
        scales[0].transpose(0, 2, 1)[~of_block] = bad


@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention(gpu, case):
    lengths, heads, query_heads, width, page_tokens, block, window, half, order, pad = ATTENTION[case]
    rng = np.random.default_rng(2000 + case)
    row_pages = -(-max(lengths) // page_tokens) + 2
    pages = sum(-(-n // page_tokens) for n in lengths) + 2
    cache = CacheF8(rng, pages, page_tokens, heads, width, block, order, pad)
    # entries past a sequence's pages are not read, whatever they hold
    table = table_of(rng, lengths, page_tokens, pages, row_pages, rest=2 ** 30)
    q = (rng.standard_normal((len(lengths), query_heads, width)) * 2).astype(np.float16 if half else np.float32)
    spoil(cache, table, lengths, window)
    y, _ = run_attention(cache, table, lengths, q, window, pad=3 * pad)
    gold, tol = gold_attention(cache, table, lengths, q, window, width ** -0.5)
    check(y, gold, tol)
    again, _ = run_attention(cache, table, lengths, q, window, pad=3 * pad)
    assert np.array_equal(y, again), "the same call gives other bits"
    assert gpu.kv_cache_status(0) == 0
    # a looser bound on the lengths splits otherwise and gives the same within the tolerance
    y, _ = run_attention(cache, table, lengths, q, window, longest=row_pages * page_tokens)
    check(y, gold, tol)


# sequences, heads, query heads, width, tokens of a page, of a block, longest, order, route: every kernel at full rows and
# at each way to find scales
ROUTES = [
    (64, 8, 8, 128, 16, 16, 2816, "heads", "paged_attention_f8_even"),
    (64, 8, 24, 128, 32, 8, 2816, "tokens", "paged_attention_f8_even"),
    (64, 8, 8, 128, 16, 1, 2816, "heads", "paged_attention_f8_even"),
    (48, 4, 4, 64, 64, 64, 9000, "heads", "paged_attention_f8_even"),
    (48, 4, 8, 96, 16, 2, 6000, "tokens", "paged_attention_f8_even"),
    (40, 4, 4, 256, 16, 4, 2800, "heads", "paged_attention_f8_even"),
    (24, 8, 8, 192, 32, 32, 3500, "tokens", "paged_attention_f8_even"),
    (2, 4, 4, 128, 16, 16, 6000, "heads", "paged_attention_f8_split"),
    (2, 4, 4, 128, 32, 4, 6000, "tokens", "paged_attention_f8_split"),
    (2, 4, 64, 128, 16, 2, 6000, "heads", "paged_attention_f8_split"),
    (600, 2, 2, 64, 16, 16, 100, "heads", "paged_attention_f8"),
    (600, 2, 2, 128, 16, 1, 100, "heads", "paged_attention_f8"),
    (300, 4, 4, 128, 16, 4, 900, "heads", "paged_attention_f8"),
    (8, 8, 8, 128, 16, 8, 500, "heads", "paged_attention_f8"),
]


@pytest.mark.parametrize("case", range(len(ROUTES)))
def test_attention_routes(gpu, case):
    sequences, heads, query_heads, width, page_tokens, block, longest, order, route = ROUTES[case]
    rng = np.random.default_rng(3000 + case)
    lengths = np.exp(rng.uniform(0, np.log(longest), sequences)).astype(int)
    lengths[0], lengths[sequences // 2] = longest, 0
    # the sequences share a few pages: what is read is what counts here
    pages = -(-longest // page_tokens) + 3
    table = rng.integers(0, pages, (sequences, pages)).astype(np.int32)
    cache = CacheF8(rng, pages, page_tokens, heads, width, block, order)
    q = rng.standard_normal((sequences, query_heads, width)).astype(np.float32)
    y, took = run_attention(cache, table, lengths, q)
    assert took == route
    gold, tol = gold_attention(cache, table, lengths, q, 0, width ** -0.5)
    check(y, gold, tol)
    window = longest // 3
    y, _ = run_attention(cache, table, lengths, q, window)
    gold, tol = gold_attention(cache, table, lengths, q, window, width ** -0.5)
    check(y, gold, tol)
    assert gpu.kv_cache_status(0) == 0


# kernels: whole rows, parts, equal shares
KERNELS = [([70, 300], 2, 4, 64, 16, 16), ([6000], 2, 4, 128, 16, 4), ([2816] * 20 + [100, 1], 8, 8, 128, 16, 1),
           ([300, 20], 2, 4, 80, 20, 4)]


def make(case, seed, longest=None):
    lengths, heads, query_heads, width, page_tokens, block = KERNELS[case]
    rng = np.random.default_rng(seed)
    pages = -(-max(lengths) // page_tokens) + 3
    table = np.stack([rng.permutation(pages) for _ in lengths]).astype(np.int32)
    cache = CacheF8(rng, pages, page_tokens, heads, width, block)
    q = rng.standard_normal((len(lengths), query_heads, width)).astype(np.float32)
    return rng, lengths, table, cache, q


@pytest.mark.parametrize("case", range(len(KERNELS)))
@pytest.mark.parametrize("kind", ["wide", "any", "one_large", "small", "large"])
def test_attention_value_scales(gpu, case, kind):
    """Value scales of any size beside one another, powers of two or not, negative, zero."""
    rng, lengths, table, cache, q = make(case, 40)
    shape = cache.vs.shape
    if kind == "wide":
        cache.vs[...] = 2.0 ** rng.integers(-60, 60, shape)
    elif kind == "any":
        cache.vs[...] = rng.standard_normal(shape) * (rng.random(shape) < 0.9)
        cache.ks[...] = rng.standard_normal(shape) / 300
    elif kind == "one_large":
        # the first tokens' values are 2^50 times the others' and weigh e^-60 of them and less
        cache.vs[...] = 2.0 ** -8
        c = cache.layout.cache
        for row in table:
            cache.vs[0, row[0]] = 2.0 ** 42
            cache.k[0, row[0]] = encode(-np.abs(VALUES[cache.k[0, row[0]]]))
            cache.ks[0, row[0]] = 2.0 ** -4
        q = np.abs(q) + 0.5
        assert c.page_tokens > 1
    else:
        cache.vs[...] = 2.0 ** (-64 if kind == "small" else 100)
    y, _ = run_attention(cache, table, lengths, q)
    gold, tol = gold_attention(cache, table, lengths, q, 0, q.shape[2] ** -0.5)
    check(y, gold, tol)


@pytest.mark.parametrize("case", range(len(KERNELS)))
def test_attention_key_scales(gpu, case):
    """Key scales of any size beside one another; a few tokens with all the weight."""
    rng, lengths, table, cache, q = make(case, 41)
    cache.ks[...] = 2.0 ** rng.integers(-64, -6, cache.ks.shape)
    y, _ = run_attention(cache, table, lengths, q)
    gold, tol = gold_attention(cache, table, lengths, q, 0, q.shape[2] ** -0.5)
    check(y, gold, tol)


@pytest.mark.parametrize("case", range(len(KERNELS)))
def test_attention_not_a_number(gpu, case):
    """A scale or a code that is not a number reaches the heads that read it and no others."""
    _, lengths, table, cache, q = make(case, 42)
    c, group = cache.layout.cache, q.shape[1] // cache.layout.cache.heads
    row, where = 0, min(lengths[0] - 1, 37)
    page, at = table[row, where // c.page_tokens], where % c.page_tokens
    for scales in (cache.ks, cache.vs):
        kept = scales[0, page, 1, at // cache.layout.block_tokens]
        scales[0, page, 1, at // cache.layout.block_tokens] = np.nan
        y, _ = run_attention(cache, table[:1], lengths[:1], q[:1])
        assert np.all(np.isnan(y[0, group:2 * group]))
        scales[0, page, 1, at // cache.layout.block_tokens] = kept
        gold, tol = gold_attention(cache, table[:1], lengths[:1], q[:1], 0, q.shape[2] ** -0.5)
        check(y[:, :group], gold[:, :group], tol[:, :group])
        check(y[:, 2 * group:], gold[:, 2 * group:], tol[:, 2 * group:])
    cache.v[0, page, 1, at, 5] = 0x7f
    y, _ = run_attention(cache, table[:1], lengths[:1], q[:1])
    assert np.all(np.isnan(y[0, group:2 * group, 5])) and np.isnan(y).sum() == group
    cache.k[0, page, 0, at, 5] = 0xff
    y, _ = run_attention(cache, table[:1], lengths[:1], q[:1])
    assert np.all(np.isnan(y[0, :group]))


@pytest.mark.parametrize("case", range(len(KERNELS)))
def test_attention_infinite_queries(gpu, case):
    """All scores -inf: zeros. A query that is not a number: its own head alone."""
    _, lengths, table, cache, q = make(case, 43)
    cache.k[..., 3] = 0x81 | cache.k[..., 3] & 0x3f      # below 0 everywhere
    q[0, 1] = np.abs(q[0, 1])
    q[0, 1, 3] = np.inf
    q[-1, -1, 7] = np.nan
    y, _ = run_attention(cache, table, lengths, q)
    assert np.all(y[0, 1] == 0) and np.all(np.isnan(y[-1, -1]))
    q[0, 1, 3] = q[-1, -1, 7] = 0
    gold, tol = gold_attention(cache, table, lengths, q, 0, q.shape[2] ** -0.5)
    rest = np.ones(q.shape[:2], bool)
    rest[0, 1] = rest[-1, -1] = False
    check(y[rest], gold[rest], tol[rest])


@pytest.mark.parametrize("scale", [0.0, -0.5, 1e-20, 30.0])
@pytest.mark.parametrize("size", [1e-30, 1.0, 1e4])
def test_attention_scales(gpu, scale, size):
    rng = np.random.default_rng(6)
    cache = CacheF8(rng, 20, 16, 2, 64, 4)
    table = table_of(rng, [200], 16, 20, 13)
    q = (rng.standard_normal((1, 4, 64)) * size).astype(np.float32)
    y, _ = run_attention(cache, table, [200], q, scale=scale)
    gold, tol = gold_attention(cache, table, [200], q, 0, float(np.float32(scale)))
    # scores of several thousand: their error makes the tolerance more than the values
    check(y, gold, np.minimum(tol, 20.0))


def test_attention_reports(gpu):
    """Pages outside the pool are left out, lengths past the bound cut, and both reported once."""
    rng = np.random.default_rng(9)
    lengths = [150, 400]
    for page_tokens in (16, 20):
        cache = CacheF8(rng, 40, page_tokens, 2, 64, 4)
        table = table_of(rng, lengths, page_tokens, 40, 26)
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


def test_offsets_past_32_bits(gpu):
    """Pages more than 4 GiB apart: append, attention, read-back and copies reach them."""
    rng = np.random.default_rng(11)
    pages, pt, heads, width = 3, 16, 2, 64
    stride = (1 << 32) + 1024
    layout = kl.KVCacheF8Layout(kl.KVCacheLayout(pages, pt, heads, width, stride, pt * width, width), 8)
    small = CacheF8(rng, pages, pt, heads, width, 8)
    n = heads * pt * width
    size = (pages - 1) * stride + n
    lengths = [40]
    table = np.array([[2, 0, 1]], np.int32)
    q = rng.standard_normal((1, 4, width)).astype(np.float32)
    with kl.Buffer(0, size) as kb, kl.Buffer(0, size) as vb:
        for p in range(pages):
            for b, flat in zip((kb, vb), small.flat):
                b.upload(flat[p * n:(p + 1) * n], offset=p * stride)
        scales = [upload(x) for x in small.scales]
        pools = [kb.data, vb.data, scales[0].data, scales[1].data]
        new = rng.standard_normal((1, 2 * heads * width)).astype(np.float32)
        rows, y = upload(new), upload(np.zeros_like(q))
        ints = [upload(np.array(x, np.int32)) for x in (lengths, table)]
        append = kl.KVAppendLayout(1, 1, 3, 0, 0, 256, 256, 0, 0, 0, HALVES, kl.InputType.f32)
        kernel = kl.Kernel()
        assert kl.kv_append_f8(kernel, 0, *pools, None, None, rows.data, rows.data + 512, None, None, ints[0].data,
                               ints[1].data, None, None, layout, append)
        x = new.reshape(1, 2, heads, width)
        model_append(small, table, [0], [39], x[:, 0], x[:, 1], (), (), HALVES, 0)
        call = kl.PagedAttentionLayout(1, 4, 48, 0, 3, 256, 256, 0.125, kl.InputType.f32)
        q_buffer = upload(q)
        assert kl.paged_attention_f8(kernel, 0, y.data, q_buffer.data, *pools, ints[1].data, ints[0].data, layout, call)
        finish()
        gold, tol = gold_attention(small, table, lengths, q, 0, 0.125)
        check(y.download(q.shape, np.float32), gold, tol)
        source, target = upload(np.array([1], np.int32)), upload(np.array([0], np.int32))
        assert kl.kv_copy_pages_f8(kernel, 0, *pools, source.data, target.data, 1, layout, kl.KVPagesLayout(1, 3, 1, 0))
        finish()
        for b, flat in zip((kb, vb), small.flat):
            assert np.array_equal(b.download(n, np.uint8, offset=2 * stride), flat[2 * n:3 * n])
            assert np.array_equal(b.download(n, np.uint8, offset=0), flat[n:2 * n])
    assert gpu.kv_cache_status(0) == 0


# --- append and read-back ---------------------------------------------------------------------

# (past, new) of each sequence, heads, query heads, width, tokens of a page, of a block, rotary, pairs, F16, order, padding,
# values the rows are off 16 bytes
APPEND = [
    ([(0, 1)], 1, 1, 8, 1, 1, 8, ADJACENT, False, "heads", 0, 0),
    ([(5, 1), (0, 1), (15, 1), (16, 1)], 2, 4, 64, 16, 16, 64, ADJACENT, False, "heads", 0, 0),
    ([(5, 1), (0, 1), (15, 1), (16, 1)], 4, 4, 128, 16, 4, 128, HALVES, True, "heads", 0, 0),
    ([(7, 50), (0, 33), (31, 2)], 3, 6, 128, 32, 16, 64, HALVES, False, "tokens", 0, 0),
    ([(7, 50), (0, 33), (31, 2)], 3, 6, 128, 32, 32, 64, ADJACENT, True, "heads", 1, 0),
    ([(63, 130), (1, 64)], 2, 2, 256, 64, 64, 256, HALVES, False, "heads", 0, 0),
    ([(63, 130), (1, 64)], 2, 2, 128, 128, 64, 0, HALVES, True, "tokens", 1, 0),
    ([(3, 40)], 5, 10, 80, 20, 4, 80, HALVES, False, "heads", 0, 0),
    ([(3, 40)], 5, 10, 80, 20, 1, 36, HALVES, False, "heads", 0, 0),         # turned pairs that end inside a unit
    ([(3, 40)], 2, 2, 24, 24, 8, 10, ADJACENT, True, "tokens", 1, 0),
    ([(3, 40), (2, 5)], 2, 2, 40, 8, 2, 2, HALVES, False, "heads", 0, 1),
    ([(11, 60)], 2, 6, 72, 12, 4, 72, HALVES, True, "heads", 0, 3),
    ([(11, 60), (0, 9)], 1, 8, 136, 16, 8, 64, ADJACENT, False, "tokens", 0, 2),
    ([(30, 70)], 1, 1, 256, 64, 32, 128, ADJACENT, False, "heads", 2, 0),
    ([(0, 300)], 8, 8, 64, 16, 16, 64, HALVES, False, "heads", 0, 0),
    ([(2, 100)], 1, 2, 8, 64, 64, 4, HALVES, False, "heads", 0, 0),
]


def angles(most, half):
    a = np.arange(most)[:, None] / 10000.0 ** (np.arange(max(half, 1)) / max(half, 1))[None, :]
    return np.cos(a).astype(np.float32)[:, :half], np.sin(a).astype(np.float32)[:, :half]


def check_queries(y, q, stored, position, cos, sin, pairs, rotary):
    """Two products and their sum in F32: 2^-23 of the products' sizes; then an F16 row's rounding."""
    for i in np.flatnonzero(stored):
        c, s = (cos[position[i]], sin[position[i]]) if rotary else ((), ())
        gold = turned(q[i], np.asarray(c), np.asarray(s), pairs)
        size = turned(np.abs(q[i]), np.abs(np.asarray(c)), -np.abs(np.asarray(s)), pairs) + np.abs(
            turned(np.abs(q[i]), np.abs(np.asarray(c)), np.abs(np.asarray(s)), pairs)) + np.abs(gold)
        tol = 2.0 ** -23 * size + (2.0 ** -11 * np.abs(gold) * 1.01 + 2.0 ** -25 if y.dtype == np.float16 else 0)
        assert np.all(np.abs(y[i].astype(np.float64) - gold) <= tol)
    assert np.all(y[~stored] == np.array(GUARD, y.dtype)) or np.array_equal(y[~stored], q[~stored])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(gpu, case, in_place):
    parts, heads, query_heads, width, page_tokens, block, rotary, pairs, half, order, pad, offset = APPEND[case]
    rng = np.random.default_rng(4000 + case)
    lengths = [a + b for a, b in parts]
    row_pages = -(-max(lengths) // page_tokens) + 1
    pages = sum(-(-n // page_tokens) for n in lengths) + 2
    cache = CacheF8(rng, pages, page_tokens, heads, width, block, order, pad)
    table = table_of(rng, lengths, page_tokens, pages, row_pages)
    sequence = np.concatenate([np.full(n, s) for s, (_, n) in enumerate(parts)])
    position = np.concatenate([np.arange(a, a + n) for a, n in parts])
    dtype = np.float16 if half else np.float32
    tokens = len(sequence)
    # sizes that differ from token to token, so that scales grow and stay
    size = 2.0 ** rng.integers(-4, 5, (tokens, 1, 1))
    q, k, v = ((rng.standard_normal((tokens, h, width)) * size).astype(dtype) for h in (query_heads, heads, heads))
    cos, sin = angles(max(lengths), rotary // 2)
    model = cache.copy()
    stored, status = model_append(model, table, sequence, position, k, v, cos, sin, pairs, rotary)
    assert stored.all() and status == 0
    cache.upload()
    y = run_append(cache, table, sequence, position, q, k, v, cos, sin, pairs, rotary, pad=4 * pad, offset=offset,
                   in_place=in_place)
    cache.download()
    assert cache.same_as(model)
    check_queries(y, q, stored, position, cos, sin, pairs, rotary)
    assert gpu.kv_cache_status(0) == 0
    # read back, every token of every sequence in any order
    order_of = rng.permutation(sum(lengths))
    all_s = np.concatenate([np.full(n, s) for s, n in enumerate(lengths)])[order_of]
    all_p = np.concatenate([np.arange(n) for n in lengths])[order_of]
    for kind, common in ((dtype, False), (np.float32, True)):
        got = run_read(cache, table, all_s, all_p, kind, pad=2 * pad, offset=offset, common=common)
        for a, b in zip(got, model_read(model, table, all_s, all_p, kind)):
            assert np.array_equal(a, b, equal_nan=True)
    assert gpu.kv_cache_status(0) == 0


@pytest.mark.parametrize("block,width", [(16, 128), (64, 256), (4, 40), (1, 64)])
def test_append_token_by_token(gpu, block, width):
    """A block filled one token at a time, with sizes that grow and fall; then rolled back and written on."""
    rng = np.random.default_rng(12)
    heads, page_tokens = 2, 64
    cache = CacheF8(rng, 4, page_tokens, heads, width, block)
    table = table_of(rng, [100], page_tokens, 4, 2)
    model = cache.copy()
    cache.upload()
    kernel = kl.Kernel()
    cos, sin = angles(128, width // 2)
    # (position 40 comes again after the roll-back)
    for p in list(range(70)) + list(range(40, 60)):
        size = 2.0 ** (rng.integers(-12, 12) if p % 3 == 0 else 0)
        k, v = ((rng.standard_normal((1, heads, width)) * size).astype(np.float32) for _ in range(2))
        model_append(model, table, [0], [p], k, v, cos, sin, HALVES, width)
        run_append(cache, table, [0], [p], None, k, v, cos, sin, HALVES, width, kernel=kernel)
        cache.download()
        assert cache.same_as(model), p
    assert gpu.kv_cache_status(0) == 0


def test_append_at_once_or_one_by_one(gpu):
    """The same block either way, where codes stay above the subnormal ones."""
    rng = np.random.default_rng(13)
    x = rng.choice([-1.0, 1.0], (2, 32, 2, 64)) * rng.uniform(1, 40, (2, 32, 2, 64))
    k, v = x.astype(np.float32)
    table = np.array([[1, 0]], np.int32)
    caches = [CacheF8(np.random.default_rng(0), 2, 16, 2, 64, 16) for _ in range(2)]
    for cache in caches:
        cache.upload()
    run_append(caches[0], table, np.zeros(32, int), np.arange(32), None, k, v, (), (), HALVES, 0)
    for t in range(32):
        run_append(caches[1], table, [0], [t], None, k[t:t + 1], v[t:t + 1], (), (), HALVES, 0)
    for cache in caches:
        cache.download()
    assert caches[0].same_as(caches[1])


def test_append_values_at_the_ends(gpu):
    """Zeros, the smallest and largest F32 values, borders of a scale, ties; rounding to the nearest code, once."""
    rng = np.random.default_rng(14)
    width, rows = 64, []
    rows.append(np.zeros(width))
    rows.append(np.full(width, -0.0))
    rows.append(np.full(width, 1e-45))
    rows.append(np.full(width, 3.4028234e38))
    rows.append(np.where(np.arange(width) == 9, 2.0 ** -70, 2.0 ** -74))
    for top in (448.0, np.nextafter(np.float32(448), np.float32(500)), np.nextafter(np.float32(448), np.float32(0)), 1.75, 1.0):
        x = rng.standard_normal(width)
        x[0] = top
        rows.append(np.clip(x, -top, top))
    middles = (VALUES[:126] + VALUES[1:127]) / 2       # half way between codes, and one F32 step off it
    for i in range(0, 126, 42):
        for x in (middles[i:i + 42], np.nextafter(middles[i:i + 42].astype(np.float32), np.float32(0)),
                  np.nextafter(middles[i:i + 42].astype(np.float32), np.float32(500))):
            rows.append(np.concatenate([[448], x, -x])[:width])
    k = np.array(rows, np.float32)[:, None, :]
    v = -k[::-1]
    n = len(rows)
    table = np.array([list(range(-(-n // 16)))], np.int32)
    for block in (1, 2, 16):
        cache = CacheF8(rng, table.shape[1], 16, 1, width, block)
        model = cache.copy()
        cache.upload()
        model_append(model, table, np.zeros(n, int), np.arange(n), k, v, (), (), HALVES, 0)
        run_append(cache, table, np.zeros(n, int), np.arange(n), None, k, v, (), (), HALVES, 0)
        cache.download()
        assert cache.same_as(model)


def test_append_rounds_the_rotation_once(gpu):
    """Turned keys that F32 would put on a tie: 1 + 2^-4 and a little, from products that F32 rounds away."""
    width, n = 8, 64
    rng = np.random.default_rng(15)
    k = np.zeros((n, 1, width), np.float32)
    cos, sin = np.ones((n, 4), np.float32), np.zeros((n, 4), np.float32)
    k[:, 0, 7] = 448
    for t in range(n):
        tie = np.float32((8 + t % 8 + 0.5) / 8)
        k[t, 0, 0], k[t, 0, 4] = tie, rng.choice([-1, 1]) * 2.0 ** -20
        sin[t, 0] = rng.choice([-1, 1]) * 2.0 ** -20          # +-2^-40 beside the tie
    cache = CacheF8(rng, 4, 16, 1, width, 16)
    model = cache.copy()
    cache.upload()
    table = np.array([[3, 1, 0, 2]], np.int32)
    args = (np.zeros(n, int), np.arange(n))
    model_append(model, table, *args, k, k, cos, sin, HALVES, 8)
    run_append(cache, table, *args, None, k, k, cos, sin, HALVES, 8)
    cache.download()
    assert cache.same_as(model)
    up = VALUES[cache.k[0, table[0, np.arange(n) // 16], 0, np.arange(n) % 16, 0]] > k[:, 0, 0]
    assert up.any() and not up.all()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("block", [1, 8, 16, 64])
def test_append_not_finite(gpu, bad, block):
    """The block reads as not a number, alone, until it is begun again."""
    rng = np.random.default_rng(16)
    cache = CacheF8(rng, 2, 64, 2, 128, block)
    table = np.array([[1, 0]], np.int32)
    model = cache.copy()
    cache.upload()
    for step, (first, count, spoiled) in enumerate(((0, 20, -1), (20, 3, 21), (23, 10, -1), (20 // block * block, 30, -1))):
        k, v = (rng.standard_normal((count, 2, 128)).astype(np.float32) for _ in range(2))
        if spoiled >= 0:
            k[spoiled - first, 1, 7] = bad
            v[spoiled - first, 0, 127] = bad
        at = (np.zeros(count, int), np.arange(first, first + count))
        model_append(model, table, *at, k, v, (), (), HALVES, 0)
        run_append(cache, table, *at, None, k, v, (), (), HALVES, 0)
        cache.download()
        assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(cache.scales, model.scales))
        n = first + count
        got, want = run_read(cache, table, np.zeros(n, int), np.arange(n), np.float32), model_read(
            model, table, np.zeros(n, int), np.arange(n), np.float32)
        for a, b in zip(got, want):
            assert np.array_equal(a, b, equal_nan=True)
        nan_blocks = np.isnan(cache.ks[0, 1]).sum()
        # the spoiled block lasts until its first token comes again
        assert nan_blocks == (1 if step in (1, 2) else 0)


def test_append_over_other_scales(gpu):
    """Earlier tokens' scales that are no powers of two (or 0) are kept or grow to one; values stay within a code's half step."""
    rng = np.random.default_rng(17)
    cache = CacheF8(rng, 1, 64, 4, 128, 16)
    cache.ks[...] = rng.uniform(0.001, 0.1, cache.ks.shape)
    cache.vs[...] = rng.uniform(0.001, 0.1, cache.vs.shape)
    cache.ks[0, 0, 1] = 0
    before = cache.copy()
    table = np.zeros((4, 1), np.int32)
    cache.upload()
    at = np.array([9, 25, 41, 57])
    k, v = (rng.standard_normal((4, 4, 128)).astype(np.float32) * np.array([1, 4, 16, 64], np.float32)[:, None, None]
            for _ in range(2))
    run_append(cache, table, np.arange(4), at, None, k, v, (), (), HALVES, 0)
    cache.download()
    for pool, x, old, new in (("k", k, before.ks, cache.ks), ("v", v, before.vs, cache.vs)):
        top = np.abs(x).max(2).T                                       # [head][block]
        least = 2.0 ** np.ceil(np.log2(top / 448))
        want = np.maximum(old[0, 0].astype(np.float64), least)
        assert np.array_equal(new[0, 0], want.astype(np.float32))
        values, earlier = cache.values(pool)[0, 0], before.values(pool)[0, 0]
        for b in range(4):
            step = want[:, b, None] * 2.0 ** -10                       # half the least step between codes
            got = values[:, at[b]]
            assert np.all(np.abs(got - x[b]) <= np.maximum(np.abs(x[b]) * (2.0 ** -4 + 2.0 ** -20), step))
            was = earlier[:, b * 16:at[b]]
            assert np.all(np.abs(values[:, b * 16:at[b]] - was) <=
                          np.maximum(np.abs(was) * (2.0 ** -4 + 2.0 ** -20), step[..., None]))


def test_append_newest_and_left_out(gpu):
    """Without lists the newest token of each sequence; negative entries are left out, others out of range reported."""
    rng = np.random.default_rng(18)
    heads, width, page_tokens, block = 2, 64, 16, 8
    lengths = np.array([1, 17, 0, 24, 40], np.int32)
    cache = CacheF8(rng, 20, page_tokens, heads, width, block)
    table = table_of(rng, lengths, page_tokens, 20, 3)
    cos, sin = angles(48, 32)
    q, k, v = (rng.standard_normal((5, h, width)).astype(np.float32) for h in (4, heads, heads))
    model = cache.copy()
    stored, _ = model_append(model, table, range(5), lengths - 1, k, v, cos, sin, ADJACENT, 64)
    assert list(stored) == [True, True, False, True, True]
    cache.upload()
    y = run_append(cache, table, None, None, q, k, v, cos, sin, ADJACENT, 64, lengths=lengths)
    cache.download()
    assert cache.same_as(model) and gpu.kv_cache_status(0) == 0
    check_queries(y, q, stored, lengths - 1, cos, sin, ADJACENT, 64)
    newest = run_read(cache, table, None, None, np.float32, lengths=lengths)
    keep = lengths > 0
    for a, b in zip(newest, model_read(model, table, np.arange(5)[keep], lengths[keep] - 1, np.float32)):
        assert np.array_equal(a[keep], b) and np.all(a[~keep] == np.float32(GUARD))
    # lists with gaps: a run of sequence 4's tokens with one left out, sequences and positions out of range, a page that is not there
    table[3, 1] = 20
    sequence = np.array([4, 4, 4, -1, 4, 5, 1, 1, 1, 3, 3, 0, 0, 2 ** 30, 1])
    position = np.array([30, 31, 32, 33, 34, 0, 46, 47, 48, 15, 16, -1, 0, 3, 2 ** 30])
    table[1, 2] = [p for p in range(20) if p not in table][0]
    n = len(sequence)
    q, k, v = (rng.standard_normal((n, h, width)).astype(np.float32) for h in (4, heads, heads))
    stored, status = model_append(model, table, sequence, position, k, v, cos, sin, ADJACENT, 64)
    assert status == kl.KV_BAD_INDEX | kl.KV_BAD_PAGE and stored.sum() == 4 + 2 + 1 + 1
    cache.upload()
    y = run_append(cache, table, sequence, position, q, k, v, cos, sin, ADJACENT, 64)
    assert gpu.kv_cache_status(0) == status
    cache.download()
    assert cache.same_as(model)
    check_queries(y, q, stored, position, cos, sin, ADJACENT, 64)
    got = run_read(cache, table, sequence, position, np.float16)
    assert gpu.kv_cache_status(0) == status
    for a, b in zip(got, model_read(model, table, sequence[stored], position[stored], np.float16)):
        assert np.array_equal(a[stored], b) and np.all(a[~stored] == np.float16(GUARD))


def test_append_two_blocks_of_one_call(gpu):
    """Runs of one sequence that begin and end inside blocks, of several sequences in turn."""
    rng = np.random.default_rng(19)
    cache = CacheF8(rng, 12, 32, 2, 96, 16, "tokens")
    lengths = [60, 60, 60]
    table = table_of(rng, lengths, 32, 12, 2)
    sequence = np.concatenate([np.full(9, 1), np.full(20, 0), np.full(1, 2), np.full(30, 1)])
    position = np.concatenate([np.arange(3, 12), np.arange(14, 34), [33], np.arange(16, 46)])
    k, v = ((rng.standard_normal((60, 2, 96)) * 2.0 ** rng.integers(-6, 6, (60, 1, 1))).astype(np.float16) for _ in range(2))
    cos, sin = angles(60, 48)
    model = cache.copy()
    model_append(model, table, sequence, position, k, v, cos, sin, HALVES, 96)
    cache.upload()
    run_append(cache, table, sequence, position, None, k, v, cos, sin, HALVES, 96)
    cache.download()
    assert cache.same_as(model) and gpu.kv_cache_status(0) == 0


def test_read_rounds_once(gpu):
    """F16 rows: values past its range are infinite, small ones subnormal, scales that are no powers of two."""
    rng = np.random.default_rng(20)
    cache = CacheF8(rng, 2, 16, 1, 256, 4)
    cache.k[0, 0, 0] = np.arange(256, dtype=np.uint8)
    cache.ks[0, 0, 0] = [1.0, 300.0, 1e-7, 0.3]
    cache.vs[0, 0, 0] = [np.nan, np.inf, 0.0, -1.5]
    cache.upload()
    table = np.array([[0, 1]], np.int32)
    s, p = np.zeros(16, int), np.arange(16)
    with np.errstate(invalid="ignore"):
        for dtype in (np.float16, np.float32):
            for a, b in zip(run_read(cache, table, s, p, dtype), model_read(cache, table, s, p, dtype)):
                assert np.array_equal(a, b, equal_nan=True)


# --- pages ------------------------------------------------------------------------------------

PAGES = [(1, 4, 64, 16, 16, "heads", 0), (3, 2, 128, 32, 4, "tokens", 0), (2, 3, 40, 12, 2, "heads", 1),
         (2, 5, 80, 20, 1, "tokens", 0), (1, 1, 8, 1, 1, "heads", 0), (2, 2, 96, 64, 64, "heads", 2)]


@pytest.mark.parametrize("case", range(len(PAGES)))
def test_pages_life(gpu, case):
    """Forked, released, compacted and copied: tables and counts are those that the F16 cache's operations give, every
    sequence keeps its tokens' codes and scales, and nothing else changes."""
    layers, heads, width, page_tokens, block, order, pad = PAGES[case]
    rng = np.random.default_rng(5000 + case)
    rows, row_pages, pages = 9, 6, 40
    cache = CacheF8(rng, pages, page_tokens, heads, width, block, order, pad, layers)
    kv_pages = kl.KVPagesLayout(rows, row_pages, layers, cache.layer)
    assert kl.kv_pages_f8_reason(cache.layout, kv_pages) == ""
    lengths = rng.integers(1, row_pages * page_tokens + 1, rows).astype(np.int32)
    lengths[[5, 6, 7]] = 0
    while (-(-lengths // page_tokens)).sum() > pages - 8:
        lengths = np.maximum(lengths - page_tokens, np.minimum(lengths, 1)).astype(np.int32)
    table = table_of(rng, lengths, page_tokens, pages, row_pages)
    references = np.bincount(table[table >= 0], minlength=pages).astype(np.int32)
    pools = cache.upload()
    kernel = kl.Kernel()

    def state():
        return [b.download(x.shape, np.int32) for b, x in zip(tables, (table, lengths, references))]

    tables = [upload(x) for x in (table, lengths, references)]
    at = [b.data for b in tables]
    # the same tables over F16 pools, for what they become
    f16 = kl.KVCacheLayout(pages, page_tokens, heads, 8, heads * page_tokens * 8, page_tokens * 8, 8)
    f16_pages = kl.KVPagesLayout(rows, row_pages, 1, 0)
    f16_pools = [upload(np.zeros(pages * heads * page_tokens * 8, np.float16)) for _ in range(2)]
    twins = [upload(x) for x in (table, lengths, references)]
    twin_at = [b.data for b in twins]

    def tokens_of(c, t, n):
        """Every token's codes and scales of a sequence, layer by layer."""
        i = np.arange(n)
        page, where = t[i // page_tokens], i % page_tokens
        return [x[:, page, :, where].copy() for x in (c.k, c.v)] + [x[:, page, :, where // block].copy() for x in (c.ks, c.vs)]

    def same(a, b):
        return all(np.array_equal(x, y) for x, y in zip(a, b))

    kept = [tokens_of(cache, table[s], lengths[s]) for s in range(rows)]
    lists = [upload(np.array(x, np.int32)) for x in ([0, 0, 3], [5, 6, 7])]
    before = cache.copy()
    assert kl.kv_fork_f8(kernel, 0, *pools, *at, lists[0].data, lists[1].data, 3, cache.layout, kv_pages)
    assert kernel.route == "kv_fork_f8"
    assert kl.kv_fork(kernel, 0, f16_pools[0], f16_pools[1], *twin_at, lists[0].data, lists[1].data, 3, f16, f16_pages)
    finish()
    assert gpu.kv_cache_status(0) == 0
    t, n, r = state()
    for a, b in zip((t, n, r), twins):
        assert np.array_equal(a, b.download(a.shape, np.int32))
    cache.download()
    for child, parent in ((5, 0), (6, 0), (7, 3)):
        kept[child] = kept[parent]
    for s in range(rows):
        assert same(tokens_of(cache, t[s], n[s]), kept[s]), s
    fresh = references == 0
    old_pages = np.flatnonzero(~fresh)
    for a, b in zip((cache.k, cache.v, cache.ks, cache.vs), (before.k, before.v, before.ks, before.vs)):
        assert np.array_equal(a[:, old_pages], b[:, old_pages])

    # release some, compact
    gone = upload(np.array([0, 4], np.int32))
    assert kl.kv_free(kernel, 0, *at, gone.data, 2, cache.layout.cache, kv_pages)
    assert kl.kv_free(kernel, 0, *twin_at, gone.data, 2, f16, f16_pages)
    used, used_twin = upload(np.zeros(1, np.int32)), upload(np.zeros(1, np.int32))
    assert kl.kv_compact_f8(kernel, 0, *pools, at[0], at[2], used.data, *at, cache.layout, kv_pages)
    assert kernel.route == "kv_compact_f8"
    assert kl.kv_compact(kernel, 0, f16_pools[0], f16_pools[1], twin_at[0], twin_at[2], used_twin.data, *twin_at, f16, f16_pages)
    finish()
    assert gpu.kv_cache_status(0) == 0
    t, n, r = state()
    for a, b in zip((t, n, r), twins):
        assert np.array_equal(a, b.download(a.shape, np.int32))
    total = int(used.download(1, np.int32)[0])
    assert total == int(used_twin.download(1, np.int32)[0]) == (r > 0).sum() and (r[:total] > 0).all()
    cache.download()
    for s in range(rows):
        if n[s]:
            assert same(tokens_of(cache, t[s], n[s]), kept[s]), s

    # copies, padding and all other pages left alone
    before = cache.copy()
    source, target = np.array([0, -1, 1], np.int32), np.array([pages - 1, 3, pages - 3], np.int32)
    lists = [upload(source), upload(target)]
    assert kl.kv_copy_pages_f8(kernel, 0, *pools, lists[0].data, lists[1].data, 3, cache.layout, kv_pages)
    finish()
    cache.download()
    for a, b in ((0, pages - 1), (1, pages - 3)):
        for x in (before.k, before.v, before.ks, before.vs):
            x[:, b] = x[:, a]
    assert cache.same_as(before)
    assert gpu.kv_cache_status(0) == 0


def test_decoding_over_forks(gpu):
    """Append, attention, fork, release and compaction in turn, as a server uses them, against a model that keeps every
    sequence's codes by itself."""
    rng = np.random.default_rng(21)
    rows, row_pages, pages, heads, query_heads, width, page_tokens, block = 5, 8, 30, 2, 4, 64, 16, 8
    cache = CacheF8(rng, pages, page_tokens, heads, width, block)
    model = CacheF8(rng, rows * row_pages, page_tokens, heads, width, block)   # row s owns pages s * row_pages..
    own = np.arange(rows * row_pages, dtype=np.int32).reshape(rows, row_pages)
    pools = cache.upload()
    table, lengths, references = (upload(np.full((rows, row_pages), -1, np.int32)), upload(np.zeros(rows, np.int32)),
                                  upload(np.zeros(pages, np.int32)))
    every = upload(np.arange(rows, dtype=np.int32))
    kv_pages = kl.KVPagesLayout(rows, row_pages, 1, 0)
    kernel, n = kl.Kernel(), np.zeros(rows, int)
    cos, sin = angles(row_pages * page_tokens, width // 2)

    def step(added):
        wanted = upload(np.asarray(added, np.int32))
        assert kl.kv_reserve(kernel, 0, table.data, lengths.data, references.data, every.data, wanted.data, rows,
                             cache.layout.cache, kv_pages)
        finish()
        t = table.download((rows, row_pages), np.int32)
        sequence = np.repeat(np.arange(rows), added)
        position = np.concatenate([np.arange(a, a + b) for a, b in zip(n, added)])
        n[:] += added
        q = rng.standard_normal((rows, query_heads, width)).astype(np.float32)
        k, v = ((rng.standard_normal((len(sequence), heads, width)) * 2.0 ** rng.integers(-2, 3)).astype(np.float32)
                for _ in range(2))
        run_append(cache, t, sequence, position, None, k, v, cos, sin, HALVES, width, kernel=kernel)
        model_append(model, own, sequence, position, k, v, cos, sin, HALVES, width)
        call = kl.PagedAttentionLayout(rows, query_heads, row_pages * page_tokens, 0, row_pages, 256, 256, 0.125, kl.InputType.f32)
        y, q_buffer = upload(np.zeros_like(q)), upload(q)
        assert kl.paged_attention_f8(kernel, 0, y.data, q_buffer.data, *pools, table.data, lengths.data, cache.layout, call)
        finish()
        assert gpu.kv_cache_status(0) == 0
        gold, tol = gold_attention(model, own, n, q, 0, 0.125)
        check(y.download(q.shape, np.float32), gold, tol)

    def take_over(child, parent):
        n[child] = n[parent]
        for x in (model.k, model.v, model.ks, model.vs):
            x[0, own[child]] = x[0, own[parent]]

    step([20, 7, 0, 0, 33])
    for _ in range(5):
        step([1, 1, 0, 0, 1])
    lists = [upload(np.array(x, np.int32)) for x in ([0, 4, 0], [2, 3, 1])]
    assert kl.kv_fork_f8(kernel, 0, *pools, table.data, lengths.data, references.data, lists[0].data, lists[1].data, 3,
                         cache.layout, kv_pages)
    for child, parent in ((2, 0), (3, 4), (1, 0)):
        take_over(child, parent)
    for _ in range(10):
        step([1, 1, 1, 1, 1])
    gone = upload(np.array([0, 3], np.int32))
    assert kl.kv_free(kernel, 0, table.data, lengths.data, references.data, gone.data, 2, cache.layout.cache, kv_pages)
    n[[0, 3]] = 0
    used = upload(np.zeros(1, np.int32))
    assert kl.kv_compact_f8(kernel, 0, *pools, table.data, references.data, used.data, table.data, lengths.data,
                            references.data, cache.layout, kv_pages)
    for _ in range(4):
        step([2, 1, 1, 0, 3])
