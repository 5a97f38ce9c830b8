"""The paged cache's and the logits step's contracts where lists, weights and infinities go to their ends:
entries that are refused or named twice, tokens of very small weight, what is left out."""
import numpy as np
import pytest

import kunlunk200_lib_amd as kl
from test_gpu_kv_cache import F16, F32, GUARD, Book, Cache, finish, lists, run_attention, table_of, upload

pytestmark = pytest.mark.gpu


# --- kv_reserve and kv_fork: lists ----------------------------------------------------------

def reserve_rule(book, rows, added):
    """In list order: an entry out of range is left out, of those that name one sequence the first counts, and
    one that counts is granted if its pages are there. Returns the status."""
    status, seen = 0, set()
    free = list(np.flatnonzero(book.references == 0))
    sequences, row_pages = book.table.shape
    for r, a in zip(rows, added):
        if not 0 <= r < sequences or a < 0 or book.lengths[r] + a > row_pages * book.pt and r not in seen or r in seen:
            status |= kl.KV_BAD_INDEX
            continue
        seen.add(r)
        held, need = book.held(book.lengths[r]), book.held(book.lengths[r] + a)
        if need - held > len(free):
            status |= kl.KV_NO_PAGE
            continue
        for j in range(held, need):
            page = free.pop(0)
            book.table[r, j], book.references[page] = page, 1
        book.lengths[r] += a
    return status


def reserve(book, rows, added):
    r, a = lists(rows, added)
    status = reserve_rule(book, rows, added)
    assert kl.kv_reserve(book.kernel, 0, *book.p, r.data, a.data, len(rows), book.cache.layout, book.pages)
    book.check(status)
    return status


def book_of(seed, sequences, row_pages, pages, pt):
    book = Book(np.random.default_rng(seed), sequences, row_pages, pages, pt, heads=1, width=8, layers=1)
    book.upload()
    return book


def test_reserve_first_of_a_sequence_counts(gpu):
    """The entries left out take no pages: six are free and six are asked for by those that count."""
    book = book_of(1, 4, 5, 6, 8)
    assert reserve(book, [1, 1, 0], [30, 25, 9]) == kl.KV_BAD_INDEX
    assert book.lengths.tolist() == [9, 30, 0, 0] and book.table[0].tolist() == [4, 5, -1, -1, -1]


def test_reserve_first_in_range_counts(gpu):
    """An entry out of range is not the first of its sequence."""
    book = book_of(2, 4, 5, 24, 8)
    assert reserve(book, [2, 2, 9, 2], [41, 10, 3, 17]) == kl.KV_BAD_INDEX
    assert book.lengths.tolist() == [0, 0, 10, 0]


@pytest.mark.parametrize("sequences", [300, 3000, 6000])
def test_reserve_named_twice_in_long_lists(gpu, sequences):
    rng = np.random.default_rng(sequences)
    book = book_of(3, sequences, 4, 4 * sequences, 8)
    for _ in range(3):
        rows = rng.integers(0, sequences, sequences)
        added = rng.integers(0, 32, sequences)
        assert reserve(book, rows, added) == kl.KV_BAD_INDEX


@pytest.mark.parametrize("needs,granted", [
    ([20, 1], [1]), ([100, 1], [1]), ([4, 7, 6, 1], [0, 2]), ([10, 1, 1], [0]), ([3, 8, 8, 7, 1], [0, 3]),
    ([1, 10, 2, 9, 3, 8, 4, 7], [0, 2, 4, 6]), ([11, 12, 13], [])])
def test_reserve_refused_take_no_pages(gpu, needs, granted):
    """Ten pages are free; an entry that does not fit leaves them to those after it."""
    book = book_of(4, len(needs) + 1, 128, 10, 4)
    book_rows = np.arange(len(needs))
    assert bool(reserve(book, book_rows, [4 * n for n in needs]) & kl.KV_NO_PAGE) == (len(granted) < len(needs))
    assert np.flatnonzero(book.lengths).tolist() == granted


@pytest.mark.parametrize("sequences,pages,most", [(70, 60, 9), (1500, 900, 2), (2500, 3000, 40), (5000, 20000, 8)])
def test_reserve_short_of_pages(gpu, sequences, pages, most):
    """Lists that ask for more than there is, over several steps of the plan, some of them named twice or out of range."""
    rng = np.random.default_rng(pages)
    book = book_of(5, sequences, 3 * most, pages, 4)
    for turn in range(4):
        n = int(rng.integers(sequences // 2, sequences + 1))
        rows = rng.permutation(sequences)[:n]
        if turn % 2:
            rows[rng.integers(0, n, n // 10)] = rng.integers(-1, sequences + 1, n // 10)
        added = rng.integers(0, 4 * most, n)
        added[rng.integers(0, n, n // 20)] = 4 * 3 * most
        reserve(book, rows, added)
        rows = rng.permutation(sequences)[: sequences // 4]
        book.free(rows)
        r, = lists(rows)
        assert kl.kv_free(book.kernel, 0, *book.p, r.data, len(rows), book.cache.layout, book.pages)
        book.check()


def fork(book, parents, children):
    p, c = lists(parents, children)
    first = [i for i, child in enumerate(children) if child not in children[:i]]
    book.fork(np.array(parents)[first], np.array(children)[first])
    assert kl.kv_fork(book.kernel, 0, *book.pools, *book.p, p.data, c.data, len(parents), book.cache.layout, book.pages)
    book.check(kl.KV_BAD_INDEX if len(first) < len(parents) else 0)


def test_fork_first_to_a_child_counts(gpu):
    """The forks left out take no pages: two are free and two forks that count need one each."""
    book = book_of(6, 4, 5, 10, 8)
    reserve(book, [0, 1], [30, 25])
    fork(book, [0, 1, 0], [2, 2, 3])
    assert book.lengths.tolist() == [30, 25, 30, 30] and np.all(book.references[:10] > 0)


def test_fork_named_twice_in_long_lists(gpu):
    rng = np.random.default_rng(61)
    book = book_of(7, 2600, 3, 12000, 8)
    reserve(book, np.arange(2600), rng.integers(0, 25, 2600))
    for _ in range(3):
        fork(book, rng.integers(0, 2600, 2500).tolist(), rng.integers(0, 2600, 2500).tolist())


def test_free_list_past_a_grid(gpu):
    """More sequences than one launch dimension of whole workgroups holds."""
    sequences = (1 << 24) + 70
    layout = kl.KVCacheLayout(8, 16, 1, 8, 128, 128, 8)
    pages = kl.KVPagesLayout(sequences, 1, 1, 0)
    table, lengths = np.full((sequences, 1), -1, np.int32), np.zeros(sequences, np.int32)
    at = [0, 5, 1 << 23, sequences - 1]
    table[at, 0], lengths[at] = [3, 1, 3, 7], 9
    references = np.bincount([3, 1, 3, 7], minlength=8).astype(np.int32)
    b = [upload(x) for x in (table, lengths, references, np.arange(sequences, dtype=np.int32))]
    assert kl.kv_free(kl.Kernel(), 0, *[x.data for x in b], sequences, layout, pages)
    assert kl.kv_cache_status(0) == 0
    assert not b[1].download(sequences, np.int32).any() and not b[2].download(8, np.int32).any()
    assert np.all(b[0].download(sequences, np.int32) == -1)


# --- paged_attention: weights and infinities --------------------------------------------------

@pytest.mark.parametrize("heads,query_heads,width,page_tokens,longest", [
    (8, 8, 64, 16, 40), (8, 8, 128, 20, 40), (1, 16, 64, 16, 40), (8, 8, 128, 16, 2816)])
def test_attention_weights_in_f32(gpu, heads, query_heads, width, page_tokens, longest):
    """Weights near the row's largest are as good as an F32 exponential.

    Values of +1 and -1 make every sum of products exact (parts are multiples of 2^-10 up to 2^14 each), scores below
    2^-10 leave weights within [0.998, 1]: exponential 1 ulp, 2^-24; the weight's parts 2^-10 / 2^14 = 2^-24 of the largest.
    Scores: a = sum |q k|, e_s = a (2^-22 + (width + 3) 2^-24) twice (subtracted from the largest). Quotient: 2^-24 |y|,
    and |y| <= 1."""
    rng = np.random.default_rng(81)
    lengths = [int(n) for n in rng.integers(1, 17, 64) * 2]
    pages = sum(-(-n // page_tokens) for n in lengths) + 1
    cache = Cache(rng, pages, page_tokens, heads, width)
    table = table_of(rng, lengths, page_tokens, pages, -(-longest // page_tokens))
    for s, n in enumerate(lengths):
        for t in range(n):
            cache.v[0, table[s, t // page_tokens], :, t % page_tokens] = 1 - 2 * (t % 2)
    q = (rng.standard_normal((64, query_heads, width)) * 2.0 ** -17).astype(np.float32)
    y, _ = run_attention(cache, table, lengths, q, scale=1.0, longest=longest)
    for s, n in enumerate(lengths):
        t = np.arange(n)
        for h in range(query_heads):
            k = cache.k[0, table[s, t // page_tokens], h * heads // query_heads, t % page_tokens].astype(np.float64)
            score = k @ q[s, h].astype(np.float64)
            assert np.abs(score).max() < 2.0 ** -10
            p = np.exp(score - score.max())
            gold = (p * (1 - 2 * (t % 2))).sum() / p.sum()
            a = np.abs(k * q[s, h]).sum(1).max()
            tol = 2.0 ** -24 * (1 + 1 + abs(gold)) + 2 * a * (2.0 ** -22 + (width + 3) * 2.0 ** -24)
            assert np.abs(y[s, h] - gold).max() <= tol, (s, h, np.abs(y[s, h] - gold).max(), tol)


# heads, query heads, width, tokens of a page, length, `longest`, order: whole rows, column tiles, split, equal shares
ROUTES = [
    (2, 4, 64, 16, 60, 60, "heads"),
    (2, 4, 72, 20, 60, 60, "tokens"),
    (1, 16, 128, 16, 60, 60, "heads"),
    (2, 2, 256, 16, 60, 60, "heads"),
    (1, 2, 128, 16, 3000, 3000, "heads"),
    (8, 8, 128, 16, 700, 2816, "heads"),
]


def one_score_cache(rng, heads, width, page_tokens, n, order, score):
    """A cache of one sequence (the first of eight) whose key t gives `score[t]` to the query (1, 0, ...)."""
    cache = Cache(rng, -(-n // page_tokens) + 1, page_tokens, heads, width, order)
    table = table_of(rng, [n], page_tokens, cache.layout.pages, -(-n // page_tokens))
    t = np.arange(n)
    place = (0, table[0, t // page_tokens], slice(None), t % page_tokens)
    cache.k[place] = 0
    cache.k[place + (0,)] = np.float16(score)[:, None]
    return cache, table, place


def run_one(cache, table, n, q, longest):
    """The row of one sequence, beside seven empty ones where `longest` is more (so that it is shared out)."""
    beside = 7 if longest > n else 0
    row_pages = -(-longest // cache.layout.page_tokens)
    rows = np.full((1 + beside, row_pages), -1, np.int32)
    rows[0, :table.shape[1]] = table[0]
    y, route = run_attention(cache, rows, [n] + [0] * beside, np.repeat(q[None], 1 + beside, 0), scale=1.0,
                             longest=longest)
    assert not beside or route == "paged_attention_even"
    return y[0]


@pytest.mark.parametrize("route", range(len(ROUTES)))
@pytest.mark.parametrize("gap", [20, 30, 45, 60, 80])
@pytest.mark.parametrize("first", [False, True])
def test_attention_infinite_values_of_small_weight(gpu, route, gap, first):
    """An infinite value whose weight is e^-gap of the row's largest, far below what its F16 parts hold, gives its
    infinity, before and after the largest; the other columns stay what they are."""
    heads, query_heads, width, page_tokens, n, longest, order = ROUTES[route]
    rng = np.random.default_rng(82)
    score = np.full(n, -float(gap))
    heavy = n - 1 if first else 0
    score[heavy] = 0.0
    cache, table, place = one_score_cache(rng, heads, width, page_tokens, n, order, score)
    for t, d, x in ((n // 2, 3, np.inf), (n // 3, 4, -np.inf), (5, 5, np.inf), (n - 7, 5, -np.inf), (17, 6, np.nan)):
        cache.v[0, place[1][t], :, place[3][t], d] = x
    q = np.zeros((query_heads, width), np.float32)
    q[:, 0] = 1.0
    y = run_one(cache, table, n, q, longest)
    assert np.all(y[:, 3] == np.inf) and np.all(y[:, 4] == -np.inf) and np.all(np.isnan(y[:, 5:7]))
    p = np.exp(score)
    v = cache.v[place].astype(np.float64)                                   # [token, head, value]
    others = [d for d in range(width) if not 3 <= d <= 6]
    for h in range(query_heads):
        x = v[:, h * heads // query_heads][:, others]
        gold, size = p @ x / p.sum(), p @ np.abs(x) / p.sum()
        # the scores are exact but for their factor (up to gap * 2^-22); parts below 2^-38 of the largest weight are lost
        tol = size * (2 * gap * 2.0 ** -22 + 2.0 ** -20 + 2 * n * 2.0 ** -24) + 2.0 ** -38 * np.abs(x).sum(0)
        assert np.all(np.abs(y[h, others] - gold) <= tol)


@pytest.mark.parametrize("route", range(len(ROUTES)))
def test_attention_infinite_values_of_no_weight(gpu, route):
    """A weight below the smallest F32 number is 0, and 0 times infinity not a number, as products of F32 have it."""
    heads, query_heads, width, page_tokens, n, longest, order = ROUTES[route]
    rng = np.random.default_rng(83)
    score = np.full(n, -120.0)
    score[n // 4] = 0.0
    cache, table, place = one_score_cache(rng, heads, width, page_tokens, n, order, score)
    for t, d in ((2, 3), (n - 2, 4)):
        cache.v[0, place[1][t], :, place[3][t], d] = np.inf
    q = np.zeros((query_heads, width), np.float32)
    q[:, 0] = 1.0
    y = run_one(cache, table, n, q, longest)
    odd = np.zeros(width, bool)
    odd[3:5] = True
    assert np.all(np.isnan(y[:, odd])) and np.all(np.isfinite(y[:, ~odd]))


@pytest.mark.parametrize("route", range(len(ROUTES)))
@pytest.mark.parametrize("small", [1e-6, -1e-12, 1e-30])
def test_attention_infinite_keys_under_small_queries(gpu, route, small):
    """An infinite key gives its infinity to the score however small the query's value beside the others is."""
    heads, query_heads, width, page_tokens, n, longest, order = ROUTES[route]
    rng = np.random.default_rng(84)
    score = rng.integers(-16, 17, n) / 8.0
    cache, table, place = one_score_cache(rng, heads, width, page_tokens, n, order, score)
    gone = [3, n // 2, n - 1]
    for t in gone:
        cache.k[0, place[1][t], :, place[3][t], 1] = -np.inf * np.sign(small)
    q = np.zeros((query_heads, width), np.float32)
    q[:, 0], q[:, 1] = 1.0, small
    y = run_one(cache, table, n, q, longest)
    p = np.exp(score - score.max())
    p[gone] = 0
    v = cache.v[place].astype(np.float64)
    for h in range(query_heads):
        x = v[:, h * heads // query_heads]
        tol = (p @ np.abs(x)) / p.sum() * (2.0 ** -19 + 2 * n * 2.0 ** -24)
        assert np.all(np.abs(y[h] - p @ x / p.sum()) <= tol)
    cache.k[0, place[1][7], :, place[3][7], 1] = np.inf * np.sign(small)    # a score of +Inf: not a number
    assert np.all(np.isnan(run_one(cache, table, n, q, longest)))


@pytest.mark.parametrize("route", range(len(ROUTES)))
def test_attention_infinite_queries(gpu, route):
    """An infinite query value beside large finite ones: its infinity alone decides the scores."""
    heads, query_heads, width, page_tokens, n, longest, order = ROUTES[route]
    rng = np.random.default_rng(85)
    score = np.where(np.arange(n) % 3, -1.0, -2.0)
    cache, table, place = one_score_cache(rng, heads, width, page_tokens, n, order, score)
    cache.k[place + (1,)] = 1.0
    q = np.zeros((query_heads, width), np.float32)
    q[:, 0], q[:, 1] = np.inf, 1e30
    q[:, 2:] = 0.0
    cache.k[place + (slice(2, None),)] = 0
    y = run_one(cache, table, n, q, longest)
    assert np.all(y == 0)                                                  # every score -Inf
    cache.k[place + (0,)] = 1.0
    assert np.all(np.isnan(run_one(cache, table, n, q, longest)))          # every score +Inf


# --- kv_append ------------------------------------------------------------------------------

def test_append_without_queries_ignores_their_layout(gpu):
    rng = np.random.default_rng(91)
    cache = Cache(rng, 4, 16, 2, 64)
    rows = rng.standard_normal((3, 256)).astype(np.float32)
    k_pool, v_pool = cache.upload()
    r, s, p, t = upload(rows), *lists([0, 0, 0], [0, 5, 17], [[2, 1]])
    kernel = kl.Kernel()
    for query_heads, stride in ((4, 0), (5000, 0), (-1, -7), (4, 1 << 50)):
        call = kl.KVAppendLayout(3, 1, 2, query_heads, stride, 256, 256, stride, 0, 0, kl.RotaryPairs.adjacent, F32)
        assert kl.kv_append(kernel, 0, k_pool, v_pool, None, None, r.data, r.data + 512, s.data, p.data, None, t.data,
                            None, None, cache.layout, call), (query_heads, stride)
        assert kl.kv_cache_status(0) == 0
    _, (k, v) = cache.download()
    for i, (page, at) in enumerate(((2, 0), (2, 5), (1, 1))):
        assert np.array_equal(k[0, page, :, at], rows[i, :128].reshape(2, 64).astype(np.float16))
        assert np.array_equal(v[0, page, :, at], rows[i, 128:].reshape(2, 64).astype(np.float16))


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rotary,pairs", [(64, 0), (64, 1), (6, 0), (0, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_append_leaves_the_whole_token_out(gpu, half, rotary, pairs, in_place):
    """A token without a page is left out with its query, as one out of range is."""
    rng = np.random.default_rng(92)
    dtype = np.float16 if half else np.float32
    cache = Cache(rng, 4, 16, 2, 64)
    rows = rng.standard_normal((5, 512)).astype(dtype)                     # 4 query heads, 2 + 2
    k_pool, v_pool = cache.upload()
    r, out = upload(rows), upload(np.full((5, 256), GUARD, dtype))
    s, p, t = lists([0, 1, 0, 1, -1], [3, 20, 16, 2, 0], [[2, -1], [1, 4]])
    angle = rng.standard_normal((32, max(1, rotary // 2)))
    cosine, sine = upload(np.cos(angle).astype(np.float32)), upload(np.sin(angle).astype(np.float32))
    size = rows.itemsize
    call = kl.KVAppendLayout(5, 2, 2, 4, 512, 512, 512, 512 if in_place else 256, rotary, 32, kl.RotaryPairs(pairs),
                             F16 if half else F32)
    assert kl.kv_append(kl.Kernel(), 0, k_pool, v_pool, r.data if in_place else out.data, r.data, r.data + 256 * size,
                        r.data + 384 * size, s.data, p.data, None, t.data, cosine.data, sine.data, cache.layout, call)
    assert kl.kv_cache_status(0) == kl.KV_BAD_PAGE
    q = (r.download(rows.shape, dtype)[:, :256] if in_place else out.download((5, 256), dtype))
    before = rows[:, :256] if in_place else np.full((5, 256), GUARD, dtype)
    for i, there in enumerate((True, False, False, True, False)):
        if not there:
            assert np.array_equal(q[i], before[i]), f"token {i} wrote its query"
        else:
            assert not np.any(q[i] == np.array(GUARD, dtype))
            assert np.array_equal(q[i].reshape(4, 64)[:, rotary:], rows[i, :256].reshape(4, 64)[:, rotary:])
    _, (k, _) = cache.download()
    want = cache.k.copy()
    for page, at in ((2, 3), (1, 2)):
        want[0, page, :, at] = k[0, page, :, at]
    assert np.array_equal(k, want)


# --- process_logits -------------------------------------------------------------------------

def logits_call(rows, vocabulary, past, biases, history_stride, bias_stride, history_lengths, bias_lengths):
    rng = np.random.default_rng(95)
    z = rng.standard_normal((rows, vocabulary)).astype(np.float32)
    history = rng.integers(0, vocabulary, (rows, past)).astype(np.int32)
    ids = rng.integers(0, vocabulary, (rows, biases)).astype(np.int32)
    values = rng.standard_normal((rows, biases)).astype(np.float32)
    penalties = np.tile(np.float32([1.5, 0.25, 0.5]), (rows, 1))
    y = upload(np.full((rows, vocabulary), GUARD, np.float32))
    b = [upload(z), upload(penalties), upload(history), upload(np.int32(history_lengths)), upload(ids), upload(values),
         upload(np.int32(bias_lengths))]
    call = kl.LogitsLayout(rows, vocabulary, vocabulary, vocabulary, history_stride, bias_stride, 0)
    done = kl.process_logits(kl.Kernel(), 0, y.data, *[x.data for x in b], None, call)
    finish()
    gold = z.astype(np.float64)
    for i in range(rows):
        h = history[i, :max(0, history_lengths[i])]
        n = np.bincount(h, minlength=vocabulary)
        gold[i] = np.where(n > 0, np.where(gold[i] > 0, gold[i] / 1.5, gold[i] * 1.5) - n * 0.25 - 0.5, gold[i])
        last = dict(zip(ids[i, :max(0, bias_lengths[i])], values[i]))
        for t, x in last.items():
            gold[i, t] += np.float64(x)
    return done, y.download((rows, vocabulary), np.float32), gold, past


@pytest.mark.parametrize("history_stride,bias_stride", [(0, 3), (7, 0), (0, 0)])
def test_logits_refuses_lists_without_room(gpu, history_stride, bias_stride):
    """A stride of 0 leaves a given list no room: refused, not passed over."""
    done, y, _, _ = logits_call(1, 50, 7, 3, history_stride, bias_stride, [7], [3])
    assert done is False and np.all(y == GUARD)


@pytest.mark.parametrize("history_lengths,bias_lengths,status", [
    ([7, 0, 3], [3, 0, 1], 0), ([8, 0, 3], [3, 0, 1], 2), ([7, -1, 3], [3, 0, 1], 2), ([7, 0, 3], [3, 0, 2 ** 31 - 1], 2),
    ([7, 0, 3], [-5, 0, 1], 2)])
@pytest.mark.parametrize("vocabulary", [50, 3000])
def test_logits_reports_lengths_out_of_range(gpu, history_lengths, bias_lengths, status, vocabulary):
    """A list's length is cut to its row, and reported as the cache's lengths are."""
    assert gpu.kv_cache_status(0) == 0
    done, y, gold, past = logits_call(3, vocabulary, 7, 3, 7, 3, history_lengths, bias_lengths)
    assert done is True and gpu.kv_cache_status(0) == status
    assert np.all(np.abs(y - gold) <= 4 * 2.0 ** -24 * (2 * np.abs(gold) + 2 + past + 5))

