"""The 8-bit key-value cache: the longest lists, scales that something else has made, tokens in any order, and kernels that
ordinary sizes do not reach; against plain computations in 64 bits."""
import numpy as np
import pytest

import kunlunk200_lib_amd as kl
from kv_f8 import (VALUES, CacheF8, check, encode, finish, gold_attention, least_scale, model_append, model_read, run_append,
                   run_attention, run_read, table_of, turned, upload)
from test_gpu_kv_cache_f8 import KERNELS, angles, check_queries, make

pytestmark = pytest.mark.gpu
HALVES = kl.RotaryPairs.halves


def test_read_of_the_longest_lists(gpu):
    """Rows of 16 bytes, of which one launch of fewer than 2^32 threads could not take a wave each."""
    rng = np.random.default_rng(6000)
    tokens, per_launch = (1 << 26) + 5, 1 << 25
    cache = CacheF8(rng, 1, 64, 1, 8, 4)
    pools = cache.upload()
    position = (np.arange(tokens, dtype=np.int32) * 37) % 64
    lists = [upload(np.zeros(tokens, np.int32)), upload(position), upload(np.zeros((1, 1), np.int32))]
    call = kl.KVReadLayout(tokens, 1, 1, 8, 8, kl.InputType.f16)
    assert kl.kv_read_f8_reason(cache.layout, call) == ""
    with kl.Buffer(0, tokens * 16) as k, kl.Buffer(0, tokens * 16) as v:
        assert kl.kv_read_f8(kl.Kernel(), 0, k.data, v.data, *pools, lists[0].data, lists[1].data, None, lists[2].data,
                             cache.layout, call)
        finish()
        for first in (0, per_launch - 300, 2 * per_launch - 300, tokens - 300):
            n = min(600, tokens - first)
            for buffer, pool in ((k, "k"), (v, "v")):
                want = cache.values(pool)[0, 0, 0, position[first:first + n]].astype(np.float16)
                assert np.array_equal(buffer.download((n, 8), np.float16, offset=first * 16), want)
    assert gpu.kv_cache_status(0) == 0


def append_behind(cache, page, at, k, v):
    """The model of one new token behind others of its block at place `at` of a page, with any finite scale there: kept where
    it is at least as large in size as the new value needs, else the codes move to the least power of two."""
    block = cache.layout.block_tokens
    b, earlier = at // block, slice(at // block * block, at)
    for codes, scales, x in ((cache.k, cache.ks, k), (cache.v, cache.vs, v)):
        for h in range(cache.layout.cache.heads):
            old, need = float(scales[0, page, h, b]), float(least_scale(np.abs(x[h]).max()))
            scale = old if abs(old) >= need else need
            if scale != old:
                codes[0, page, h, earlier] = encode(VALUES[codes[0, page, h, earlier]] * old / scale)
            scales[0, page, h, b] = scale
            # (a quotient in 64 bits is on a tie between codes only where the exact one is)
            codes[0, page, h, at] = encode(x[h].astype(np.float64) / scale)


@pytest.mark.parametrize("block", [2, 16, 64])
def test_append_behind_negative_scales(gpu, block):
    """Scales of either sign, smaller and larger than the new token's and equal to it."""
    rng = np.random.default_rng(6001)
    heads, width, page_tokens, rows = 3, 64, 64, 24
    cache = CacheF8(rng, rows, page_tokens, heads, width, block)
    for scales in cache.scales:
        scales[...] = rng.choice([-1, 1], scales.shape) * 2.0 ** rng.integers(-12, 0, scales.shape)
    model, at = cache.copy(), np.where(np.arange(rows) % 2, block - 1, block * (page_tokens // block - 1) + 1)
    # needs of 2^-12 to 2^-1
    top = 448 * 2.0 ** rng.integers(-12, 0, (2, rows, heads, 1))
    k, v = (rng.uniform(-1, 1, (2, rows, heads, width)) * top).astype(np.float32)
    for x, t in ((k, top[0]), (v, top[1])):
        x[:, :, 5] = t[:, :, 0]
    for row in range(rows):
        append_behind(model, row, at[row], k[row], v[row])
    cache.upload()
    table = np.arange(rows, dtype=np.int32)[:, None]
    run_append(cache, table, np.arange(rows), at, None, k, v, (), (), HALVES, 0)
    cache.download()
    old = cache.scales[0][0, np.arange(rows), :, at // block]
    assert (old < 0).any() and (old > 0).any()
    assert cache.same_as(model)
    assert gpu.kv_cache_status(0) == 0


@pytest.mark.parametrize("width", [8, 128])
def test_read_rounds_any_scale_once(gpu, width):
    """F16 rows beside scales of 24 bits: products whose nearest F32 lies on a tie between two F16 numbers, which the exact ones
    do not; of every size from F16's subnormals to past its range, of both signs."""
    rng = np.random.default_rng(6002)
    pages, page_tokens, heads = 64, 64, 128 // width * 4
    cache = CacheF8(rng, pages, page_tokens, heads, width, 1)
    for flat, scales in zip(cache.flat, cache.scales):
        flat[...] = rng.integers(0, 127, flat.shape) + 128 * rng.integers(0, 2, flat.shape)
        scales[...] = rng.choice([-1, 1], scales.shape) * rng.uniform(1, 2, scales.shape) * 2.0 ** rng.integers(-24, 9, scales.shape)
    cache.upload()
    n = pages * page_tokens
    table, position = np.arange(pages, dtype=np.int32)[None, :], np.arange(n)
    twice = 0
    for got, pool in zip(run_read(cache, table, np.zeros(n, int), position, np.float16), "kv"):
        exact = cache.values(pool)[0].transpose(0, 2, 1, 3).reshape(got.shape)
        with np.errstate(over="ignore"):
            want = exact.astype(np.float16)
            twice += (exact.astype(np.float32).astype(np.float16) != want).sum()
        assert np.array_equal(got, want)
    assert twice > 20, "no product that F32 takes to a tie"


def test_append_rounds_earlier_codes_once(gpu):
    """Codes that move from a scale of 24 bits to a new one: products whose nearest F32 is a tie between two codes."""
    rng = np.random.default_rng(6003)
    rows, heads, width = 128, 1, 128
    cache = CacheF8(rng, rows, 16, heads, width, 16)
    # scale = tie / code and the numbers beside it, so that code * scale is within 2^-24 of a tie in the new scale, 1
    tie = (np.arange(8, 16) + 0.5) / 8
    code = rng.integers(9, 120, (2, rows))
    for scales, codes, c in zip(cache.scales, (cache.k, cache.v), code):
        s = (rng.choice(tie, rows) * 2.0 ** rng.integers(-4, 2, rows) / VALUES[c]).astype(np.float32)
        s = np.where(s < 0.99, s, s / 256)
        scales[0, :, 0, 0] = [np.nextafter(x, np.float32(rng.choice([0, x, 1]))) for x in s]
        codes[0, :, 0, :, ::2] = c[:, None, None]
    model = cache.copy()
    k, v = rng.uniform(-1, 1, (2, rows, heads, width)).astype(np.float32)
    k[:, :, 0] = v[:, :, 0] = 448
    at = np.full(rows, 9)
    for row in range(rows):
        append_behind(model, row, at[row], k[row], v[row])
    twice = 0
    for codes, scales in ((cache.k, cache.scales[0]), (cache.v, cache.scales[1])):
        y = VALUES[codes[0, :, 0, :9]].astype(np.float32) * scales[0, :, 0, 0, None, None]
        twice += (encode(y) != encode(VALUES[codes[0, :, 0, :9]] * scales[0, :, 0, 0, None, None].astype(np.float64))).sum()
    assert twice > 20, "no product that F32 takes to a tie"
    cache.upload()
    run_append(cache, np.arange(rows, dtype=np.int32)[:, None], np.arange(rows), at, None, k, v, (), (), HALVES, 0)
    cache.download()
    assert cache.same_as(model)
    assert gpu.kv_cache_status(0) == 0


def to_odd(x):
    """F32 of 64-bit values, rounded to odd: towards zero, the last bit set where that is not exact."""
    near = x.astype(np.float32)
    bits = near.view(np.uint32) - (np.abs(near.astype(np.float64)) > np.abs(x))
    return np.where(near == x, near, (bits.astype(np.uint32) | 1).view(np.float32))


@pytest.mark.parametrize("block,width,rotary", [(2, 8, 0), (16, 64, 0), (16, 64, 32), (64, 256, 256)])
def test_append_rounds_once_beside_any_scale(gpu, block, width, rotary):
    """New values at ties between codes beside a kept scale of 24 bits, and the F32 numbers around; turned by angles so small
    that only F64 sees them. More than one new token of a block, and blocks whose scale is a power of two among them."""
    rng = np.random.default_rng(6004)
    rows, heads, page_tokens, new = 40, 2, 64, min(3, block - 1)
    cache = CacheF8(rng, rows, page_tokens, heads, width, block)
    for scales in cache.scales:
        scales[...] = rng.choice([-1, 1], scales.shape) * rng.uniform(0.001, 0.1, scales.shape)
        scales[0, ::7] = 2.0 ** -8
    model = cache.copy()
    b = rng.integers(0, page_tokens // block, rows)
    first = b * block + block - new
    ties = (VALUES[:126] + VALUES[1:127]) / 2
    x = []
    for scales in cache.scales:
        s = scales[0, np.arange(rows), :, b].astype(np.float64)[:, None, :, None]
        value = (rng.choice(ties, (rows, new, heads, width)) * s).astype(np.float32)
        x.append(np.where(rng.random(value.shape) < 0.5, np.nextafter(value, np.float32(0)), value))
    k, v = x
    k[3, 0, 0, 5], v[3, 0, 0, 5] = 0.0, -0.0
    half = rotary // 2
    position = first[:, None] + np.arange(new)
    cos, sin = np.ones((page_tokens, half), np.float32), rng.choice([-1, 1], (page_tokens, half)).astype(np.float32) * np.float32(2 ** -20)
    twice = 0
    for row in range(rows):
        at = position[row]
        turn = np.stack([turned(y, cos[p], sin[p], HALVES) for y, p in zip(k[row], at)])
        for codes, scales, exact in ((model.k, model.ks, turn), (model.v, model.vs, v[row].astype(np.float64))):
            for h in range(heads):
                old, need = float(scales[0, row, h, b[row]]), float(least_scale(np.abs(exact[:, h]).max()))
                scale = old if abs(old) >= need else need
                earlier = slice(b[row] * block, first[row])
                if scale != old:
                    codes[0, row, h, earlier] = encode(VALUES[codes[0, row, h, earlier]] * old / scale)
                scales[0, row, h, b[row]] = scale
                # beside a power of two the nearest code of the exact value is that of the odd F32 number
                values = to_odd(exact[:, h])
                codes[0, row, h, at] = encode(values.astype(np.float64) / scale)
                rough = values * (np.float32(1) / np.float32(scale))
                twice += (encode(rough.astype(np.float64)) != encode(values.astype(np.float64) / scale)).sum()
    assert twice > 0, "no quotient that F32 takes to a tie"
    cache.upload()
    flat = lambda y: y.reshape(rows * new, heads, width)  # noqa: E731
    run_append(cache, np.arange(rows, dtype=np.int32)[:, None], np.repeat(np.arange(rows), new), position.reshape(-1), None,
               flat(k), flat(v), cos, sin, HALVES, rotary)
    cache.download()
    assert all(np.array_equal(p, q) for p, q in zip(cache.scales, model.scales))
    assert cache.same_as(model)
    assert gpu.kv_cache_status(0) == 0


def lists_of_runs(rng, rows, most, block):
    """(sequence, position) of whole and partial runs of blocks in any order, each block's tokens together; some left out."""
    sequence, position = [], []
    runs = [(s, b) for s in range(rows) for b in range(most // block)]
    for r in rng.permutation(len(runs)):
        s, b = runs[r]
        lo, hi = sorted(rng.integers(0, block + 1, 2))
        sequence += [s] * (hi - lo)
        position += list(range(b * block + lo, b * block + hi))
    out = rng.random(len(position)) < 0.1
    return np.where(out & (rng.random(len(out)) < 0.5), -1, sequence), np.where(out, -1, position)


@pytest.mark.parametrize("rows,most,block,width", [(7, 64, 16, 64), (60, 128, 4, 8), (3, 4096, 2, 24), (40, 128, 64, 256)])
def test_append_blocks_in_any_order(gpu, rows, most, block, width):
    """What the rule allows is not reported, in lists of one checking workgroup and of several."""
    rng = np.random.default_rng(6005)
    cache = CacheF8(rng, rows * most // 64, 64, 1, width, block)
    table = rng.permutation(rows * most // 64).astype(np.int32).reshape(rows, -1)
    sequence, position = lists_of_runs(rng, rows, most, block)
    k, v = rng.standard_normal((2, len(sequence), 1, width)).astype(np.float32)
    model = cache.copy()
    stored, status = model_append(model, table, sequence, position, k, v, (), (), HALVES, 0)
    assert status == 0 and stored.sum() > 100
    cache.upload()
    run_append(cache, table, sequence, position, None, k, v, (), (), HALVES, 0)
    assert gpu.kv_cache_status(0) == 0
    cache.download()
    assert cache.same_as(model)


@pytest.mark.parametrize("block,width,half", [(16, 128, False), (2, 64, True), (64, 256, False), (4, 8, True)])
def test_append_reports_blocks_in_pieces(gpu, block, width, half):
    """Tokens of one block apart in the list: sequences in turn, positions backwards, one token of a long list far off. The
    blocks that stand together in the same call are stored as ever."""
    rng = np.random.default_rng(6006)
    rows, most, dtype = 90, 256, np.float16 if half else np.float32
    cache = CacheF8(rng, rows * most // 64, 64, 1, width, block)
    table = rng.permutation(rows * most // 64).astype(np.int32).reshape(rows, -1)
    together = np.repeat(np.arange(2, rows), 40), np.tile(np.arange(128, 168), rows - 2)
    n = len(together[0])
    lists = {
        "in turn": (np.tile([0, 1], 8), np.repeat(np.arange(8), 2)),
        "all in turn": (np.tile(np.arange(rows), 3), np.repeat(np.arange(3), rows)),
        "backwards": (np.zeros(9, int), np.arange(9, 0, -1)),
        "a gap": (np.zeros(4, int), np.array([0, 1, block, 1])),
        "far off": (np.concatenate([[0], together[0], [0]]), np.concatenate([[block - 1], together[1], [0]])),
        "far off, the first first": (np.concatenate([[1], together[0], [1]]), np.concatenate([[0], together[1], [block - 1]])),
    }
    for name, (sequence, position) in lists.items():
        print(name, flush=True)
        k, v = rng.standard_normal((2, len(sequence), 1, width)).astype(dtype)
        model = cache.copy()
        cache.upload()
        run_append(cache, table, sequence, position, None, k, v, (), (), HALVES, 0)
        assert gpu.kv_cache_status(0) == kl.KV_BAD_INDEX, name
        assert gpu.kv_cache_status(0) == 0
        if len(sequence) > n:
            cache.download()
            inside = slice(1, n + 1)
            model_append(model, table, *together, k[inside], v[inside], (), (), HALVES, 0)
            untouched = np.ones(rows * most // 64, bool)
            untouched[table[:2]] = False
            for a, b in zip((cache.k, cache.v, cache.ks, cache.vs), (model.k, model.v, model.ks, model.vs)):
                assert np.array_equal(a[:, untouched], b[:, untouched])


# --- attention --------------------------------------------------------------------------------

@pytest.mark.parametrize("exponent", [-124, -112, -100, -64, 0, 90])
@pytest.mark.parametrize("case", range(len(KERNELS)))
def test_attention_value_scales_of_any_size(gpu, case, exponent):
    """Value scales of 24 bits about one power of two, beside keys of 0, which make every weight 1.

    All but four tokens' codes are 0, so a sum has four terms that are not, each held to 2^-22 of itself, 2^-38 of the largest
    (at most 448 / 2 of a term) or 2^-149; two parts of four terms each, their sum, the joins of up to 8 waves' and 2 parts' sums and
    the division round fewer than 32 times, by 2^-24 each."""
    rng, lengths, table, cache, q = make(case, 60)
    c = cache.layout.cache
    cache.ks[...] = 0
    cache.vs[...] = rng.choice([-1, 1], cache.vs.shape) * rng.uniform(1, 2, cache.vs.shape) * 2.0 ** exponent
    gold, tol = np.zeros(q.shape), np.zeros(q.shape)
    values = cache.v.copy()
    cache.v[...] = 0
    shown = {}
    for s, n in enumerate(lengths):
        for t in rng.choice(n, min(n, 4), replace=False):
            page, at = table[s, t // c.page_tokens], t % c.page_tokens
            shown[page, at] = True
            cache.v[0, page, :, at] = values[0, page, :, at]
    for s, n in enumerate(lengths):                      # (rows may share pages: more than four terms then)
        t = np.arange(n)
        page, at = table[s, t // c.page_tokens], t % c.page_tokens
        keep = np.array([(p, a) in shown for p, a in zip(page, at)])
        v = cache.values("v")[0, page[keep], :, at[keep]]                        # [term][head][value]
        scales = np.abs(cache.vs[0, page[keep], :, at[keep] // cache.layout.block_tokens].astype(np.float64))
        group = q.shape[1] // c.heads
        each = np.abs(v) * (2.0 ** -22 + 8 * len(v) * 2.0 ** -24)
        lost = 448 * np.maximum(2.0 ** -38 * scales.max(0), 2.0 ** -149)[:, None] * len(v)
        gold[s] = np.repeat(v.sum(0) / n, group, 0)
        tol[s] = np.repeat((each.sum(0) + lost) / n, group, 0) + 2.0 ** -149
    y, _ = run_attention(cache, table, lengths, q)
    err = np.abs(y.astype(np.float64) - gold)
    assert np.all(np.isfinite(y))
    assert np.all(err <= tol), f"worst {np.max(err / tol):.3g} of the tolerance"


@pytest.mark.parametrize("scale,size", [(30.0, 1e4), (-0.5, 1e4), (0.125, 1e6), (-3e-9, 1e14)])
@pytest.mark.parametrize("case", range(len(KERNELS)))
def test_attention_far_scores(gpu, case, scale, size):
    """Scores of up to 10^7: where the best token is ahead by more than the scores' error and 130, the others' weights are below
    e^-130 and y is its value row, to 2^-22 for its weight's parts and some roundings of 2^-24."""
    _, lengths, table, cache, q = make(case, 61)
    c, group = cache.layout.cache, q.shape[1] // cache.layout.cache.heads
    q = (q * size).astype(np.float32)
    y, _ = run_attention(cache, table, lengths, q, scale=scale)
    keys, values, clear, factor = cache.values("k")[0], cache.values("v")[0], 0, abs(float(np.float32(scale)))
    for s, n in enumerate(lengths):
        t = np.arange(n)
        page, at = table[s, t // c.page_tokens], t % c.page_tokens
        for h in range(q.shape[1]):
            k, qh = keys[page, h // group, at], q[s, h].astype(np.float64)
            score = (k @ qh) * float(np.float32(scale))
            error = np.abs(k * qh).sum(1).max() * factor * (2.0 ** -21 + len(qh) * 2.0 ** -24 + 2.0 ** -22)
            best = np.argsort(score)[-2:] if n > 1 else np.array([0, 0])
            if n > 1 and score[best[1]] - score[best[0]] <= 2 * error + 130:
                continue
            clear += 1
            want = values[page[best[1]], h // group, at[best[1]]]
            assert np.all(np.abs(y[s, h] - want) <= np.abs(want) * (2.0 ** -22 + 8 * 2.0 ** -24)), (s, h)
    assert clear > 0.8 * q.shape[0] * q.shape[1]


# sequences, heads, query heads, width, tokens of a page, of a block, longest, window: many rows that one wave takes each, of up
# to eight steps, above width 128, with widths that are no multiple of 32, page ids in LDS and two column tiles
NARROW = [(1100, 2, 2, 128, 16, 16, 250, 0), (1100, 2, 4, 120, 16, 4, 250, 100), (300, 2, 2, 256, 16, 2, 250, 0),
          (300, 2, 18, 256, 32, 32, 129, 0), (600, 1, 1, 200, 16, 16, 250, 0), (600, 2, 6, 80, 20, 4, 128, 0),
          (600, 2, 2, 168, 12, 4, 220, 60), (600, 1, 3, 24, 1, 1, 90, 0), (1100, 2, 2, 104, 24, 8, 256, 0)]


@pytest.mark.parametrize("case", range(len(NARROW)))
def test_attention_one_wave(gpu, case):
    sequences, heads, query_heads, width, page_tokens, block, longest, window = NARROW[case]
    rng = np.random.default_rng(6100 + case)
    lengths = rng.integers(0, longest + 1, sequences)
    lengths[0] = longest
    pages = -(-longest // page_tokens) + 3
    # the sequences share a few pages: what is read is what counts here
    table = rng.integers(0, pages, (sequences, pages)).astype(np.int32)
    cache = CacheF8(rng, pages, page_tokens, heads, width, block, ("heads", "tokens")[case % 2], case % 3)
    q = rng.standard_normal((sequences, query_heads, width)).astype((np.float32, np.float16)[case % 2])
    y, route = run_attention(cache, table, lengths, q, window)
    assert route == "paged_attention_f8"
    gold, tol = gold_attention(cache, table, lengths, q, window, width ** -0.5)
    check(y, gold, tol)
    assert gpu.kv_cache_status(0) == 0


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads,width,page_tokens,block", [(32, 128, 16, 16), (9, 120, 16, 4), (64, 256, 64, 64), (5, 104, 20, 1)])
def test_wide_tokens(gpu, heads, width, page_tokens, block, half):
    """Tokens that several waves read back, the last one less than whole."""
    rng = np.random.default_rng(6200)
    dtype, parts = (np.float16 if half else np.float32), [(3, 20), (0, 1), (page_tokens, 2)]
    lengths = [a + b for a, b in parts]
    cache = CacheF8(rng, 12, page_tokens, heads, width, block)
    table = table_of(rng, lengths, page_tokens, 12, 3)
    sequence = np.concatenate([np.full(n, s) for s, (_, n) in enumerate(parts)])
    position = np.concatenate([np.arange(a, a + n) for a, n in parts])
    q, k, v = (rng.standard_normal((len(sequence), h, width)).astype(dtype) for h in (heads + 3, heads, heads))
    cos, sin = angles(max(lengths), width // 2)
    model = cache.copy()
    stored, status = model_append(model, table, sequence, position, k, v, cos, sin, HALVES, width)
    cache.upload()
    y = run_append(cache, table, sequence, position, q, k, v, cos, sin, HALVES, width)
    cache.download()
    assert cache.same_as(model)
    check_queries(y, q, stored, position, cos, sin, HALVES, width)
    of, at = np.concatenate([np.full(n, s) for s, n in enumerate(lengths)]), np.concatenate([np.arange(n) for n in lengths])
    for kind, common in ((np.float32, False), (np.float16, True)):
        for a, b in zip(run_read(cache, table, of, at, kind, common=common), model_read(model, table, of, at, kind)):
            assert np.array_equal(a, b)
    assert gpu.kv_cache_status(0) == 0
