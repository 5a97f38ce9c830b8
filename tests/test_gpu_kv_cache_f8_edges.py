"""The 8-bit key-value cache at the ends of its ranges and with calls one behind the other: against 64 bits or against the
same call alone."""
import numpy as np
import pytest

import kunlunk200_lib_amd as kl
from kv_f8 import GUARD, CacheF8, check, finish, gold_attention, run_attention, run_read, table_of, upload

pytestmark = pytest.mark.gpu

# sequences, heads, query heads, width, tokens of a page, of a block, longest: whole rows, parts, equal shares, pages
# looked up one by one, two column tiles, one wave
SHAPES = [
    (3, 2, 4, 64, 16, 16, 150),
    (2, 2, 2, 128, 16, 4, 4000),
    (64, 8, 8, 128, 16, 16, 2100),
    (2, 3, 6, 80, 20, 2, 700),
    (1, 1, 12, 96, 16, 1, 300),
    (600, 2, 2, 64, 16, 8, 70),
]


@pytest.mark.parametrize("size", [1e34, 1e20, 1e-30])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_attention_scales_against_queries(gpu, case, size):
    """Key scales that bring the scores of very large or small queries to ordinary size. A block of zero codes scores 0
    whatever its finite scale, though that times the queries' size is infinite."""
    sequences, heads, query_heads, width, page_tokens, block, longest = SHAPES[case]
    rng = np.random.default_rng(4000 + case)
    lengths = rng.integers(1, longest + 1, sequences)
    lengths[0] = longest
    pages = -(-longest // page_tokens) + 3
    cache = CacheF8(rng, pages, page_tokens, heads, width, block)
    table = np.stack([rng.permutation(pages) for _ in lengths]).astype(np.int32)
    # codes of about 100, so a score's terms sum to about 4 in size
    cache.ks[...] = (0.05 / (size * np.sqrt(width)) * rng.uniform(0.5, 1.0, cache.ks.shape)).astype(np.float32)
    zero = rng.random(cache.ks.shape) < 0.1
    cache.ks[zero] = 1e30
    cache.k[np.repeat(zero, block, 3)] = 0
    q = (rng.standard_normal((sequences, query_heads, width)) * size).astype(np.float32)
    y, _ = run_attention(cache, table, lengths, q)
    gold, tol = gold_attention(cache, table, lengths, q, 0, float(np.float32(width ** -0.5)))
    check(y, gold, tol)


def test_attention_calls_in_a_queue(gpu):
    """Calls of one Kernel that share its workspace, submitted without a wait between them, the larger needs last: each
    gives the bits that it gives alone. Rows behind the last sequence stay as they were."""
    kernel = kl.Kernel()
    cases = []
    for i, (sequences, heads, query_heads, width, page_tokens, block, longest) in enumerate(SHAPES):
        rng = np.random.default_rng(4100 + i)
        lengths = rng.integers(0, longest + 1, sequences).astype(np.int32)
        lengths[-1] = longest
        pages = -(-longest // page_tokens) + 3
        cache = CacheF8(rng, pages, page_tokens, heads, width, block)
        table = np.stack([rng.permutation(pages) for _ in lengths]).astype(np.int32)
        q = rng.standard_normal((sequences, query_heads, width)).astype(np.float32)
        alone, _ = run_attention(cache, table, lengths, q)
        row = query_heads * width
        call = kl.PagedAttentionLayout(sequences, query_heads, longest, 0, pages, row, row, width ** -0.5,
                                       kl.InputType.f32)
        out = np.full((sequences + 2, row), GUARD, np.float32)
        cases.append((cache, cache.upload(), [upload(x) for x in (out, q, table, lengths)], call, alone, out))
    order = [0, 1, 2, 3, 4, 5, 2, 1, 5, 0, 3]
    for i in order:
        cache, pools, bufs, call, _, _ = cases[i]
        assert kl.paged_attention_f8(kernel, 0, bufs[0], bufs[1], *pools, bufs[2], bufs[3], cache.layout, call)
    finish()
    for cache, pools, bufs, call, alone, out in cases:
        y = bufs[0].download(out.shape, np.float32)
        assert np.array_equal(y[:-2].reshape(alone.shape), alone)
        assert np.all(y[-2:] == np.float32(GUARD)), "wrote behind the last sequence"
    assert gpu.kv_cache_status(0) == 0


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_read_in_any_order(gpu, dtype):
    """Tokens named several times, backwards and out of their sequences' order."""
    rng = np.random.default_rng(4200)
    lengths = [45, 17, 80]
    cache = CacheF8(rng, 12, 16, 3, 40, 4)
    table = table_of(rng, lengths, 16, 12, 5)
    cache.upload()
    sequence = rng.integers(0, 3, 150)
    position = np.array([rng.integers(0, lengths[s]) for s in sequence])
    sequence[7:9], position[7:9] = sequence[3], position[3]
    k, v = run_read(cache, table, sequence, position, dtype)
    for got, pool in ((k, "k"), (v, "v")):
        values = cache.values(pool)[0]
        want = values[table[sequence, position // 16], :, position % 16]
        assert np.array_equal(got, want.astype(dtype))
    assert gpu.kv_cache_status(0) == 0


@pytest.mark.parametrize("block,width", [(4, 64), (64, 128)])
def test_append_with_nothing_to_store(gpu, block, width):
    """A call whose entries are all left out changes neither pools nor rows."""
    rng = np.random.default_rng(4300)
    cache = CacheF8(rng, 2, 64, 1, width, block)
    pools = cache.upload()
    before = cache.copy()
    n = 130
    x = rng.standard_normal((n, 3 * width)).astype(np.float32)
    rows, out = upload(x), upload(np.full((n, width), GUARD, np.float32))
    angles = [upload(f(np.arange(64 * (width // 2), dtype=np.float64) / 97).astype(np.float32)) for f in (np.cos, np.sin)]
    at = [rows.data + i * 4 * width for i in range(3)]
    call = kl.KVAppendLayout(n, 1, 1, 1, 3 * width, 3 * width, 3 * width, width, width, 64, kl.RotaryPairs.halves,
                             kl.InputType.f32)
    none = upload(np.full(n, -1, np.int32))
    places, table = upload(np.arange(n, dtype=np.int32) % 64), upload(np.array([[1]], np.int32))
    assert kl.kv_append_f8(kl.Kernel(), 0, *pools, out, *at, none, places, None, table, *angles, cache.layout, call)
    finish()
    cache.download()
    assert cache.same_as(before)
    assert np.all(out.download((n, width), np.float32) == np.float32(GUARD))
    assert gpu.kv_cache_status(0) == 0
