"""Plain models of the 8-bit key-value cache for its tests: e4m3 codes, pools in either order with padding, and in 64
bits what append, read-back and attention are to give."""
from __future__ import annotations

import numpy as np

import kunlunk200_lib_amd as kl

F32, F16 = kl.InputType.f32, kl.InputType.f16
GUARD = -12345.0


def _code_values():
    code = np.arange(256)
    exponent, mantissa = (code >> 3) & 15, code & 7
    size = np.where(exponent > 0, (8 + mantissa) * 2.0 ** (exponent - 10.0), mantissa * 2.0 ** -9)
    size[[127, 255]] = np.nan
    return np.where(code > 127, -size, size)


VALUES = _code_values()                        # of the 256 codes
SIZES = VALUES[:127]                           # 0 to 448, rising


def encode(x):
    """The nearest codes of x (64 bits, at most 448 or what rounds to it), ties to the even code."""
    x = np.asarray(x, np.float64)
    size = np.abs(x)
    above = np.clip(np.searchsorted(SIZES, size), 1, 126)
    low, high = SIZES[above - 1], SIZES[above]
    up = (size - low > high - size) | ((size - low == high - size) & (above % 2 == 0))
    code = np.where(up, above, above - 1)
    code = np.where(np.isnan(size), 127, code)
    return (code + 128 * np.signbit(x)).astype(np.uint8)


def least_scale(top):
    """The least power of two from 2^-64 up that takes `top` to 448."""
    mantissa, exponent = np.frexp(top / 448.0)     # top / 448 = mantissa * 2^exponent
    exponent = np.where(mantissa == 0.5, exponent - 1, exponent)
    least = 2.0 ** np.maximum(np.where(np.asarray(top) > 0, exponent, -64), -64.0)
    return np.where(np.isfinite(top), least, np.nan)


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


class CacheF8:
    """Pools of codes in either order with optional padding, and their scales: `k`, `v` as [layer][page][head][token][value],
    `ks`, `vs` as [layer][page][head][block]."""

    def __init__(self, rng, pages, page_tokens, heads, width, block_tokens, order="heads", pad=0, layers=1):
        w = width + 8 * pad
        if order == "heads":
            strides = (page_tokens * w * heads + 16 * pad, page_tokens * w, w)
        else:
            strides = (page_tokens * w * heads + 16 * pad, w, w * heads)
        self.layout = kl.KVCacheF8Layout(kl.KVCacheLayout(pages, page_tokens, heads, width, *strides), block_tokens)
        assert kl.kv_cache_f8_reason(self.layout) == ""
        self.layers, self.layer = layers, strides[0] * pages
        self.flat = [encode(np.clip(rng.standard_normal(self.layer * layers) * 100, -448, 448)) for _ in range(2)]
        shape = (layers, pages, heads, page_tokens // block_tokens)
        self.scales = [(2.0 ** rng.integers(-10, -5, shape)).astype(np.float32) for _ in range(2)]
        self.k, self.v = (self.view(x) for x in self.flat)
        self.ks, self.vs = self.scales
        self.buffers = None

    def view(self, flat):
        c = self.layout.cache
        return np.lib.stride_tricks.as_strided(
            flat, (self.layers, c.pages, c.heads, c.page_tokens, c.width),
            (self.layer, c.page_stride, c.head_stride, c.token_stride, 1))

    def values(self, pool):
        """[layer][page][head][token][value] in 64 bits."""
        codes, scales = (self.k, self.ks) if pool == "k" else (self.v, self.vs)
        scales = np.repeat(scales.astype(np.float64), self.layout.block_tokens, 3)
        return VALUES[codes] * scales[..., None]

    def upload(self):
        self.buffers = [upload(x) for x in (*self.flat, *self.scales)]
        return [b.data for b in self.buffers]

    def pools(self):
        return [b.data for b in self.buffers]

    def download(self):
        """What the device holds now, into this object."""
        for b, x in zip(self.buffers, (*self.flat, *self.scales)):
            x[...] = b.download(x.shape, x.dtype)

    def copy(self):
        other = object.__new__(CacheF8)
        other.__dict__.update(self.__dict__)
        other.flat, other.scales = [x.copy() for x in self.flat], [x.copy() for x in self.scales]
        other.k, other.v = (other.view(x) for x in other.flat)
        other.ks, other.vs = other.scales
        return other

    def same_as(self, other):
        return (all(np.array_equal(a, b) for a, b in zip(self.flat, other.flat)) and
                all(np.array_equal(a, b, equal_nan=True) for a, b in zip(self.scales, other.scales)))


def table_of(rng, lengths, page_tokens, pages, row_pages, rest=-1):
    ids = list(rng.permutation(pages))
    table = np.full((len(lengths), row_pages), rest, np.int32)
    for s, n in enumerate(lengths):
        for j in range(-(-n // page_tokens)):
            table[s, j] = ids.pop()
    return table


# --- attention ----------------------------------------------------------------------------

def gold_attention(cache, table, lengths, q, window, scale, skip=()):
    """(y, tolerance without the output's rounding) in 64 bits; `skip`: page ids whose tokens are left out.

    A score's error is at most e_s = a (2^-21 + width 2^-24 + 2^-22) with a = max_t sum_d |scale q_d k_td|: two
    F16 parts hold a query value to 2^-22 of itself (what they hold to 2^-34 of the row's largest is within 2^-24 a
    for rows whose largest value meets a code other than 0), codes are exact, sums are F32, two factors are rounded
    once each. A weight's relative error is e_w = e_s + 2^-20 (exponential, its value scale and its own parts), and
    2^-38 of the largest weight times scale and code besides; sums add n 2^-24."""
    c, block = cache.layout.cache, cache.layout.block_tokens
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
        at = t % c.page_tokens
        for h in range(query_heads):
            kv = h // group
            ks = cache.ks[0, page, kv, at // block].astype(np.float64)[:, None]
            vs = cache.vs[0, page, kv, at // block].astype(np.float64)[:, None]
            with np.errstate(invalid="ignore", over="ignore"):
                k, v = VALUES[cache.k[0, page, kv, at]] * ks, VALUES[cache.v[0, page, kv, at]] * vs
                qh = q[s, h].astype(np.float64)
                score = (k @ qh) * scale
                if np.all(score == -np.inf):
                    continue
                p = np.exp(score - score.max())
                y[s, h] = p @ v / p.sum()
                a = np.nanmax(np.abs(k * qh).sum(1), initial=0.0) * abs(scale)
                e_w = a * (2.0 ** -21 + width * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -20
                lost = len(t) * 2.0 ** -38 * 448 * np.max(p * np.abs(vs[:, 0]))
                tol[s, h] = ((2 * e_w + 2 * len(t) * 2.0 ** -24) * (p @ np.abs(v)) + lost) / p.sum()
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
    pools = cache.upload()
    bufs = [upload(x) for x in (out, rows, np.asarray(table, np.int32), np.asarray(lengths, np.int32))]
    call = kl.PagedAttentionLayout(n, query_heads, longest, window, table.shape[1], row + pad, row + pad, scale, kind)
    assert kl.paged_attention_f8_reason(cache.layout, call) == ""
    kernel = kernel or kl.Kernel()
    assert kl.paged_attention_f8(kernel, 0, bufs[0].data, bufs[1].data, *pools, bufs[2].data, bufs[3].data, cache.layout, call)
    finish()
    y = bufs[0].download(out.shape, q.dtype)
    assert np.all(y[:, row:] == np.array(GUARD, q.dtype)), "wrote between rows"
    before = cache.copy()
    cache.download()
    assert cache.same_as(before), "cache changed"
    return y[:, :row].reshape(q.shape), kernel.route


def check(y, gold, tol):
    if y.dtype == np.float16:
        tol = tol + 2.0 ** -11 * np.abs(gold) * 1.01 + 2.0 ** -25
    err = np.abs(y.astype(np.float64) - gold)
    assert np.all(np.isfinite(y))
    assert np.all(err <= tol + 1e-37), f"worst {np.max(err / (tol + 1e-37)):.3g} of the tolerance"


# --- append and read-back -------------------------------------------------------------------

def turned(x, cos, sin, pairs):
    """x [heads, width] in 64 bits with its first 2 * len(cos) values turned."""
    half = len(cos)
    y = x.astype(np.float64)
    if half == 0:
        return y
    cos, sin = cos.astype(np.float64), sin.astype(np.float64)
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if pairs == kl.RotaryPairs.adjacent else (
        slice(0, half), slice(half, 2 * half))
    with np.errstate(invalid="ignore"):
        a, b = y[:, first].copy(), y[:, second].copy()
        y[:, first], y[:, second] = a * cos - b * sin, a * sin + b * cos
    return y


def model_append(cache, table, sequence, position, k, v, cos, sin, pairs, rotary, layer=0):
    """kv_append_f8 on the model. k, v: [tokens, heads, width]; returns (tokens stored, status bits)."""
    c, block = cache.layout.cache, cache.layout.block_tokens
    rows, row_pages = table.shape
    place, status = [], 0
    for i, (s, p) in enumerate(zip(sequence, position)):
        place.append(None)
        if s < 0 or (s < rows and p < 0):
            continue
        if s >= rows or p // c.page_tokens >= row_pages or (rotary > 0 and p >= len(cos)):
            status |= kl.KV_BAD_INDEX
        else:
            place[i] = (s, p)
    stored, done = np.zeros(len(place), bool), np.zeros(len(place), bool)
    for i in range(len(place)):
        if place[i] is None or done[i]:
            continue
        s, p = place[i]
        earlier = p % c.page_tokens % block
        members = [j for j in range(min(block - earlier, len(place) - i)) if place[i + j] == (s, p + j)]
        done[[i + j for j in members]] = True
        page, at = table[s, p // c.page_tokens], p % c.page_tokens
        if not 0 <= page < c.pages:
            status |= kl.KV_BAD_PAGE
            continue
        stored[[i + j for j in members]] = True
        for codes, scales, x, is_k in ((cache.k, cache.ks, k, True), (cache.v, cache.vs, v, False)):
            angles = (lambda t: (cos[t, :rotary // 2], sin[t, :rotary // 2])) if is_k and rotary else (lambda t: ((), ()))
            new = np.stack([turned(x[i + j], *map(np.asarray, angles(p + j)), pairs) for j in members])
            b = at // block
            for h in range(c.heads):
                top = np.abs(new[:, h]).max() if np.all(np.isfinite(new[:, h])) else np.nan
                scale = np.float32(least_scale(top))
                old = scales[layer, page, h, b]
                if earlier and scale == scale and not old <= scale:
                    scale = old
                if earlier and scale > old:
                    before = slice(at - earlier, at)
                    codes[layer, page, h, before] = encode(VALUES[codes[layer, page, h, before]] * float(old / scale))
                scales[layer, page, h, b] = scale
                codes[layer, page, h, [at + j for j in members]] = encode(new[:, h] / float(scale))
    return stored, status


def run_append(cache, table, sequence, position, q, k, v, cos, sin, pairs, rotary, lengths=None, pad=0, offset=0,
               in_place=False, kernel=None):
    """kv_append_f8 on the uploaded cache. q, k, v: [tokens, heads, width]; sequence and position None: the newest of each
    sequence. Returns q_out."""
    c = cache.layout.cache
    tokens, query_heads = k.shape[0], q.shape[1] if q is not None else 0
    kind = F16 if k.dtype == np.float16 else F32
    size = k.dtype.itemsize
    parts = [x.reshape(tokens, -1) for x in ([q] if q is not None else []) + [k, v]]
    row = sum(p.shape[1] for p in parts) + pad
    rows = np.full((tokens, row), GUARD, k.dtype)
    rows[:, :row - pad] = np.concatenate(parts, 1)
    buffer = kl.Buffer(0, rows.nbytes + offset * size + 16)
    buffer.upload(rows.reshape(-1), offset=offset * size)
    at = buffer.data + offset * size
    q_row, kv_row = query_heads * c.width, c.heads * c.width
    out = np.full((tokens, q_row + pad), GUARD, k.dtype)
    out_buffer = upload(out)
    ints = [upload(np.asarray(x, np.int32)) if x is not None else None for x in (sequence, position, lengths, table)]
    angles = [upload(x.astype(np.float32)) if rotary else None for x in (cos, sin)]
    call = kl.KVAppendLayout(tokens, table.shape[0], table.shape[1], query_heads, row, row, row, row if in_place else q_row + pad,
                             rotary, len(cos) if rotary else 0, pairs, kind)
    assert kl.kv_append_f8_reason(cache.layout, call) == ""
    q_at = at if q is not None else None
    q_out = (at if in_place else out_buffer.data) if q is not None else None
    assert kl.kv_append_f8(kernel or kl.Kernel(), 0, *cache.pools(), q_out, q_at, at + q_row * size,
                           at + (q_row + kv_row) * size, *ints, *angles, cache.layout, call)
    finish()
    after = buffer.download(rows.shape, rows.dtype, offset=offset * size)
    if q is None:
        assert np.array_equal(after, rows, equal_nan=True), "inputs changed"
        return None
    if in_place:
        assert np.array_equal(after[:, q_row:], rows[:, q_row:], equal_nan=True), "wrote beside the queries"
        return after[:, :q_row].reshape(q.shape)
    assert np.array_equal(after, rows, equal_nan=True), "inputs changed"
    y = out_buffer.download(out.shape, out.dtype)
    assert np.all(y[:, q_row:] == np.array(GUARD, k.dtype)), "wrote between rows"
    return y[:, :q_row].reshape(q.shape)


def run_read(cache, table, sequence, position, dtype, lengths=None, pad=0, offset=0, common=False):
    """kv_read_f8 of the uploaded cache: k, v [tokens, heads, width] (rows that were left out hold GUARD)."""
    c = cache.layout.cache
    tokens = len(sequence) if sequence is not None else table.shape[0]
    width, size = c.heads * c.width, np.dtype(dtype).itemsize
    row = (2 * width if common else width) + pad
    out = np.full(offset + (1 if common else 2) * tokens * row, GUARD, dtype)
    buffer = upload(out)
    at = buffer.data + offset * size
    v_at = at + (width if common else tokens * row) * size
    ints = [upload(np.asarray(x, np.int32)) if x is not None else None for x in (sequence, position, lengths, table)]
    call = kl.KVReadLayout(tokens, table.shape[0], table.shape[1], row, row, F16 if dtype == np.float16 else F32)
    assert kl.kv_read_f8_reason(cache.layout, call) == ""
    assert kl.kv_read_f8(kl.Kernel(), 0, at, v_at, *cache.pools(), *ints, cache.layout, call)
    finish()
    flat = buffer.download(out.shape, dtype)
    assert np.all(flat[:offset] == np.array(GUARD, dtype))
    rows = flat[offset:].reshape(1 if common else 2, tokens, row)
    assert np.all(rows[:, :, row - pad:] == np.array(GUARD, dtype)), "wrote between rows"
    k, v = (rows[0, :, :width], rows[0, :, width:2 * width]) if common else (rows[0, :, :width], rows[1, :, :width])
    return [np.ascontiguousarray(x).reshape(tokens, c.heads, c.width) for x in (k, v)]


def model_read(cache, table, sequence, position, dtype, layer=0):
    c, block = cache.layout.cache, cache.layout.block_tokens
    page, at = table[sequence, position // c.page_tokens], position % c.page_tokens
    out = []
    for codes, scales in ((cache.k, cache.ks), (cache.v, cache.vs)):
        values = VALUES[codes[layer, page, :, at]] * scales[layer, page, :, at // block].astype(np.float64)[..., None]
        with np.errstate(over="ignore"):
            out.append(values.astype(dtype))
    return out
