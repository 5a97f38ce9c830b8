"""The decoding loop of examples/decode_loop.py over the 8-bit cache: each step's logits against the same model in 64
bits that attends to what the cache holds, and what the cache holds against the keys and values that went in."""
import importlib.util
import os

import numpy as np
import pytest

import kunlunk200_lib_amd as kl

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decode_loop.py")


@pytest.fixture(scope="module")
def loop():
    spec = importlib.util.spec_from_file_location("decode_loop", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def norm(x):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5)


class Model:
    """The newest token of a row in 64 bits, its attention over the given keys and values of each layer."""

    def __init__(self, c, w, decode):
        self.c, self.w = c, w
        self.layers = [{name: decode(q4) for name, q4 in host.items()} for host in w.host]
        self.head = decode(w.head_host)

    def turn(self, a, position):                   # [heads, width]
        half = self.c.width // 2
        angle = position / 10000.0 ** (np.arange(half) / half)
        cos, sin = (f(angle).astype(np.float32).astype(np.float64) for f in (np.cos, np.sin))
        a1, a2 = a[..., :half], a[..., half:]
        return np.concatenate([a1 * cos - a2 * sin, a1 * sin + a2 * cos], -1)

    def step(self, tokens, cached):
        """Logits, and per layer the newest token's key and value before they were rounded."""
        c, n, group = self.c, len(tokens), self.c.query_heads // self.c.heads
        x, fresh = self.w.embedding[tokens[-1]].astype(np.float64), []
        for m, (keys, values) in zip(self.layers, cached):
            y = (m["qkv"] @ norm(x)).reshape(-1, c.width)
            q, k, v = np.split(y, [c.query_heads, c.query_heads + c.heads])
            q = self.turn(q, n - 1)
            fresh.append((self.turn(k, n - 1), v))
            score = (np.repeat(keys, group, 1) * q).sum(-1) / np.sqrt(c.width)         # [tokens, query heads]
            p = np.exp(score - score.max(0))
            p /= p.sum(0)
            x = x + m["o"] @ (p[..., None] * np.repeat(values, group, 1)).sum(0).reshape(-1)
            h = norm(x)
            g = m["gate"] @ h
            x = x + m["down"] @ (g / (1 + np.exp(-g)) * (m["up"] @ h))
        z = self.head @ norm(x)
        times = np.bincount(tokens, minlength=c.vocabulary)
        r, f, p = (float(np.float32(t)) for t in (1.1, 0.05, 0.05))
        z = np.where(times > 0, np.where(z > 0, z / r, z * r) - times * f - p, z)
        z[:2] = -np.inf
        return z, fresh


@pytest.mark.parametrize("block_tokens", [1, 4, 16])
def test_decode_loop_f8(gpu, oracle, loop, block_tokens):
    c = loop.Config()
    w = loop.Weights(c, 7)
    decoder = loop.Decoder(c, w, block_tokens)
    rng = np.random.default_rng(8)
    prompts = [list(rng.integers(2, c.vocabulary, n)) for n in (20, 7, 33, 16)]

    def decode(q4):
        n = q4.shape[0]
        return oracle.q4_decode(q4, q4.size // n // 18 * 32, n).astype(np.float64)

    model = Model(c, w, decode)
    count = c.heads * c.width
    blocks = c.page_tokens // block_tokens

    def contents(row, n):
        """Per layer the first n keys and values of a row, [n, heads, width]."""
        call = kl.KVReadLayout(n, c.rows, c.row_pages, count, count, kl.InputType.f32)
        rows, at = loop.upload(np.full(n, row, np.int32)), loop.upload(np.arange(n, dtype=np.int32))
        out = []
        for i in range(c.layers):
            k, v = kl.Buffer(0, 4 * n * count), kl.Buffer(0, 4 * n * count)
            pools = [p.data + i * decoder.layer_bytes for p in (decoder.k, decoder.v)]
            scales = [s.data + i * decoder.scale_layer for s in (decoder.k_scales, decoder.v_scales)]
            kl.require(kl.kv_read_f8(decoder.kernel, 0, k, v, *pools, *scales, rows, at, None, decoder.table,
                                     decoder.cache8, call))
            kl.check(kl.wait())
            out.append([b.download((n, c.heads, c.width), np.float32).astype(np.float64) for b in (k, v)])
        return out

    def scales_of(row, n):
        """Per layer the scales of the first n tokens' keys and values, [n, heads]."""
        table = decoder.table.download((c.rows, c.row_pages), np.int32)[row]
        token = np.arange(n)
        out = []
        for s in (decoder.k_scales, decoder.v_scales):
            s = s.download((c.layers, c.pages, c.heads, blocks), np.float32).astype(np.float64)
            out.append(s[:, table[token // c.page_tokens], :, token % c.page_tokens // block_tokens])  # [n, layers, heads]
        return [[out[0][:, i], out[1][:, i]] for i in range(c.layers)]

    fresh = {}                                     # of each row: per token, per layer, the key and value that went in
    checked = []

    def observe(tokens, logits):
        for row in np.flatnonzero(tokens >= 0):
            sequence = list(decoder.history[row])
            n = len(sequence)
            assert sequence[-1] == tokens[row]
            if row >= c.rows - 2 and row not in fresh:
                fresh[row] = fresh[0][:n - 1]      # forked from row 0, whose list may be one longer already
            cached = contents(row, n)
            z, new = model.step(np.array(sequence), cached)
            fresh.setdefault(row, []).append(new)
            got = logits[row].astype(np.float64)
            assert np.array_equal(np.isneginf(z), np.isneginf(got))
            # F32 sums through two layers: a thousandth of the logits' size is a hundred times what they leave
            size = np.sqrt((z[2:] ** 2).mean())
            assert np.abs(got[2:] - z[2:]).max() <= 1e-3 * size, (row, n)
            # A code is off by half a step: 2^-4 of the value, or 2^-10 scales where it is subnormal. A block's scale
            # only doubles, which leaves normal codes exact; each growth rounds the subnormal ones again, by 2^-10 of
            # scales that end at the present one: 2^-9 of it together.
            # The fresh values come from products as exact as the logits.
            for layer, (pair, scale) in enumerate(zip(cached, scales_of(row, n))):
                for which in (0, 1):
                    went_in = np.stack([f[layer][which] for f in fresh[row]])
                    assert went_in.shape == pair[which].shape
                    exact = 1e-3 * np.sqrt((went_in ** 2).mean())
                    bound = np.abs(went_in) * 2.0 ** -4 + scale[which][..., None] * 2.0 ** -9 + exact
                    assert (np.abs(pair[which] - went_in) <= bound).all(), (row, n, layer, which)
            checked.append(row)

    out = loop.run(c, decoder, prompts, 24, observe)
    assert set(checked) >= {0, 1, 2, 3, c.rows - 2, c.rows - 1}
    lengths = decoder.lengths_now()
    assert lengths[1] == 0 and lengths[0] == 20 + len(out[0]) - 1      # all but the newest token are in the cache
    assert out[0][:24] == out[-1][:24] == out[-2][:24] and len({out[i][24] for i in (0, -1, -2)}) == 3
    used = int((decoder.references.download(c.pages, np.int32) > 0).sum())
    assert decoder.compact() == used
    assert kl.kv_cache_status(0) == 0
