"""The decoding loop of examples/decode_loop.py, which runs the paged cache's operators
together, against the same model in 64 bits over the whole of each sequence."""
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


def whole_sequence(c, w, decode, tokens):
    """Logits after the last of `tokens`, everything in 64 bits except the cache's F16 rounding of keys and values."""
    x = w.embedding[tokens].astype(np.float64)
    n, half, group = len(tokens), c.width // 2, c.query_heads // c.heads
    angle = np.arange(n)[:, None] / 10000.0 ** (np.arange(half) / half)[None, :]
    cos, sin = np.cos(angle).astype(np.float32).astype(np.float64), np.sin(angle).astype(np.float32).astype(np.float64)

    def turn(a):                                   # [tokens, heads, width]
        a1, a2 = a[..., :half], a[..., half:]
        return np.concatenate([a1 * cos[:, None] - a2 * sin[:, None], a1 * sin[:, None] + a2 * cos[:, None]], -1)

    for host in w.host:
        m = {name: decode(q4) for name, q4 in host.items()}
        y = (norm(x) @ m["qkv"].T).reshape(n, -1, c.width)
        q, k, v = np.split(y, [c.query_heads, c.query_heads + c.heads], 1)
        q, k, v = turn(q), turn(k).astype(np.float16).astype(np.float64), v.astype(np.float16).astype(np.float64)
        score = np.einsum("qhd,khd->hqk", q, np.repeat(k, group, 1)) / np.sqrt(c.width)
        score = np.where(np.tril(np.ones((n, n), bool)), score, -np.inf)
        p = np.exp(score - score.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        x = x + np.einsum("hqk,khd->qhd", p, np.repeat(v, group, 1)).reshape(n, -1) @ m["o"].T
        h = norm(x)
        g = h @ m["gate"].T
        x = x + (g / (1 + np.exp(-g)) * (h @ m["up"].T)) @ m["down"].T
    z = norm(x[-1]) @ decode(w.head_host).T
    times = np.bincount(tokens, minlength=c.vocabulary)
    r, f, p = (float(np.float32(t)) for t in (1.1, 0.05, 0.05))
    z = np.where(times > 0, np.where(z > 0, z / r, z * r) - times * f - p, z)
    z[:2] = -np.inf
    return z


def test_decode_loop(gpu, oracle, loop):
    c = loop.Config()
    w = loop.Weights(c, 7)
    decoder = loop.Decoder(c, w)
    rng = np.random.default_rng(8)
    prompts = [list(rng.integers(2, c.vocabulary, n)) for n in (20, 7, 33, 16)]

    def decode(q4):
        n = q4.shape[0]
        return oracle.q4_decode(q4, q4.size // n // 18 * 32, n).astype(np.float64)

    rows = [[] for _ in range(c.rows)]
    checked = []

    def observe(tokens, logits):
        for row in np.flatnonzero(tokens >= 0):
            rows[row] = list(decoder.history[row])
            assert rows[row][-1] == tokens[row]
            if len(rows[row]) % 5 and row < c.rows - 2:
                continue                           # every fifth length, and every step of the forked rows
            z = whole_sequence(c, w, decode, np.array(rows[row]))
            got = logits[row].astype(np.float64)
            assert np.array_equal(np.isneginf(z), np.isneginf(got))
            # F32 sums through two layers: a thousandth of the logits' size is a hundred times what they leave
            size = np.sqrt((z[2:] ** 2).mean())
            assert np.abs(got[2:] - z[2:]).max() <= 1e-3 * size, (row, len(rows[row]))
            checked.append(row)

    out = loop.run(c, decoder, prompts, 24, observe)
    assert set(checked) >= {0, 2, c.rows - 2, c.rows - 1} and len(checked) > 30
    lengths = decoder.lengths_now()
    # all but the newest token are in the cache
    assert lengths[1] == 0 and lengths[0] == 20 + len(out[0]) - 1
    # row 0 answered alone for the 13 tokens that the longest prompt has more, then 11 times with the others
    assert out[0][:24] == out[-1][:24] == out[-2][:24] and len({out[i][24] for i in (0, -1, -2)}) == 3
    used = int((decoder.references.download(c.pages, np.int32) > 0).sum())
    assert decoder.compact() == used
    assert kl.kv_cache_status(0) == 0
