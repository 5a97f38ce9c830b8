"""A decoding loop over the paged key-value cache: a small Llama-like model with Q4_0 weights (random
ones, since the loop is the point) decodes several prompts at once, continues one of them in three ways, gives the
finished sequences' pages back and compacts the pool.

Each step takes one token of every row: room for it (kv_reserve), then per layer the QKV
product, its rotation and storage (kv_append), attention over the pages (paged_attention), the output product and the
feed-forward block, then the LM head and the penalties on its logits (process_logits).

Run on a machine with the library built:  python examples/decode_loop.py
"""
import os
import sys

import numpy as np

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import kunlunk200_lib_amd as kl  # noqa: E402

DEVICE = 0
EPS = 1e-5


class Config:
    hidden, ffn, layers, vocabulary = 256, 512, 2, 1000
    query_heads, heads, width = 4, 2, 64
    pages, page_tokens, row_pages, rows = 64, 16, 8, 6

    @property
    def qkv(self):
        return (self.query_heads + 2 * self.heads) * self.width


def upload(array):
    array = np.ascontiguousarray(array)
    buffer = kl.Buffer(DEVICE, max(array.nbytes, 16))
    buffer.upload(array)
    return buffer


class Weights:
    """Q4_0 projections on the device; `host` keeps what was quantized, by name."""

    def __init__(self, c, seed):
        rng = np.random.default_rng(seed)
        self.embedding = rng.standard_normal((c.vocabulary, c.hidden)).astype(np.float32)
        self.layers, self.host = [], []
        shapes = {"qkv": (c.qkv, c.hidden), "o": (c.hidden, c.query_heads * c.width), "gate": (c.ffn, c.hidden),
                  "up": (c.ffn, c.hidden), "down": (c.hidden, c.ffn)}
        for _ in range(c.layers):
            host = {n: kl.quantize_q4_0((rng.standard_normal(s) / np.sqrt(s[1])).astype(np.float32))
                    for n, s in shapes.items()}
            self.host.append(host)
            self.layers.append({n: upload(w) for n, w in host.items()})
        self.head_host = kl.quantize_q4_0((rng.standard_normal((c.vocabulary, c.hidden)) / 8).astype(np.float32))
        self.head = upload(self.head_host)


class Decoder:
    def __init__(self, c, weights):
        self.c, self.w, self.kernel = c, weights, kl.Kernel()
        pool = c.heads * c.page_tokens * c.width                       # values of a page
        self.cache = kl.KVCacheLayout(c.pages, c.page_tokens, c.heads, c.width, pool, c.page_tokens * c.width, c.width)
        self.pages = kl.KVPagesLayout(c.rows, c.row_pages, c.layers, c.pages * pool)
        self.layer_bytes = c.pages * pool * 2
        zeros = np.zeros(c.layers * c.pages * pool, np.float16)
        self.k, self.v = upload(zeros), upload(zeros)
        self.table = upload(np.full((c.rows, c.row_pages), -1, np.int32))
        self.lengths = upload(np.zeros(c.rows, np.int32))
        self.references = upload(np.zeros(c.pages, np.int32))
        self.every_row = upload(np.arange(c.rows, dtype=np.int32))
        most = c.row_pages * c.page_tokens
        angle = np.arange(most)[:, None] / 10000.0 ** (np.arange(c.width // 2) / (c.width // 2))[None, :]
        self.cosine, self.sine = upload(np.cos(angle).astype(np.float32)), upload(np.sin(angle).astype(np.float32))
        f = lambda n: kl.Buffer(DEVICE, 4 * c.rows * n)  # noqa: E731
        self.x, self.h, self.y = f(c.hidden), f(c.hidden), f(c.hidden)
        self.qkv, self.q, self.attended, self.act = f(c.qkv), f(c.query_heads * c.width), f(c.query_heads * c.width), f(c.ffn)
        self.logits = f(c.vocabulary)
        self.history = [[] for _ in range(c.rows)]
        q, row = c.query_heads * c.width, c.qkv
        self.append = kl.KVAppendLayout(c.rows, c.rows, c.row_pages, c.query_heads, row, row, row, q, c.width, most,
                                        kl.RotaryPairs.halves, kl.InputType.f32)
        self.attend = kl.PagedAttentionLayout(c.rows, c.query_heads, most, 0, c.row_pages, q, q, c.width ** -0.5,
                                              kl.InputType.f32)

    def lengths_now(self):
        return self.lengths.download(self.c.rows, np.int32)

    def step(self, tokens, penalties=(1.1, 0.05, 0.05), forbidden=()):
        """One token of each row (negative: the row rests); the logits [rows, vocabulary] of what follows."""
        c, kernel = self.c, self.kernel
        rests = tokens < 0
        self.x.upload(self.w.embedding[np.maximum(tokens, 0)])
        for row in np.flatnonzero(~rests):
            self.history[row].append(int(tokens[row]))
        added = upload((~rests).astype(np.int32))
        # rows that rest are left out of the append by a negative position, the others' token is their newest
        at = np.where(rests, -1, self.lengths_now()).astype(np.int32)
        position = upload(at)
        with kl.runtime_mutex():
            kl.require(kl.kv_reserve(kernel, DEVICE, self.table, self.lengths, self.references, self.every_row, added,
                                     c.rows, self.cache, self.pages))
            for i in range(c.layers):
                self._layer(i, position)
            self._norm(self.h, self.x)
            kl.matmul(kernel, DEVICE, self.logits, self.w.head, self.h, c.hidden, c.vocabulary, c.rows,
                      kl.WeightType.q4_0)
            self._penalties(penalties, forbidden)
            kl.select(DEVICE)
            kl.check(kl.wait())
        kl.require(kl.kv_cache_status(DEVICE) == 0)
        return self.logits.download((c.rows, c.vocabulary), np.float32)

    def _norm(self, y, x):
        c = self.c
        kl.elementwise(self.kernel, DEVICE, y, x, x, c.rows * c.hidden, c.hidden, c.rows * c.hidden,
                       kl.ElementwiseOp.rms_norm, EPS)

    def _add(self, y, a, b):
        c = self.c
        kl.elementwise(self.kernel, DEVICE, y, a, b, c.rows * c.hidden, c.hidden, c.rows * c.hidden,
                       kl.ElementwiseOp.add)

    def _layer(self, i, position):
        c, kernel, w, q4 = self.c, self.kernel, self.w.layers[i], kl.WeightType.q4_0
        k, v = self.k.data + i * self.layer_bytes, self.v.data + i * self.layer_bytes
        q_bytes, kv_bytes = 4 * c.query_heads * c.width, 4 * c.heads * c.width
        self._norm(self.h, self.x)
        kl.matmul(kernel, DEVICE, self.qkv, w["qkv"], self.h, c.hidden, c.qkv, c.rows, q4)
        at = self.qkv.data
        kl.require(kl.kv_append(kernel, DEVICE, k, v, self.q, at, at + q_bytes, at + q_bytes + kv_bytes, self.every_row,
                                position, None, self.table, self.cosine, self.sine, self.cache, self.append))
        kl.require(kl.paged_attention(kernel, DEVICE, self.attended, self.q, k, v, self.table, self.lengths, self.cache,
                                      self.attend))
        kl.matmul(kernel, DEVICE, self.y, w["o"], self.attended, c.query_heads * c.width, c.hidden, c.rows, q4)
        self._add(self.x, self.x, self.y)
        self._norm(self.h, self.x)
        kl.matmul_swiglu(kernel, DEVICE, self.act, w["gate"], w["up"], self.h, c.hidden, c.ffn, c.rows, q4)
        kl.matmul(kernel, DEVICE, self.y, w["down"], self.act, c.ffn, c.hidden, c.rows, q4)
        self._add(self.x, self.x, self.y)

    def _penalties(self, penalties, forbidden):
        c = self.c
        longest = max(1, max(len(h) for h in self.history))
        history = np.full((c.rows, longest), -1, np.int32)
        for row, h in enumerate(self.history):
            history[row, :len(h)] = h
        words = np.full((c.vocabulary + 31) // 32, 0xffffffff, np.uint32)
        for token in forbidden:
            words[token // 32] &= ~np.uint32(1 << (token % 32))
        b = [upload(x) for x in (np.tile(np.float32(penalties), (c.rows, 1)), history,
                                 np.array([len(h) for h in self.history], np.int32), words)]
        call = kl.LogitsLayout(c.rows, c.vocabulary, c.vocabulary, c.vocabulary, longest, 0, 0)
        kl.require(kl.process_logits(self.kernel, DEVICE, self.logits, self.logits, b[0], b[1], b[2], None, None, None,
                                     b[3], call))
        kl.check(kl.wait())                                # the lists are freed when this returns

    def fork(self, parents, children):
        """children[i] goes on where parents[i] stands."""
        p, c = upload(np.array(parents, np.int32)), upload(np.array(children, np.int32))
        kl.require(kl.kv_fork(self.kernel, DEVICE, self.k, self.v, self.table, self.lengths, self.references, p, c,
                              len(parents), self.cache, self.pages))
        kl.require(kl.kv_cache_status(DEVICE) == 0)
        histories = [list(self.history[i]) for i in parents]
        for child, h in zip(children, histories):
            self.history[child] = h

    def free(self, rows):
        r = upload(np.array(rows, np.int32))
        kl.require(kl.kv_free(self.kernel, DEVICE, self.table, self.lengths, self.references, r, len(rows), self.cache,
                              self.pages))
        kl.require(kl.kv_cache_status(DEVICE) == 0)
        for row in rows:
            self.history[row] = []

    def compact(self):
        """Moves the used pages to the low end; how many there are."""
        used = upload(np.zeros(1, np.int32))
        kl.require(kl.kv_compact(self.kernel, DEVICE, self.k, self.v, self.table, self.references, used, self.table,
                                 self.lengths, self.references, self.cache, self.pages))
        kl.require(kl.kv_cache_status(DEVICE) == 0)
        return int(used.download(1, np.int32)[0])


def run(c, decoder, prompts, steps, observe=lambda tokens, logits: None):
    """Prompts (at most rows - 2 of them) token by token, then `steps` greedy tokens; after half of them row 0 goes on in
    rows rows - 2 and rows - 1 too, with its second and third choice, row 1 ends and the pool is compacted. Every step's
    tokens and logits go to `observe`; returns the tokens of each row."""
    out = [[] for _ in range(c.rows)]
    pending = [list(p) for p in prompts] + [[] for _ in range(c.rows - len(prompts))]
    tokens = np.array([p.pop(0) if p else -1 for p in pending])
    active = tokens >= 0
    made = 0
    while made < steps:
        logits = decoder.step(tokens, forbidden=(0, 1))
        observe(tokens.copy(), logits)
        best = np.argsort(-logits, axis=1, kind="stable")
        tokens = np.where(active, best[:, 0], -1)
        prompting = [row for row in np.flatnonzero(active) if pending[row]]
        for row in prompting:
            tokens[row] = pending[row].pop(0)
        if not prompting:
            made += 1
            if made == steps // 2:
                branches = [c.rows - 2, c.rows - 1]
                decoder.fork([0, 0], branches)
                for place, row in enumerate(branches):
                    out[row], active[row], tokens[row] = list(out[0]), True, best[0, place + 1]
                decoder.free([1])
                active[1], tokens[1] = False, -1
                decoder.compact()
        for row in np.flatnonzero(active):
            if row not in prompting:
                out[row].append(int(tokens[row]))
    return out


def main():
    c = Config()
    decoder = Decoder(c, Weights(c, 1))
    rng = np.random.default_rng(2)
    prompts = [list(rng.integers(2, c.vocabulary, n)) for n in (20, 7, 33, 16)]
    for row, tokens in enumerate(run(c, decoder, prompts, 24)):
        print(f"row {row}: {tokens}")
    print("tokens in the cache:", decoder.lengths_now().tolist())


if __name__ == "__main__":
    main()
