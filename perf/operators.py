"""The operators around a paged key-value cache, and those on logits, as cases that can be timed and checked.

`run` computes them in their plain form (elementary torch operations in 32 bits) or, where
`own` is true, by the calls a program makes of kunlunk200_lib_amd. Head counts, widths and the
vocabulary are the Llama-2-7B ones that bench.py and the tests use (32 heads of 128, 32000
tokens), the same with 8 key-value heads, and odd ones.

`op` of a case:
  attention  one new token of each sequence over its pages of the cache (paged_attention)
  append     rotary rotation of new tokens' queries and keys, keys and values stored into
             their pages (kv_append)
  fork       sequences that continue others: full pages shared, the last one copied (kv_fork)
  compact    used pages moved to the low end of the pool, tables rewritten (kv_compact)
  logits     penalties for repeated tokens, biases and a grammar mask (process_logits)
"""
import torch

DEV = 0
own = False
_kernel = None


def listed():
    return [
        # one user's first tokens after a short question: launch and call cost
        {"name": "attn_b1_l33", "op": "attention", "sequences": 1, "query_heads": 32, "heads": 32, "width": 128,
         "page_tokens": 16, "longest": 33, "window": 0, "order": "heads", "f16": False},
        # one user with a long document, few key-value heads: the length has to be split
        {"name": "attn_b1_l32768", "op": "attention", "sequences": 1, "query_heads": 32, "heads": 8, "width": 128,
         "page_tokens": 64, "longest": 32768, "window": 0, "order": "heads", "f16": False},
        # continuous batching of ragged conversations, as many key-value heads as query heads
        {"name": "attn_b32_l4096", "op": "attention", "sequences": 32, "query_heads": 32, "heads": 32, "width": 128,
         "page_tokens": 16, "longest": 4096, "window": 0, "order": "heads", "f16": False},
        # a busy server in half precision, pages laid out token by token
        {"name": "attn_b64_l2048_f16", "op": "attention", "sequences": 64, "query_heads": 32, "heads": 8, "width": 128,
         "page_tokens": 32, "longest": 2048, "window": 0, "order": "tokens", "f16": True},
        # a sliding window, odd page, head and width sizes
        {"name": "attn_b7_window", "op": "attention", "sequences": 7, "query_heads": 15, "heads": 5, "width": 80,
         "page_tokens": 20, "longest": 3001, "window": 1000, "order": "heads", "f16": True},
        # a decode step of 32 sequences on the QKV product's rows
        {"name": "append_b32", "op": "append", "sequences": 32, "tokens": 32, "query_heads": 32, "heads": 32,
         "width": 128, "rotary": 128, "pairs": "adjacent", "page_tokens": 16, "order": "heads", "f16": False},
        # prompts of three users in one batch, a part of each head rotated in halves
        {"name": "append_t2047", "op": "append", "sequences": 3, "tokens": 2047, "query_heads": 32, "heads": 8,
         "width": 128, "rotary": 64, "pairs": "halves", "page_tokens": 64, "order": "tokens", "f16": False},
        # beam search of width 4
        {"name": "fork_4", "op": "fork", "sequences": 8, "forks": 4, "layers": 2, "pages": 256, "heads": 32,
         "width": 128, "page_tokens": 16, "longest": 500},
        # many samples of shared prompts
        {"name": "fork_100", "op": "fork", "sequences": 131, "forks": 100, "layers": 4, "pages": 4096, "heads": 8,
         "width": 128, "page_tokens": 32, "longest": 1500},
        # half the pool free in holes before a big prompt
        {"name": "compact_2048", "op": "compact", "sequences": 48, "layers": 4, "pages": 2048, "heads": 8,
         "width": 128, "page_tokens": 64, "longest": 1700},
        # one user's greedy step after a long answer
        {"name": "logits_b1", "op": "logits", "rows": 1, "vocabulary": 32000, "history": 700, "biases": 20},
        # a server's step: every row with its own history, biases and grammar
        {"name": "logits_b200", "op": "logits", "rows": 200, "vocabulary": 32000, "history": 3000, "biases": 300},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "append", "fork", "compact", "logits"])
    if op == "logits":
        vocabulary = _log(rng, 1000, 152000)
        return {"op": op, "rows": _log(rng, 1, min(200, 6400000 // vocabulary)), "vocabulary": vocabulary,
                "history": _log(rng, 1, 8000), "biases": _log(rng, 1, 400)}
    heads = rng.choice([1, 2, 4, 5, 8, 8, 32])
    width = rng.choice([64, 80, 96, 128, 128, 128, 256])
    token = heads * width * 2                       # values of one token in the cache, keys and values
    if op in ("attention", "append"):
        case = {"op": op, "sequences": _log(rng, 1, 64),
                "query_heads": heads * (1 if heads == 32 else rng.choice([1, 2, 3, 4, 7, 8])), "heads": heads,
                "width": width, "page_tokens": rng.choice([1, 16, 16, 20, 32, 64, 128]),
                "order": rng.choice(["heads", "heads", "tokens"]), "f16": rng.random() < 0.4}
        if op == "attention":
            case["longest"] = _log(rng, 1, max(64, min(40000, (1 << 28) // (token * case["sequences"]))))
            case["window"] = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
        else:
            case["tokens"] = _log(rng, 1, 2048)
            case["sequences"] = min(case["sequences"], case["tokens"])
            case["rotary"] = rng.choice([width, width, width // 2, 0])
            case["pairs"] = rng.choice(["adjacent", "halves"])
        return case
    layers, page_tokens = rng.choice([1, 2, 4]), rng.choice([16, 16, 24, 32, 64])
    pages = _log(rng, 64, max(128, min(4096, (1 << 27) // (token * page_tokens * layers))))
    case = {"op": op, "sequences": _log(rng, 4, 128), "layers": layers, "pages": pages, "heads": heads, "width": width,
            "page_tokens": page_tokens}
    case["longest"] = _log(rng, page_tokens, max(page_tokens + 1, pages * page_tokens // (case["sequences"] + 4)))
    if op == "fork":
        case["forks"] = max(1, int(case["sequences"] * rng.choice([0.25, 0.5, 0.75])))
    return case


# --- inputs ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _gauss(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * scale


def _half_pool(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float16)


def _ints(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)


def _lengths(g, n, longest):
    """Ragged lengths from one token up, as many in each octave; the first sequence is the longest, and of
    eight or more one is empty (a free place of the batch)."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    lengths = torch.exp(u * torch.log(torch.tensor(float(longest), dtype=torch.float64))).long().clamp(1, longest)
    # conversations that have gone on for a while: half of them in the upper half of the range
    lengths[1::2] = longest - lengths[1::2] // 2
    lengths[0] = longest
    if n >= 8:
        lengths[n // 2] = 0
    return lengths


def _rows_of_pages(lengths, page_tokens, ids, row_pages):
    """Table rows: sequence s takes its pages from `ids` in order; -1 past its last page."""
    need = (lengths + page_tokens - 1) // page_tokens
    first = torch.cumsum(need, 0) - need
    j = torch.arange(row_pages, device="cuda")
    at = (first[:, None] + j[None, :]).clamp(max=ids.numel() - 1)
    return torch.where(j[None, :] < need[:, None], ids[at], torch.full_like(at, -1)).int()


def _pool(g, case, pages, layers=1):
    shape = ((layers, pages, case["heads"], case["page_tokens"], case["width"]) if case.get("order", "heads") == "heads"
             else (layers, pages, case["page_tokens"], case["heads"], case["width"]))
    return _half_pool(g, *shape), _half_pool(g, *shape)


def _attention_inputs(case, seed):
    g, n, pt = _gen(seed), case["sequences"], case["page_tokens"]
    lengths = _lengths(g, n, case["longest"])
    row_pages = -(-case["longest"] // pt) + 3
    need = int(((lengths + pt - 1) // pt).sum())
    pages = need + need // 8 + 1
    table = _rows_of_pages(lengths, pt, torch.randperm(pages, generator=g, device="cuda"), row_pages)
    k, v = _pool(g, case, pages)
    q = _gauss(g, n, case["query_heads"], case["width"], scale=1.5)
    return {"k": k, "v": v, "table": table, "lengths": lengths.int(), "q": q.half() if case["f16"] else q}


def _append_inputs(case, seed):
    g, n, t, pt, w = _gen(seed), case["sequences"], case["tokens"], case["page_tokens"], case["width"]
    # tokens in order of their sequences; each sequence has a past of up to 300 tokens
    each = torch.full((n,), t // n, device="cuda", dtype=torch.int64)
    each[: t % n] += 1
    past = _ints(g, 0, 300, n).long()
    first = torch.cumsum(each, 0) - each
    sequence = torch.repeat_interleave(torch.arange(n, device="cuda"), each, output_size=t)
    position = past[sequence] + torch.arange(t, device="cuda") - first[sequence]
    lengths = past + each
    row_pages = -(-(300 + t) // pt)
    pages = n * -(-(300 + -(-t // n)) // pt) + 1
    table = _rows_of_pages(lengths, pt, torch.randperm(pages, generator=g, device="cuda"), row_pages)
    k, v = _pool(g, case, pages)
    rows = (case["query_heads"] + 2 * case["heads"]) * w
    qkv = _gauss(g, t, rows, scale=2.0)
    positions, half = 300 + t, case["rotary"] // 2
    angle = None
    if half:
        inverse = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * inverse[None, :]
    return {"k": k, "v": v, "table": table, "sequence": sequence.int(), "position": position.int(),
            "qkv": qkv.half() if case["f16"] else qkv,
            "cosine": torch.cos(angle).float() if half else None, "sine": torch.sin(angle).float() if half else None}


def _shared_cache(g, case, lengths, row_pages):
    """Tables and reference counts of sequences on random pages of the pool; every third sequence shares
    the full pages of the one before it as far as both go. Sequences the pool has no page for are empty."""
    pt, pages = case["page_tokens"], case["pages"]
    ids = torch.randperm(pages, generator=g, device="cuda")
    need = (lengths + pt - 1) // pt
    lengths = torch.where(torch.cumsum(need, 0) <= pages * 5 // 8, lengths, torch.zeros_like(lengths))
    table = _rows_of_pages(lengths, pt, ids, row_pages)
    n = lengths.numel()
    full = lengths // pt
    before = torch.roll(table, 1, 0)
    share = torch.minimum(full, torch.roll(full, 1, 0))
    share = torch.where(torch.arange(n, device="cuda") % 3 == 1, share, torch.zeros_like(share))
    j = torch.arange(row_pages, device="cuda")
    table = torch.where(j[None, :] < share[:, None], before, table)
    held = table >= 0
    references = torch.zeros(pages + 1, dtype=torch.int32, device="cuda")
    references.index_add_(0, torch.where(held, table, torch.full_like(table, pages)).flatten().long(),
                          torch.ones(table.numel(), dtype=torch.int32, device="cuda"))
    return table.contiguous(), lengths.int(), references[:pages].contiguous()


def _pages_inputs(case, seed):
    g, n = _gen(seed), case["sequences"]
    lengths = _ints(g, max(1, case["longest"] // 3), case["longest"] + 1, n).long()
    row_pages = -(-case["longest"] // case["page_tokens"]) + 1
    s = {}
    if case["op"] == "fork":
        order = torch.randperm(n, generator=g, device="cuda")
        children = order[: case["forks"]]
        lengths[children] = 0
        s["children"] = children.int()
        rest = order[case["forks"]:]
        s["parents"] = rest[_ints(g, 0, rest.numel(), case["forks"]).long()].int()
    table, lengths, references = _shared_cache(g, case, lengths, row_pages)
    k, v = _pool(g, case, case["pages"], case["layers"])
    return {**s, "table": table, "lengths": lengths, "references": references, "k": k, "v": v}


def _logits_inputs(case, seed):
    g, rows, vocabulary = _gen(seed), case["rows"], case["vocabulary"]
    # tokens repeat as in text: a few of them often
    u = torch.rand(rows, case["history"], generator=g, device="cuda")
    history = ((vocabulary ** u) - 1).int().clamp(0, vocabulary - 1)
    words = (vocabulary + 31) // 32
    mask = _ints(g, -(1 << 31), (1 << 31) - 1, rows, words) | _ints(g, -(1 << 31), (1 << 31) - 1, rows, words)
    mask[::3] = -1                                              # rows without a grammar: all allowed
    penalties = torch.stack([1 + 0.3 * torch.rand(rows, generator=g, device="cuda"),
                             0.5 * torch.rand(rows, generator=g, device="cuda"),
                             0.5 * torch.rand(rows, generator=g, device="cuda")], 1).contiguous()
    return {"logits": _gauss(g, rows, vocabulary, scale=3.0), "penalties": penalties, "history": history,
            "history_lengths": _ints(g, 0, case["history"] + 1, rows),
            "bias_ids": _ints(g, 0, vocabulary, rows, case["biases"]),
            "bias_values": _gauss(g, rows, case["biases"], scale=4.0),
            "bias_lengths": _ints(g, 0, case["biases"] + 1, rows), "mask": mask}


def _inputs(case, seed):
    return {"attention": _attention_inputs, "append": _append_inputs, "fork": _pages_inputs, "compact": _pages_inputs,
            "logits": _logits_inputs}[case["op"]](case, seed)


def prepare(case, seed):
    return {**_inputs(case, seed), "case": case}


# --- the plain form ---------------------------------------------------------------------

def _by_head(pool, case):
    """[layers, pages, heads, page_tokens, width] of a pool in either order."""
    return pool if case.get("order", "heads") == "heads" else pool.transpose(2, 3)


def _plain_attention(s, case):
    n, heads, width, pt = case["sequences"], case["heads"], case["width"], case["page_tokens"]
    groups = case["query_heads"] // heads
    pages = -(-case["longest"] // pt)
    at = s["table"][:, :pages].long().clamp(min=0)
    k = _by_head(s["k"], case)[0][at].float().transpose(1, 2).reshape(n, heads, pages * pt, width)
    v = _by_head(s["v"], case)[0][at].float().transpose(1, 2).reshape(n, heads, pages * pt, width)
    q = s["q"].float().view(n, heads, groups, width)
    t = torch.arange(pages * pt, device="cuda")
    length = s["lengths"].long()[:, None]
    first = (length - case["window"]).clamp(min=0) if case["window"] else torch.zeros_like(length)
    seen = ((t[None, :] < length) & (t[None, :] >= first))[:, None, None, :]
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * width ** -0.5
    score = torch.where(seen, score, torch.full_like(score, -torch.inf))
    top = score.amax(3, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(3, keepdim=True)
    y = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    return y.view(n, case["query_heads"], width).to(s["q"].dtype)


def _rotated(x, cosine, sine, pairs):
    """x [tokens, heads, width] with its first 2 * half values turned by the angles [tokens, half]."""
    if cosine is None:
        return x
    half = cosine.shape[1]
    c, s, turned = cosine[:, None, :], sine[:, None, :], x[:, :, :2 * half]
    if pairs == "adjacent":
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * s, a * s + b * c], 3).flatten(2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * c - b * s, a * s + b * c], 2)
    return torch.cat([turned, x[:, :, 2 * half:]], 2)


def _plain_append(s, case):
    t, heads, width, pt = case["tokens"], case["heads"], case["width"], case["page_tokens"]
    x = s["qkv"].float().view(t, case["query_heads"] + 2 * heads, width)
    q, k, v = x[:, :case["query_heads"]], x[:, case["query_heads"]:-heads], x[:, -heads:]
    position = s["position"].long()
    cosine = s["cosine"][position] if s["cosine"] is not None else None
    sine = s["sine"][position] if s["sine"] is not None else None
    page = s["table"][s["sequence"].long(), position // pt].long()
    _by_head(s["k"], case)[0][page, :, position % pt] = _rotated(k, cosine, sine, case["pairs"]).half()
    _by_head(s["v"], case)[0][page, :, position % pt] = v.half()
    return {"q": _rotated(q, cosine, sine, case["pairs"]).to(s["qkv"].dtype), "k": s["k"], "v": s["v"]}


def _plain_fork(s, case):
    pt, pages = case["page_tokens"], case["pages"]
    parents, children = s["parents"].long(), s["children"].long()
    table, lengths, references = s["table"], s["lengths"], s["references"]
    row_pages = table.shape[1]
    j = torch.arange(row_pages, device="cuda")[None, :]
    length = lengths[parents].long()
    full, rest = length // pt, length % pt
    need = rest > 0
    free = references == 0
    order = torch.argsort((~free).int(), stable=True)             # the free pages first, lowest first
    rank = torch.cumsum(need, 0) - 1
    granted = ~need | (rank < free.sum())
    new = order[rank.clamp(0, pages - 1)]
    old, rows = table[children], table[parents]
    last = rows.gather(1, full.clamp(max=row_pages - 1)[:, None])[:, 0].long().clamp(min=0)
    held = (lengths[children].long() + pt - 1) // pt
    counts = torch.cat([references, torch.zeros(1, dtype=torch.int32, device="cuda")])
    one = torch.ones(old.numel(), dtype=torch.int32, device="cuda")
    counts.index_add_(0, torch.where(j < held[:, None], old, torch.full_like(old, pages)).flatten().long(), -one)
    rows = torch.where((j == full[:, None]) & need[:, None], new[:, None], rows.long())
    rows = torch.where((j < full[:, None] + need[:, None]) & granted[:, None], rows, torch.full_like(rows, -1))
    counts.index_add_(0, torch.where(rows >= 0, rows, torch.full_like(rows, pages)).flatten(), one)
    references.copy_(counts[:pages])
    table[children] = rows.int()
    lengths[children] = torch.where(granted, length, torch.zeros_like(length)).int()
    copied = need & granted
    # what is not copied writes a page in use (the last of `order`: none of the new ones) over itself
    to, last = torch.where(copied, new, order[-1]), torch.where(copied, last, order[-1])
    part = (torch.arange(pt, device="cuda")[None, :] < torch.where(copied, rest, torch.full_like(rest, pt))[:, None])
    part = part[None, :, None, :, None]
    s["k"][:, to] = torch.where(part, s["k"][:, last], s["k"][:, to])
    s["v"][:, to] = torch.where(part, s["v"][:, last], s["v"][:, to])
    return {"table": table, "lengths": lengths, "references": references, "k": s["k"], "v": s["v"]}


def _plain_compact(s, case):
    pages, pt = case["pages"], case["page_tokens"]
    used = s["references"] > 0
    total = used.sum()
    ids = torch.arange(pages, device="cuda")
    hole, mover = ~used & (ids < total), used & (ids >= total)
    place = torch.cumsum(hole, 0) - 1
    holes = torch.zeros(pages + 1, dtype=torch.int64, device="cuda")
    holes[torch.where(hole, place, torch.full_like(place, pages))] = ids
    to = torch.where(mover, holes[(torch.cumsum(mover, 0) - 1).clamp(min=0)], ids)
    source = ids.clone()                                          # the page whose values a page ends with
    source = torch.cat([source, source[:1]])
    source[torch.where(mover, to, torch.full_like(to, pages))] = ids
    source = torch.where(hole, source[:pages], ids)
    s["k"].copy_(s["k"][:, source])
    s["v"].copy_(s["v"][:, source])
    held = torch.arange(s["table"].shape[1], device="cuda")[None, :] < ((s["lengths"].long() + pt - 1) // pt)[:, None]
    table = torch.where(held, to[s["table"].long().clamp(min=0)].int(), s["table"])
    references = torch.where(ids < total, s["references"][source], torch.zeros_like(s["references"]))
    return {"table": table, "references": references, "used": total.int(), "k": s["k"], "v": s["v"]}


def _plain_logits(s, case):
    rows, vocabulary = case["rows"], case["vocabulary"]
    z = s["logits"]
    ones = (torch.arange(case["history"], device="cuda")[None, :] < s["history_lengths"][:, None]).int()
    count = torch.zeros(rows, vocabulary, dtype=torch.int32, device="cuda").scatter_add_(1, s["history"].long(), ones)
    count = count.float()
    r, f, p = s["penalties"][:, 0:1], s["penalties"][:, 1:2], s["penalties"][:, 2:3]
    z = torch.where(count > 0, torch.where(z > 0, z / r, z * r), z)
    z = z - count * f - (count > 0).float() * p
    # the last entry of a token counts
    entry = torch.arange(1, case["biases"] + 1, device="cuda")[None, :].expand(rows, -1)
    entry = torch.where(entry <= s["bias_lengths"][:, None], entry, torch.zeros_like(entry))
    last = torch.zeros(rows, vocabulary, dtype=torch.int64, device="cuda")
    last.scatter_reduce_(1, s["bias_ids"].long(), entry, "amax")
    bias = s["bias_values"].gather(1, (last - 1).clamp(min=0))
    z = z + torch.where(last > 0, bias, torch.zeros_like(bias))
    t = torch.arange(vocabulary, device="cuda")
    allowed = ((s["mask"][:, t // 32] >> (t % 32)[None, :].int()) & 1) != 0
    return torch.where(allowed, z, torch.full_like(z, -torch.inf))


# --- the library's calls ------------------------------------------------------------------

def _library():
    global _kernel
    import kunlunk200_lib_amd as kl
    if _kernel is None:
        _kernel = kl.Kernel()
    return kl, _kernel


def _cache(kl, s, case):
    pages, pt, heads, width = s["k"].shape[1], case["page_tokens"], case["heads"], case["width"]
    if case.get("order", "heads") == "heads":
        return kl.KVCacheLayout(pages, pt, heads, width, heads * pt * width, pt * width, width)
    return kl.KVCacheLayout(pages, pt, heads, width, heads * pt * width, width, heads * width)


def _own_attention(s, case):
    kl, kernel = _library()
    q, table = s["q"], s["table"]
    y = torch.empty_like(q)
    row = case["query_heads"] * case["width"]
    call = kl.PagedAttentionLayout(case["sequences"], case["query_heads"], case["longest"], case["window"],
                                   table.shape[1], row, row, case["width"] ** -0.5, case["f16"])
    kl.require(kl.paged_attention(kernel, DEV, y.data_ptr(), q.data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(),
                                  table.data_ptr(), s["lengths"].data_ptr(), _cache(kl, s, case), call))
    return y


def _own_append(s, case):
    kl, kernel = _library()
    qkv, heads, width = s["qkv"], case["heads"], case["width"]
    row, size = qkv.shape[1], qkv.element_size()
    q = torch.empty(case["tokens"], case["query_heads"], width, dtype=qkv.dtype, device="cuda")
    at = qkv.data_ptr()
    pairs = kl.RotaryPairs.adjacent if case["pairs"] == "adjacent" else kl.RotaryPairs.halves
    call = kl.KVAppendLayout(case["tokens"], case["sequences"], s["table"].shape[1], case["query_heads"],
                             row, row, row, case["query_heads"] * width, case["rotary"], 300 + case["tokens"], pairs,
                             case["f16"])
    turned = s["cosine"] is not None
    kl.require(kl.kv_append(kernel, DEV, s["k"].data_ptr(), s["v"].data_ptr(), q.data_ptr(), at,
                            at + case["query_heads"] * width * size, at + (row - heads * width) * size,
                            s["sequence"].data_ptr(), s["position"].data_ptr(), None, s["table"].data_ptr(),
                            s["cosine"].data_ptr() if turned else None, s["sine"].data_ptr() if turned else None,
                            _cache(kl, s, case), call))
    return {"q": q, "k": s["k"], "v": s["v"]}


def _pages_of(kl, s, case):
    return kl.KVPagesLayout(case["sequences"], s["table"].shape[1], case["layers"], s["k"][0].numel())


def _own_fork(s, case):
    kl, kernel = _library()
    kl.require(kl.kv_fork(kernel, DEV, s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(),
                          s["lengths"].data_ptr(), s["references"].data_ptr(), s["parents"].data_ptr(),
                          s["children"].data_ptr(), case["forks"], _cache(kl, s, case), _pages_of(kl, s, case)))
    return {"table": s["table"], "lengths": s["lengths"], "references": s["references"], "k": s["k"], "v": s["v"]}


def _own_compact(s, case):
    kl, kernel = _library()
    table, references = torch.empty_like(s["table"]), torch.empty_like(s["references"])
    used = torch.empty((), dtype=torch.int32, device="cuda")
    kl.require(kl.kv_compact(kernel, DEV, s["k"].data_ptr(), s["v"].data_ptr(), table.data_ptr(),
                             references.data_ptr(), used.data_ptr(), s["table"].data_ptr(), s["lengths"].data_ptr(),
                             s["references"].data_ptr(), _cache(kl, s, case), _pages_of(kl, s, case)))
    return {"table": table, "references": references, "used": used, "k": s["k"], "v": s["v"]}


def _own_logits(s, case):
    kl, kernel = _library()
    z = s["logits"]
    y = torch.empty_like(z)
    call = kl.LogitsLayout(case["rows"], case["vocabulary"], case["vocabulary"], case["vocabulary"], case["history"],
                           case["biases"], s["mask"].shape[1])
    kl.require(kl.process_logits(kernel, DEV, y.data_ptr(), z.data_ptr(), s["penalties"].data_ptr(),
                                 s["history"].data_ptr(), s["history_lengths"].data_ptr(), s["bias_ids"].data_ptr(),
                                 s["bias_values"].data_ptr(), s["bias_lengths"].data_ptr(), s["mask"].data_ptr(), call))
    return y


def run(state):
    case = state["case"]
    if own:
        form = {"attention": _own_attention, "append": _own_append, "fork": _own_fork, "compact": _own_compact,
                "logits": _own_logits}
    else:
        form = {"attention": _plain_attention, "append": _plain_append, "fork": _plain_fork,
                "compact": _plain_compact, "logits": _plain_logits}
    return form[case["op"]](state, case)


# --- what a pass cannot do without ----------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "logits":
        rows, vocabulary = case["rows"], case["vocabulary"]
        lists = rows * (case["history"] * 4 + case["biases"] * 8) // 2      # half full on average
        return {"bytes": rows * (8 * vocabulary + vocabulary // 8 + 20) + lists, "flops": 3 * rows * vocabulary}
    heads, width, pt = case["heads"], case["width"], case["page_tokens"]
    token = 2 * heads * width * 2                                           # bytes of a token in the cache
    size = 2 if case.get("f16") else 4
    if op == "attention":
        # about the mean of _lengths()
        n, longest = case["sequences"], case["longest"]
        window = case["window"] or longest
        short, long = (min(window, part * longest) for part in ((0.13, 0.94) if n > 1 else (1, 1)))
        seen = max(1, int(n * (short + long) / 2))
        return {"bytes": seen * token + 2 * n * case["query_heads"] * width * size + 4 * -(-seen // pt) + 4 * n,
                "flops": 4 * seen * case["query_heads"] * width}
    if op == "append":
        t, values = case["tokens"], case["query_heads"] * width
        return {"bytes": t * (2 * values * size + 2 * heads * width * size + token + 4 * case["rotary"] + 12),
                "flops": 3 * t * case["rotary"] * (case["query_heads"] + heads)}
    row_pages = -(-case["longest"] // pt) + 1
    if op == "fork":
        # a copied last page is half full on average; rows are read and written, counts read
        copied = case["forks"] * token * pt // 2 * case["layers"]
        return {"bytes": 2 * copied + case["forks"] * row_pages * 8 + 4 * case["pages"], "flops": 0}
    # of the used share u of the pool, (1 - u) u pages move
    used = min(0.6, case["sequences"] * 0.55 * case["longest"] / (pt * case["pages"]))
    moved = int(case["pages"] * used * (1 - used)) * token * pt * case["layers"]
    return {"bytes": 2 * moved + case["sequences"] * row_pages * 8 + 8 * case["pages"], "flops": 0}


# --- the same in 64 bits --------------------------------------------------------------------

def _exact_attention(s, case):
    heads, width, pt = case["heads"], case["width"], case["page_tokens"]
    groups = case["query_heads"] // heads
    y = torch.zeros(case["sequences"], case["query_heads"], width, dtype=torch.float64, device="cuda")
    for i, length in enumerate(s["lengths"].tolist()):
        first = max(0, length - case["window"]) if case["window"] else 0
        if length == 0:
            continue
        t = torch.arange(first, length, device="cuda")
        page, at = s["table"][i].long()[t // pt], t % pt
        for h in range(heads):
            if case["order"] == "heads":
                k, v = s["k"][0, page, h, at].double(), s["v"][0, page, h, at].double()
            else:
                k, v = s["k"][0, page, at, h].double(), s["v"][0, page, at, h].double()
            q = s["q"][i, h * groups:(h + 1) * groups].double()
            weight = torch.softmax((k @ q.T) / width ** 0.5, 0)
            y[i, h * groups:(h + 1) * groups] = weight.T @ v
    return y


def _exact_append(s, case):
    heads, width, pt, half = case["heads"], case["width"], case["page_tokens"], case["rotary"] // 2
    x = s["qkv"].double().view(case["tokens"], -1, width)
    if half:
        position = s["position"].long()
        turn = torch.complex(s["cosine"][position].double(), s["sine"][position].double())[:, None, :]
        part = x[:, :-heads, :2 * half]
        if case["pairs"] == "adjacent":
            z = torch.complex(part[..., 0::2].contiguous(), part[..., 1::2].contiguous()) * turn
            x[:, :-heads, 0:2 * half:2], x[:, :-heads, 1:2 * half:2] = z.real, z.imag
        else:
            z = torch.complex(part[..., :half].contiguous(), part[..., half:].contiguous()) * turn
            x[:, :-heads, :half], x[:, :-heads, half:2 * half] = z.real, z.imag
    k, v = s["k"].double(), s["v"].double()
    sequence, position = s["sequence"].tolist(), s["position"].tolist()
    rows = s["table"].tolist()
    for t in range(case["tokens"]):
        page, at = rows[sequence[t]][position[t] // pt], position[t] % pt
        if case["order"] == "heads":
            k[0, page, :, at], v[0, page, :, at] = x[t, -2 * heads:-heads], x[t, -heads:]
        else:
            k[0, page, at], v[0, page, at] = x[t, -2 * heads:-heads], x[t, -heads:]
    return {"q": x[:, :case["query_heads"]].contiguous(), "k": k, "v": v}


def _exact_fork(s, case):
    pt = case["page_tokens"]
    k, v = s["k"].double(), s["v"].double()
    rows, lengths = s["table"].tolist(), s["lengths"].tolist()
    free = [p for p, c in enumerate(s["references"].tolist()) if c == 0]
    for parent in s["parents"].tolist():
        full, rest = divmod(lengths[parent], pt)
        if rest and free:
            page = free.pop(0)
            k[:, page, :, :rest] = s["k"][:, rows[parent][full], :, :rest].double()
            v[:, page, :, :rest] = s["v"][:, rows[parent][full], :, :rest].double()
    return {"table": None, "lengths": None, "references": None, "k": k, "v": v}


def _exact_compact(s, case):
    k, v = s["k"].double(), s["v"].double()
    counts = s["references"].tolist()
    total = sum(c > 0 for c in counts)
    holes = [p for p in range(total) if counts[p] == 0]
    for to, page in zip(holes, [p for p in range(total, len(counts)) if counts[p] > 0]):
        k[:, to], v[:, to] = s["k"][:, page].double(), s["v"][:, page].double()
    return {"table": None, "references": None, "used": None, "k": k, "v": v}


def _exact_logits(s, case):
    y = s["logits"].double()
    vocabulary = case["vocabulary"]
    for i in range(case["rows"]):
        r, f, p = s["penalties"][i].double().tolist()
        count = torch.bincount(s["history"][i, :int(s["history_lengths"][i])].long(), minlength=vocabulary).double()
        met = count > 0
        z = y[i]
        z[met & (z > 0)] /= r
        z[met & (s["logits"][i] <= 0)] *= r
        z -= f * count + p * met.double()
        bias = {}
        n = int(s["bias_lengths"][i])
        for token, value in zip(s["bias_ids"][i, :n].tolist(), s["bias_values"][i, :n].double().tolist()):
            bias[token] = value
        if bias:
            z[torch.tensor(list(bias), device="cuda")] += torch.tensor(list(bias.values()), dtype=torch.float64,
                                                                       device="cuda")
        bits = (s["mask"][i].long()[:, None] >> torch.arange(32, device="cuda")[None, :]) & 1
        z[bits.flatten()[:vocabulary] == 0] = -torch.inf
    return y


def exact(case, seed):
    s = _inputs(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "fork": _exact_fork, "compact": _exact_compact,
            "logits": _exact_logits}[case["op"]](s, case)
