"""The operators of a paged key-value cache held in 8 bits, as cases that can be timed and checked.

`run` computes them in their plain form (elementary torch operations in 32 bits) or, where
`own` is true, by the calls a program makes of kunlunk200_lib_amd. The pools hold e4m3 codes, and
every block of `block_tokens` tokens of a head has an F32 scale; a value is code * scale. Head counts
and widths are the Llama-2-7B ones that bench.py and the tests use (32 heads of 128), the same with
8 key-value heads, and odd ones.

`op` of a case:
  attention  one new token of each sequence over its pages of the cache (paged_attention_f8)
  append     rotary rotation of new tokens' queries and keys, keys and values quantised into their
             pages (kv_append_f8), and every block that this wrote read back (kv_read_f8)
  read       whole histories of several sequences read back as rows (kv_read_f8)
"""
import torch

DEV = 0
own = False
_kernel = None


def listed():
    return [
        # one user's first tokens after a short question: launch and call cost
        {"name": "attn_b1_l40", "op": "attention", "sequences": 1, "query_heads": 32, "heads": 32, "width": 128,
         "page_tokens": 16, "block_tokens": 16, "longest": 40, "window": 0, "order": "heads", "f16": False},
        # one user with a long document, few key-value heads: the length has to be split
        {"name": "attn_b1_l32768", "op": "attention", "sequences": 1, "query_heads": 32, "heads": 8, "width": 128,
         "page_tokens": 64, "block_tokens": 64, "longest": 32768, "window": 0, "order": "heads", "f16": False},
        # continuous batching of ragged conversations, as many key-value heads as query heads
        {"name": "attn_b32_l4096", "op": "attention", "sequences": 32, "query_heads": 32, "heads": 32, "width": 128,
         "page_tokens": 16, "block_tokens": 16, "longest": 4096, "window": 0, "order": "heads", "f16": False},
        # a busy server in half precision, pages laid out token by token, a scale for every token
        {"name": "attn_b64_l2048_f16", "op": "attention", "sequences": 64, "query_heads": 32, "heads": 8, "width": 128,
         "page_tokens": 32, "block_tokens": 1, "longest": 2048, "window": 0, "order": "tokens", "f16": True},
        # many short conversations at once
        {"name": "attn_b200_l700", "op": "attention", "sequences": 200, "query_heads": 32, "heads": 8, "width": 128,
         "page_tokens": 16, "block_tokens": 8, "longest": 700, "window": 0, "order": "heads", "f16": False},
        # a sliding window, odd page, head and width sizes
        {"name": "attn_b7_window", "op": "attention", "sequences": 7, "query_heads": 15, "heads": 5, "width": 80,
         "page_tokens": 20, "block_tokens": 4, "longest": 3001, "window": 1000, "order": "heads", "f16": True},
        # one user's decode step
        {"name": "append_b1", "op": "append", "sequences": 1, "tokens": 1, "query_heads": 32, "heads": 32,
         "width": 128, "rotary": 128, "pairs": "adjacent", "page_tokens": 16, "block_tokens": 16, "order": "heads",
         "f16": False},
        # a decode step of 32 sequences on the QKV product's rows
        {"name": "append_b32", "op": "append", "sequences": 32, "tokens": 32, "query_heads": 32, "heads": 32,
         "width": 128, "rotary": 128, "pairs": "adjacent", "page_tokens": 16, "block_tokens": 16, "order": "heads",
         "f16": False},
        # prompts of three users in one batch, a part of each head rotated in halves
        {"name": "append_t2047", "op": "append", "sequences": 3, "tokens": 2047, "query_heads": 32, "heads": 8,
         "width": 128, "rotary": 64, "pairs": "halves", "page_tokens": 64, "block_tokens": 64, "order": "tokens",
         "f16": False},
        # a prompt in half precision, a scale for every token
        {"name": "append_t1500_f16", "op": "append", "sequences": 2, "tokens": 1500, "query_heads": 32, "heads": 8,
         "width": 128, "rotary": 128, "pairs": "halves", "page_tokens": 32, "block_tokens": 1, "order": "heads",
         "f16": True},
        # one conversation taken out of the cache
        {"name": "read_b1_l500", "op": "read", "sequences": 1, "heads": 32, "width": 128, "page_tokens": 16,
         "block_tokens": 16, "longest": 500, "order": "heads", "f16": True},
        # long prefixes of many conversations
        {"name": "read_b16_l4096", "op": "read", "sequences": 16, "heads": 8, "width": 128, "page_tokens": 64,
         "block_tokens": 32, "longest": 4096, "order": "tokens", "f16": False},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "append", "read"])
    heads = rng.choice([1, 2, 4, 5, 8, 8, 32])
    width = rng.choice([64, 80, 96, 128, 128, 128, 256])
    page_tokens = rng.choice([1, 16, 16, 20, 24, 32, 64, 128])
    blocks = [b for b in (1, 2, 4, 8, 16, 32, 64) if page_tokens % b == 0]
    case = {"op": op, "sequences": _log(rng, 1, 200 if op == "attention" else 64), "heads": heads, "width": width,
            "page_tokens": page_tokens, "block_tokens": rng.choice([blocks[-1], rng.choice(blocks)]),
            "order": rng.choice(["heads", "heads", "tokens"]), "f16": rng.random() < 0.4}
    token = heads * width * 2                       # bytes of one token in the cache, keys and values
    if op == "append":
        case["query_heads"] = heads * (1 if heads == 32 else rng.choice([1, 2, 3, 4, 7, 8]))
        case["tokens"] = _log(rng, 1, 2048)
        case["sequences"] = min(case["sequences"], case["tokens"])
        case["rotary"] = rng.choice([width, width, width // 2, 0])
        case["pairs"] = rng.choice(["adjacent", "halves"])
        return case
    most = (1 << 29 if op == "attention" else 1 << 27) // (token * case["sequences"])
    case["longest"] = _log(rng, 1, max(64, min(40000, most)))
    if op == "attention":
        case["query_heads"] = heads * (1 if heads == 32 else rng.choice([1, 2, 3, 4, 7, 8]))
        case["window"] = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
    return case


# --- inputs ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _gauss(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * scale


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


def _power(exponent):
    """2^exponent in F32, from -126 to 127, exactly."""
    return ((exponent + 127) << 23).view(torch.float32)


def _pool(g, case, pages):
    """Codes as a quantiser leaves them (the largest of a block near the type's largest, 448), in bytes, and scales
    [pages, heads, blocks of a page], powers of two within a factor of 16."""
    heads, pt, width = case["heads"], case["page_tokens"], case["width"]
    shape = (pages, heads, pt, width) if case["order"] == "heads" else (pages, pt, heads, width)
    codes = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float16).mul_(100).clamp_(-448, 448)
    scales = _power(_ints(g, -9, -4, pages, heads, pt // case["block_tokens"]))
    return codes.to(torch.float8_e4m3fn).view(torch.uint8), scales


def _cache_inputs(g, case, lengths, row_pages):
    pt = case["page_tokens"]
    need = int(((lengths + pt - 1) // pt).sum())
    pages = need + need // 8 + 1
    table = _rows_of_pages(lengths, pt, torch.randperm(pages, generator=g, device="cuda"), row_pages)
    k, k_scales = _pool(g, case, pages)
    v, v_scales = _pool(g, case, pages)
    return {"k": k, "v": v, "k_scales": k_scales, "v_scales": v_scales, "table": table}


def _places(lengths, first):
    """(sequence, position) of the tokens first[s] .. lengths[s] - 1 of every sequence, in order."""
    each = lengths - first
    total = int(each.sum())
    sequence = torch.repeat_interleave(torch.arange(lengths.numel(), device="cuda"), each, output_size=total)
    at = torch.arange(total, device="cuda") - (torch.cumsum(each, 0) - each)[sequence]
    return sequence, first[sequence] + at


def _attention_inputs(case, seed):
    g, n = _gen(seed), case["sequences"]
    lengths = _lengths(g, n, case["longest"])
    s = _cache_inputs(g, case, lengths, -(-case["longest"] // case["page_tokens"]) + 3)
    q = _gauss(g, n, case["query_heads"], case["width"], scale=0.5)
    return {**s, "lengths": lengths.int(), "q": q.half() if case["f16"] else q}


def _append_inputs(case, seed):
    g, n, t, pt, w = _gen(seed), case["sequences"], case["tokens"], case["page_tokens"], case["width"]
    # tokens in order of their sequences; each sequence has a past of up to 300 tokens
    each = torch.full((n,), t // n, device="cuda", dtype=torch.int64)
    each[: t % n] += 1
    past = _ints(_gen(n * 10007 + t), 0, 300, n).long()          # of the case, so that as many rows come back for any seed
    s = _cache_inputs(g, case, past + each, -(-(300 + t) // pt))
    sequence, position = _places(past + each, past)
    # what the call writes: every block with a new token, up to the sequence's end
    read_sequence, read_position = _places(past + each, past - past % case["block_tokens"])
    qkv = _gauss(g, t, (case["query_heads"] + 2 * case["heads"]) * w, scale=2.0)
    positions, half = 300 + t, case["rotary"] // 2
    angle = None
    if half:
        inverse = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * inverse[None, :]
    return {**s, "sequence": sequence.int(), "position": position.int(), "read_sequence": read_sequence.int(),
            "read_position": read_position.int(), "qkv": qkv.half() if case["f16"] else qkv,
            "cosine": torch.cos(angle).float() if half else None, "sine": torch.sin(angle).float() if half else None}


def _read_inputs(case, seed):
    g = _gen(seed)
    # lengths of the case, so that as many rows come back for any seed
    lengths = _lengths(_gen(case["longest"]), case["sequences"], case["longest"])
    s = _cache_inputs(g, case, lengths, -(-case["longest"] // case["page_tokens"]) + 3)
    sequence, position = _places(lengths, torch.zeros_like(lengths))
    return {**s, "read_sequence": sequence.int(), "read_position": position.int()}


def _inputs(case, seed):
    return {"attention": _attention_inputs, "append": _append_inputs, "read": _read_inputs}[case["op"]](case, seed)


def prepare(case, seed):
    return {**_inputs(case, seed), "case": case}


# --- the plain form ---------------------------------------------------------------------

def _by_head(pool, case):
    """[pages, heads, page_tokens, width] of a pool in either order."""
    return pool if case["order"] == "heads" else pool.transpose(1, 2)


def _values(codes):
    return codes.view(torch.float8_e4m3fn).float()


def _gathered(codes, scales, at, case):
    """The pages `at` [sequences, row] of a pool as values [sequences, heads, tokens, width]."""
    n, heads, pt = at.shape[0], case["heads"], case["page_tokens"]
    values = _values(_by_head(codes, case)[at].contiguous())
    values = values * scales[at].repeat_interleave(case["block_tokens"], 3)[..., None]
    return values.transpose(1, 2).reshape(n, heads, at.shape[1] * pt, case["width"])


def _plain_attention(s, case):
    n, heads, width, pt = case["sequences"], case["heads"], case["width"], case["page_tokens"]
    groups = case["query_heads"] // heads
    pages = -(-case["longest"] // pt)
    at = s["table"][:, :pages].long().clamp(min=0)
    k, v = _gathered(s["k"], s["k_scales"], at, case), _gathered(s["v"], s["v_scales"], at, case)
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


def _place(s, case, sequence, position):
    """(page, token in it, block in it) of tokens."""
    pt = case["page_tokens"]
    page, at = s["table"][sequence.long(), position.long() // pt].long(), position.long() % pt
    return page, at, at // case["block_tokens"]


def _plain_read(s, case):
    page, at, block = _place(s, case, s["read_sequence"], s["read_position"])
    out = {}
    for name in ("k", "v"):
        values = _values(_by_head(s[name], case)[page, :, at]) * s[name + "_scales"][page, :, block][..., None]
        out[name] = values.half() if case["f16"] else values
    return out


def _rounded(x):
    """x in 64 bits, at most 448, to the nearest e4m3 code, in bytes (ties to the even code)."""
    exponent = torch.frexp(x)[1] - 1                # the leading bit's; the type's subnormals begin below -6
    step = _power(exponent.clamp(min=-6) - 3).double()
    return (torch.round(x / step) * step).to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_store(s, case, name, x):
    """New tokens x [tokens, heads, width] into a pool. A block's scale is the least power of two (at least 2^-64) that
    takes its new tokens to the codes' range, or its earlier tokens' scale where that is larger. In 64 bits: a code
    next to a border would be off by a whole step."""
    codes, scales = _by_head(s[name], case), s[name + "_scales"]
    blocks = scales.shape[2]
    page, at, block = _place(s, case, s["sequence"], s["position"])
    flat = page * blocks + block
    top = torch.zeros(scales.shape[0] * blocks, case["heads"], device="cuda", dtype=torch.float64)
    top.scatter_reduce_(0, flat[:, None].expand(-1, case["heads"]), x.abs().amax(2), "amax")
    mantissa, exponent = torch.frexp(top)           # top = mantissa * 2^exponent, mantissa in [0.5, 1)
    least = torch.where(top > 0, exponent - 9 + (mantissa > 0.875).int(), torch.full_like(exponent, -64))
    need = _power(least.clamp(min=-64))
    # the tokens that were in these blocks before: every one that is read back and not new
    old_page, old_at, old_block = _place(s, case, s["read_sequence"], s["read_position"])
    new_first = torch.full((case["sequences"],), 1 << 30, dtype=torch.int32, device="cuda")
    new_first.scatter_reduce_(0, s["sequence"].long(), s["position"], "amin")
    earlier = s["read_position"] < new_first[s["read_sequence"].long()]
    old = _values(codes[old_page, :, old_at])
    before = scales[old_page, :, old_block]
    floor = torch.zeros_like(need)
    floor.scatter_reduce_(0, (old_page * blocks + old_block)[:, None].expand(-1, case["heads"]),
                          torch.where(earlier[:, None], before, torch.zeros_like(before)), "amax")
    scale = torch.maximum(need, floor)
    old = old * (before / scale[old_page * blocks + old_block])[..., None]
    codes[old_page, :, old_at] = torch.where(earlier[:, None, None], _rounded(old.double()), codes[old_page, :, old_at])
    codes[page, :, at] = _rounded(x / scale[flat][..., None])
    scales[page, :, block] = scale[flat]


def _plain_append(s, case):
    t, heads, width = case["tokens"], case["heads"], case["width"]
    x = s["qkv"].double().view(t, case["query_heads"] + 2 * heads, width)
    q, k, v = x[:, :case["query_heads"]], x[:, case["query_heads"]:-heads], x[:, -heads:]
    position = s["position"].long()
    cosine = s["cosine"][position] if s["cosine"] is not None else None
    sine = s["sine"][position] if s["sine"] is not None else None
    _plain_store(s, case, "k", _rotated(k, cosine, sine, case["pairs"]))
    _plain_store(s, case, "v", v)
    q = _rotated(q.float(), cosine, sine, case["pairs"]).to(s["qkv"].dtype)
    return {"q": q, **_plain_read(s, case)}


# --- the library's calls ------------------------------------------------------------------

def _library():
    global _kernel
    import kunlunk200_lib_amd as kl
    if _kernel is None:
        _kernel = kl.Kernel()
    return kl, _kernel


def _cache(kl, s, case):
    pages, pt, heads, width = s["k"].shape[0], case["page_tokens"], case["heads"], case["width"]
    strides = (pt * width, width) if case["order"] == "heads" else (width, heads * width)
    return kl.KVCacheF8Layout(kl.KVCacheLayout(pages, pt, heads, width, heads * pt * width, *strides),
                              case["block_tokens"])


def _pools(s):
    return s["k"].data_ptr(), s["v"].data_ptr(), s["k_scales"].data_ptr(), s["v_scales"].data_ptr()


def _own_attention(s, case):
    kl, kernel = _library()
    q, table = s["q"], s["table"]
    y = torch.empty_like(q)
    row = case["query_heads"] * case["width"]
    call = kl.PagedAttentionLayout(case["sequences"], case["query_heads"], case["longest"], case["window"],
                                   table.shape[1], row, row, case["width"] ** -0.5, case["f16"])
    kl.require(kl.paged_attention_f8(kernel, DEV, y.data_ptr(), q.data_ptr(), *_pools(s), table.data_ptr(),
                                     s["lengths"].data_ptr(), _cache(kl, s, case), call))
    return y


def _own_read(s, case):
    kl, kernel = _library()
    n, heads, width = s["read_sequence"].numel(), case["heads"], case["width"]
    kind = torch.float16 if case["f16"] else torch.float32
    k, v = (torch.empty(n, heads, width, dtype=kind, device="cuda") for _ in range(2))
    call = kl.KVReadLayout(n, case["sequences"], s["table"].shape[1], heads * width, heads * width, case["f16"])
    kl.require(kl.kv_read_f8(kernel, DEV, k.data_ptr(), v.data_ptr(), *_pools(s), s["read_sequence"].data_ptr(),
                             s["read_position"].data_ptr(), None, s["table"].data_ptr(), _cache(kl, s, case), call))
    return {"k": k, "v": v}


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
    kl.require(kl.kv_append_f8(kernel, DEV, *_pools(s), q.data_ptr(), at, at + case["query_heads"] * width * size,
                               at + (row - heads * width) * size, s["sequence"].data_ptr(), s["position"].data_ptr(),
                               None, s["table"].data_ptr(), s["cosine"].data_ptr() if turned else None,
                               s["sine"].data_ptr() if turned else None, _cache(kl, s, case), call))
    return {"q": q, **_own_read(s, case)}


def run(state):
    case = state["case"]
    if own:
        form = {"attention": _own_attention, "append": _own_append, "read": _own_read}
    else:
        form = {"attention": _plain_attention, "append": _plain_append, "read": _plain_read}
    return form[case["op"]](state, case)


# --- what a pass cannot do without ----------------------------------------------------------

def work(case):
    heads, width, block = case["heads"], case["width"], case["block_tokens"]
    token = 2 * heads * width                                               # codes of a token
    scale = 2 * heads * 4 / block                                           # and its part of the scales
    size = 2 if case["f16"] else 4
    if case["op"] == "append":
        t, values = case["tokens"], case["query_heads"] * width
        # a block is half full on average when the first new token comes
        read = t + case["sequences"] * (block - 1) // 2
        stored = t * (2 * values * size + token * size + 4 * case["rotary"] + 12) + int(t * token + t * scale)
        return {"bytes": stored + int(read * (token * (1 + size) + scale + 8)),
                "flops": 3 * t * case["rotary"] * (case["query_heads"] + heads) + 2 * (t + read) * token}
    # about the mean of _lengths()
    n, longest = case["sequences"], case["longest"]
    window = case.get("window") or longest
    short, long = (min(window, part * longest) for part in ((0.13, 0.94) if n > 1 else (1, 1)))
    seen = max(1, int(n * (short + long) / 2))
    if case["op"] == "read":
        return {"bytes": int(seen * (token * (1 + size) + scale + 8)), "flops": seen * token}
    return {"bytes": int(seen * (token + scale)) + 2 * n * case["query_heads"] * width * size +
            4 * -(-seen // case["page_tokens"]) + 4 * n, "flops": 4 * seen * case["query_heads"] * width}


# --- the same in 64 bits --------------------------------------------------------------------

def _exact_rows(s, case, name, sequence, positions):
    """[tokens, heads, width]: value = code * scale, the code's bits taken apart."""
    page = s["table"][sequence].long()[positions // case["page_tokens"]]
    at = positions % case["page_tokens"]
    codes = s[name][page, :, at] if case["order"] == "heads" else s[name][page, at]
    bits = codes.long()
    exponent, mantissa = (bits >> 3) & 15, (bits & 7).double()
    size = torch.where(exponent > 0, (8 + mantissa) * (1 << exponent).double() / 1024, mantissa / 512)
    scale = s[name + "_scales"][page, :, at // case["block_tokens"]].double()
    return torch.where(bits > 127, -size, size) * scale[:, :, None]


def _exact_attention(s, case):
    groups, width = case["query_heads"] // case["heads"], case["width"]
    y = torch.zeros(case["sequences"], case["query_heads"], width, dtype=torch.float64, device="cuda")
    for i, length in enumerate(s["lengths"].tolist()):
        if length == 0:
            continue
        first = max(0, length - case["window"]) if case["window"] else 0
        t = torch.arange(first, length, device="cuda")
        k, v = _exact_rows(s, case, "k", i, t), _exact_rows(s, case, "v", i, t)
        for h in range(case["heads"]):
            q = s["q"][i, h * groups:(h + 1) * groups].double()
            weight = torch.softmax((k[:, h] @ q.T) / width ** 0.5, 0)
            y[i, h * groups:(h + 1) * groups] = weight.T @ v[:, h]
    return y


def _exact_read(s, case):
    sequence, position = s["read_sequence"].long(), s["read_position"].long()
    return {name: torch.cat([_exact_rows(s, case, name, i, position[sequence == i]) for i in sequence.unique().tolist()])
            for name in ("k", "v")}


def _nearest_code(x):
    """The nearest value that e4m3 has, of two equally near ones the one with the even code."""
    exponent = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))).long()
    step = (1 << (exponent + 6)).double() / 512
    return torch.round(x / step) * step


def _exact_append(s, case):
    heads, width, half, block = case["heads"], case["width"], case["rotary"] // 2, case["block_tokens"]
    x = s["qkv"].double().view(case["tokens"], -1, width)
    sequence, position = s["sequence"].long(), s["position"].long()
    if half:
        turn = torch.complex(s["cosine"][position].double(), s["sine"][position].double())[:, None, :]
        part = x[:, :-heads, :2 * half]
        if case["pairs"] == "adjacent":
            z = torch.complex(part[..., 0::2].contiguous(), part[..., 1::2].contiguous()) * turn
            x[:, :-heads, 0:2 * half:2], x[:, :-heads, 1:2 * half:2] = z.real, z.imag
        else:
            z = torch.complex(part[..., :half].contiguous(), part[..., half:].contiguous()) * turn
            x[:, :-heads, :half], x[:, :-heads, half:2 * half] = z.real, z.imag
    out = {"q": x[:, :case["query_heads"]].contiguous()}
    for name, new in (("k", x[:, -2 * heads:-heads]), ("v", x[:, -heads:])):
        rows = []
        for i in range(case["sequences"]):
            mine = new[sequence == i]
            end = int(position[sequence == i][-1]) + 1
            past = end - mine.shape[0]
            start = past - past % block
            old = _exact_rows(s, case, name, i, torch.arange(start, past, device="cuda"))
            for b in range(start, end, block):
                fresh = mine[max(b, past) - past:b + block - past]
                exponent = torch.ceil(torch.log2(fresh.abs().amax((0, 2)) / 448)).clamp(min=-64)
                scale = torch.tensor([2.0 ** e for e in exponent.tolist()], dtype=torch.float64, device="cuda")
                kept = fresh[:0]
                if b < past:
                    page, at = int(s["table"][i, b // case["page_tokens"]]), b % case["page_tokens"]
                    scale = torch.maximum(scale, s[name + "_scales"][page, :, at // block].double())
                    kept = old
                whole = torch.cat([kept, fresh]) / scale[None, :, None]
                rows.append(_nearest_code(whole) * scale[None, :, None])
        out[name] = torch.cat(rows)
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "read": _exact_read}[case["op"]](s, case)
