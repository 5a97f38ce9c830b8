"""Argument rules of the paged cache and logits operators: the layouts' reasons on any host, and on the GPU
that every broken rule makes a call return False with nothing written, where the same call unbroken succeeds."""
import ctypes

import numpy as np
import pytest

import kunlunk200_lib_amd as kl

F32, F16 = kl.InputType.f32, kl.InputType.f16
HEADS = dict(pages=4, page_tokens=16, heads=2, width=64, page_stride=2048, head_stride=1024, token_stride=64)
ATTEND = dict(sequences=2, query_heads=4, longest=40, window=0, row_pages=3, q_stride=256, y_stride=256, scale=0.125,
              type=F32)
APPEND = dict(tokens=3, sequences=2, row_pages=3, query_heads=4, q_stride=512, k_stride=512, v_stride=512,
              q_out_stride=256, rotary=64, positions=48, pairs=kl.RotaryPairs.halves, type=F32)
PAGES = dict(sequences=2, row_pages=3, layers=1, layer_stride=8192)
LOGITS = dict(rows=2, vocabulary=100, logits_stride=100, y_stride=100, history_stride=8, bias_stride=4, mask_stride=4)


def cache(**k):
    return kl.KVCacheLayout(**{**HEADS, **k})


def attend(**k):
    return kl.PagedAttentionLayout(**{**ATTEND, **k})


def append(**k):
    return kl.KVAppendLayout(**{**APPEND, **k})


def pages(**k):
    return kl.KVPagesLayout(**{**PAGES, **k})


def logits(**k):
    return kl.LogitsLayout(**{**LOGITS, **k})


CACHE_RULES = [
    (dict(), ""),
    (dict(page_stride=2048, head_stride=64, token_stride=128), ""),          # a token's heads together
    (dict(page_stride=4096, head_stride=1536, token_stride=72), ""),         # padding
    (dict(pages=0), "shape"), (dict(pages=-1), "shape"), (dict(page_tokens=0), "shape"),
    (dict(page_tokens=65537, page_stride=1 << 30, head_stride=1 << 28), "shape"),
    (dict(heads=0), "shape"), (dict(heads=1025, page_stride=1 << 30), "shape"),
    (dict(width=60), "shape"), (dict(width=264, token_stride=264), "shape"), (dict(width=0), "shape"),
    (dict(token_stride=56), "stride"), (dict(token_stride=68), "stride"), (dict(page_stride=2044), "stride"),
    (dict(head_stride=960), "stride"),                                       # heads overlap
    (dict(page_stride=1984), "stride"),                                      # pages overlap
    (dict(head_stride=64, token_stride=64), "stride"),                       # both orders at once
    (dict(page_stride=(1 << 40) + 8), "stride"), (dict(page_stride=-2048), "stride"),
    (dict(pages=2 ** 31 - 1, page_stride=1 << 40), "byte extent"),
]


@pytest.mark.parametrize("change,reason", CACHE_RULES)
def test_cache_reasons(kl, change, reason):
    assert kl.kv_cache_reason(cache(**change)) == reason


def test_attention_reasons(kl):
    r = lambda c={}, **k: kl.paged_attention_reason(cache(**c), attend(**k))  # noqa: E731
    assert r() == "" and r(type=F16) == "" and r(window=7) == "" and r(scale=-2.0) == ""
    assert r({"width": 60}) == "shape"
    assert r(type=2) == "type" and r(type=-1) == "type"
    assert r(sequences=0) == r(sequences=65536) == r(row_pages=0) == r(window=-1) == "shape"
    assert r(query_heads=0) == r(query_heads=3) == r(query_heads=1026) == r(query_heads=-2) == "heads"
    assert r(longest=0) == r(longest=49) == r(longest=-1) == "length" and r(longest=48) == ""
    assert r(longest=1 << 27, row_pages=1 << 24) == "length"
    assert r(scale=float("nan")) == r(scale=float("inf")) == "scale"
    assert r(q_stride=255) == r(y_stride=255) == r(y_stride=-256) == r(q_stride=(1 << 40) + 1) == "stride"


def test_append_reasons(kl):
    r = lambda c={}, **k: kl.kv_append_reason(cache(**c), append(**k))  # noqa: E731
    assert r() == "" and r(rotary=0, positions=0) == "" and r(rotary=2) == "" and r(query_heads=0, q_stride=0) == ""
    assert r({"heads": 0}) == "shape"
    assert r(type=3) == r(pairs=2) == r(pairs=-1) == "type"
    assert r(tokens=0) == r(sequences=0) == r(row_pages=-1) == r(tokens=1 << 28) == "shape"
    assert r(row_pages=1 << 24) == "length" and r(query_heads=-1) == r(query_heads=1025) == "heads"
    assert r(rotary=3) == r(rotary=66) == r(rotary=-2) == r(positions=0) == "rotary"
    assert r(k_stride=127) == r(v_stride=127) == r(q_stride=255) == r(q_out_stride=255) == "stride"


def test_pages_and_logits_reasons(kl):
    r = lambda c={}, **k: kl.kv_pages_reason(cache(**c), pages(**k))  # noqa: E731
    assert r() == "" and r(layers=1, layer_stride=0) == "" and r(layers=5) == ""
    assert r({"page_tokens": 0}) == r(sequences=0) == r(row_pages=0) == r(layers=0) == r(layers=65536) == "shape"
    assert r(row_pages=1 << 24) == "length"
    assert r(layers=2, layer_stride=8184) == r(layers=2, layer_stride=8196) == r(layers=2, layer_stride=-8192) == "stride"
    z = lambda **k: kl.logits_reason(logits(**k))  # noqa: E731
    assert z() == "" and z(mask_stride=0) == "" and z(history_stride=0, bias_stride=0) == ""
    assert z(rows=0) == z(rows=65536) == z(vocabulary=0) == z(vocabulary=(1 << 24) + 1, logits_stride=1 << 25) == "shape"
    assert z(logits_stride=99) == z(y_stride=99) == z(history_stride=-1) == z(bias_stride=-1) == z(mask_stride=3) == "stride"


def test_null_handles_and_layouts(kl):
    """The C entries refuse null handles and layouts; nothing is called."""
    lib = kl.load()
    c, a = ctypes.byref(cache()), ctypes.byref(attend())
    assert lib.kunlun_paged_attention(None, 0, 1, 1, 1, 1, 1, 1, c, a) == 0
    kernel = kl.Kernel()
    assert lib.kunlun_paged_attention(kernel.handle, 0, 4096, 8192, 1 << 20, 2 << 20, 4096, 4096, None, a) == 0
    assert lib.kunlun_paged_attention(kernel.handle, 0, 4096, 8192, 1 << 20, 2 << 20, 4096, 4096, c, None) == 0
    assert lib.kunlun_process_logits(kernel.handle, 0, 4096, 8192, *[None] * 7, None) == 0
    assert lib.kunlun_kv_free(None, 0, 1, 1, 1, 1, 1, c, ctypes.byref(pages())) == 0
    for f in ("paged_attention", "kv_append", "kv_pages"):
        assert getattr(lib, f"kunlun_{f}_reason")(None, None) == b"shape"
    assert lib.kunlun_kv_cache_reason(None) == b"shape" == lib.kunlun_logits_reason(None)
    assert kl.kv_cache_status(-1) == -1 and kl.kv_cache_status(kl_max_devices()) == -1


def kl_max_devices():
    return 8


# --- calls, with real memory ------------------------------------------------------------

class Memory:
    """One allocation cut into parts, each filled with zeros."""

    def __init__(self):
        self.buffer = kl.Buffer(0, 1 << 20)
        self.buffer.upload(np.zeros(1 << 20, np.uint8))
        self.at = self.buffer.data

    def part(self, size):
        start = self.at
        self.at += (size + 255) // 256 * 256
        assert self.at <= self.buffer.data + self.buffer.size
        return start

    def check_zero(self):
        with kl.runtime_mutex():
            kl.select(0)
            kl.check(kl.wait())
        assert not self.buffer.download(1 << 20, np.uint8).any(), "a refused call wrote"


def attention_call():
    m = Memory()
    p = dict(y=m.part(2048), q=m.part(2048), k=m.part(16384), v=m.part(16384), table=m.part(24), lengths=m.part(8))
    return m, dict(p, device=0, cache=cache(), call=attend()), lambda kernel, a: kl.paged_attention(
        kernel, a["device"], a["y"], a["q"], a["k"], a["v"], a["table"], a["lengths"], a["cache"], a["call"])


ATTENTION_BREAKS = [
    dict(device=-1), dict(device=8), dict(y=None), dict(q=None), dict(k=None), dict(v=None), dict(table=None),
    dict(lengths=None), dict(y="+2"), dict(q="+1"), dict(k="+8"), dict(v="+2"), dict(table="+2"), dict(lengths="+1"),
    dict(y="q+4"), dict(y="q"), dict(y="k+16"), dict(y="v-1024"), dict(y="table-2044"), dict(y="lengths"),
    dict(cache=cache(width=60)), dict(call=attend(query_heads=3)), dict(call=attend(longest=49)),
]


def append_call():
    m = Memory()
    rows = m.part(3 * 2048)
    p = dict(k_pool=m.part(16384), v_pool=m.part(16384), q_out=m.part(3 * 1024), q=rows, k=rows + 1024, v=rows + 1536,
             sequence=m.part(12), position=m.part(12), lengths=m.part(8), table=m.part(24), cosine=m.part(48 * 128),
             sine=m.part(48 * 128))
    return m, dict(p, device=0, cache=cache(), call=append()), lambda kernel, a: kl.kv_append(
        kernel, a["device"], a["k_pool"], a["v_pool"], a["q_out"], a["q"], a["k"], a["v"], a["sequence"], a["position"],
        a["lengths"], a["table"], a["cosine"], a["sine"], a["cache"], a["call"])


APPEND_BREAKS = [
    dict(device=-3), dict(k_pool=None), dict(v_pool=None), dict(k=None), dict(v=None), dict(table=None),
    dict(q=None), dict(q_out=None), dict(cosine=None), dict(sine=None), dict(sequence=None),
    dict(position=None), dict(position=None, sequence=None, lengths=None),
    dict(position=None, sequence=None),                    # three newest tokens of two sequences
    dict(k_pool="+8"), dict(q="+2"), dict(k="+1"), dict(sequence="+2"), dict(cosine="+2"),
    dict(k_pool="v_pool+16"), dict(k_pool="q"), dict(v_pool="table-16"), dict(q_out="k_pool"), dict(q_out="q+4"),
    dict(q_out="k-512"), dict(q_out="cosine"), dict(q_out="position-4"),
    dict(call=append(q_out_stride=512), q_out="v-512"),    # rows like the inputs', over the keys
    dict(call=append(rotary=3)), dict(call=append(query_heads=0)),
]


def pages_call(name):
    def make():
        m = Memory()
        p = dict(k=m.part(16384), v=m.part(16384), table=m.part(24), lengths=m.part(8), references=m.part(16),
                 first=m.part(8), second=m.part(8), table_out=m.part(24), references_out=m.part(16), used=m.part(4))
        a = dict(p, device=0, count=2, cache=cache(), pages=pages())

        def call(kernel, a):
            tables = (a["table"], a["lengths"], a["references"])
            if name == "kv_reserve":
                return kl.kv_reserve(kernel, a["device"], *tables, a["first"], a["second"], a["count"], a["cache"], a["pages"])
            if name == "kv_fork":
                return kl.kv_fork(kernel, a["device"], a["k"], a["v"], *tables, a["first"], a["second"], a["count"],
                                  a["cache"], a["pages"])
            if name == "kv_free":
                return kl.kv_free(kernel, a["device"], *tables, a["first"], a["count"], a["cache"], a["pages"])
            if name == "kv_compact":
                return kl.kv_compact(kernel, a["device"], a["k"], a["v"], a["table_out"], a["references_out"], a["used"],
                                     *tables, a["cache"], a["pages"])
            return kl.kv_copy_pages(kernel, a["device"], a["k"], a["v"], a["first"], a["second"], a["count"], a["cache"],
                                    a["pages"])
        return m, a, call
    return make


TABLE_BREAKS = [dict(device=-1), dict(table=None), dict(lengths=None), dict(references=None), dict(table="+2"),
                dict(lengths="table+20"), dict(references="lengths"), dict(pages=pages(sequences=0)),
                dict(cache=cache(pages=0))]
LIST_BREAKS = [dict(first=None), dict(count=0), dict(count=-1), dict(count=3), dict(first="+1"), dict(first="table")]
POOL_BREAKS = [dict(k=None), dict(v=None), dict(k="+8"), dict(v="k+16"), dict(v="k"),
               dict(pages=pages(layers=2, layer_stride=8196))]


def logits_call():
    m = Memory()
    p = dict(y=m.part(800), logits=m.part(800), penalties=m.part(24), history=m.part(64), history_lengths=m.part(8),
             bias_ids=m.part(32), bias_values=m.part(32), bias_lengths=m.part(8), mask=m.part(32))
    return m, dict(p, device=0, call=logits()), lambda kernel, a: kl.process_logits(
        kernel, a["device"], a["y"], a["logits"], a["penalties"], a["history"], a["history_lengths"], a["bias_ids"],
        a["bias_values"], a["bias_lengths"], a["mask"], a["call"])


LOGITS_BREAKS = [
    dict(device=99), dict(y=None), dict(logits=None), dict(penalties=None), dict(history_lengths=None),
    dict(bias_values=None), dict(bias_lengths=None), dict(y="+2"), dict(logits="+1"), dict(mask="+2"), dict(y="logits+4"),
    dict(y="mask-4"), dict(y="history"), dict(y="penalties-796"), dict(y="bias_values"), dict(y="bias_lengths"),
    dict(y="logits", call=logits(y_stride=101)), dict(call=logits(vocabulary=101)),
]

CALLS = {
    "paged_attention": (attention_call, ATTENTION_BREAKS),
    "kv_append": (append_call, APPEND_BREAKS),
    "kv_reserve": (pages_call("kv_reserve"), TABLE_BREAKS + LIST_BREAKS + [dict(second=None), dict(second="references")]),
    "kv_fork": (pages_call("kv_fork"), TABLE_BREAKS + LIST_BREAKS + POOL_BREAKS +
                [dict(second=None), dict(k="table-64"), dict(second="k+64")]),
    "kv_free": (pages_call("kv_free"), TABLE_BREAKS + LIST_BREAKS),
    "kv_compact": (pages_call("kv_compact"), TABLE_BREAKS + POOL_BREAKS +
                   [dict(table_out=None), dict(references_out=None), dict(used=None), dict(used="table"),
                    dict(table_out="table+4"), dict(references_out="references-4"), dict(table_out="references"),
                    dict(references_out="lengths"), dict(used="k"), dict(table_out="v+128")]),
    "kv_copy_pages": (pages_call("kv_copy_pages"), [dict(first=None), dict(second=None), dict(count=0), dict(count=5),
                                                    dict(first="+2"), dict(second="v")] + POOL_BREAKS),
    "process_logits": (logits_call, LOGITS_BREAKS),
}


def broken(args, change):
    """A changed pointer: None, "+n" (its own moved), "name", "name+n" or "name-n" (another one's)."""
    out = dict(args)
    for name, to in change.items():
        if isinstance(to, str):
            base = to.split("+")[0].split("-")[0]
            to = (args[base] if base else args[name]) + (int(to[len(base):]) if to[len(base):] else 0)
        out[name] = to
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(CALLS))
def test_refusals(gpu, name):
    make, breaks = CALLS[name]
    memory, args, call = make()
    kernel = kl.Kernel()
    for change in breaks:
        print(name, {k: v if isinstance(v, (str, int, type(None))) else "layout" for k, v in change.items()}, flush=True)
        assert call(kernel, broken(args, change)) is False, change
    assert kernel.route is None
    memory.check_zero()
    assert gpu.kv_cache_status(0) == 0
    # the unbroken call is accepted (empty sequences, lists of sequence 0, no history)
    if name in ("kv_fork", "kv_reserve", "kv_free", "kv_copy_pages"):
        args["count"] = 1
    assert call(kernel, args) is True
    assert kernel.route.startswith(name)
    assert gpu.kv_cache_status(0) == 0
