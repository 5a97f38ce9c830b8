"""Argument rules of the 8-bit cache: the layouts' reasons on any host, and on the GPU that every broken rule makes a call
return False with nothing written, where the same call unbroken succeeds."""
import ctypes

import numpy as np
import pytest

import kunlunk200_lib_amd as kl
from kv_f8 import SIZES, VALUES, encode, least_scale
from test_kv_cache_rules import (APPEND_BREAKS, ATTENTION_BREAKS, LIST_BREAKS, POOL_BREAKS, TABLE_BREAKS, Memory, append,
                                 attend, broken, cache, pages)

F32, F16 = kl.InputType.f32, kl.InputType.f16
READ = dict(tokens=3, sequences=2, row_pages=3, k_stride=128, v_stride=128, type=F32)


def f8(block=8, **k):
    return kl.KVCacheF8Layout(cache(**k), block)


def read(**k):
    return kl.KVReadLayout(**{**READ, **k})


def test_codes():
    """The model's codes against the type's definition: every code is its own nearest, ties go to the even one."""
    finite = np.array([c for c in range(256) if c % 128 != 127], np.uint8)
    assert np.array_equal(encode(VALUES[finite]), finite) and SIZES[-1] == 448 and SIZES[1] == 2.0 ** -9 and SIZES[8] == 2.0 ** -6
    middle = (SIZES[:-1] + SIZES[1:]) / 2
    assert np.all(encode(middle) % 2 == 0) and np.all(encode(np.nextafter(middle, 0)) == np.arange(126))
    assert np.all(encode(np.nextafter(middle, 500)) == np.arange(1, 127)) and encode(np.nan) == 127
    top = np.array([448.0, np.nextafter(448.0, 500), 224.0, 1.0, 0.0, 1e-30])
    assert np.array_equal(least_scale(top), [1, 2, 0.5, 2.0 ** -8, 2.0 ** -64, 2.0 ** -64])


def test_cache_reasons(kl):
    r = lambda block=8, **k: kl.kv_cache_f8_reason(f8(block, **k))  # noqa: E731
    for block in (1, 2, 4, 8, 16):
        assert r(block) == ""
    assert r(64, page_tokens=64, page_stride=8192, head_stride=4096) == ""
    assert r(0) == r(-8) == r(3) == r(32) == r(12) == "block"
    assert r(8, page_tokens=20, page_stride=2560, head_stride=1280) == "block"
    assert r(4, page_tokens=20, page_stride=2560, head_stride=1280) == ""
    assert r(128, page_tokens=128, page_stride=1 << 14, head_stride=1 << 13) == "block"
    assert r(width=60) == "shape" and r(token_stride=56) == "stride" and r(pages=0, block=3) == "shape"


def test_call_reasons(kl):
    assert kl.paged_attention_f8_reason(f8(), attend()) == kl.kv_append_f8_reason(f8(), append()) == ""
    assert kl.kv_read_f8_reason(f8(), read()) == kl.kv_pages_f8_reason(f8(), pages()) == ""
    for reason, call in ((kl.paged_attention_f8_reason, attend()), (kl.kv_append_f8_reason, append()),
                         (kl.kv_read_f8_reason, read()), (kl.kv_pages_f8_reason, pages())):
        assert reason(f8(3), call) == "block" and reason(f8(width=60), call) == "shape"
    assert kl.paged_attention_f8_reason(f8(), attend(type=2)) == "type"
    assert kl.paged_attention_f8_reason(f8(), attend(longest=49)) == "length"
    assert kl.paged_attention_f8_reason(f8(), attend(scale=3e38)) == "scale"
    assert kl.kv_append_f8_reason(f8(), append(rotary=3)) == "rotary"
    # (4 * 8 + 512 * 2) * tokens below 2^31 - 1024
    assert kl.kv_append_f8_reason(f8(), append(tokens=2033600)) == ""
    assert kl.kv_append_f8_reason(f8(), append(tokens=2033601)) == "shape"
    r = lambda **k: kl.kv_read_f8_reason(f8(), read(**k))  # noqa: E731
    assert r(type=F16) == "" and r(type=2) == r(type=-1) == "type"
    assert r(tokens=0) == r(sequences=0) == r(row_pages=-1) == r(tokens=1 << 27) == "shape" and r(tokens=(1 << 26) - 64) == ""
    assert r(row_pages=1 << 24) == "length" and r(k_stride=127) == r(v_stride=-128) == r(v_stride=(1 << 40) + 1) == "stride"
    assert kl.kv_pages_f8_reason(f8(), pages(layers=2, layer_stride=8196)) == "stride"


def test_null_handles_and_layouts(kl):
    lib = kl.load()
    c, a = ctypes.byref(f8()), ctypes.byref(attend())
    kernel = kl.Kernel()
    for handle, layout, call in ((None, c, a), (kernel.handle, None, a), (kernel.handle, c, None)):
        assert lib.kunlun_paged_attention_f8(handle, 0, *[4096] * 8, layout, call) == 0
        assert lib.kunlun_kv_append_f8(handle, 0, *[4096] * 14, layout, call) == 0
        assert lib.kunlun_kv_read_f8(handle, 0, *[4096] * 10, layout, call) == 0
        assert lib.kunlun_kv_fork_f8(handle, 0, *[4096] * 9, 1, layout, call) == 0
        assert lib.kunlun_kv_compact_f8(handle, 0, *[4096] * 10, layout, call) == 0
        assert lib.kunlun_kv_copy_pages_f8(handle, 0, *[4096] * 6, 1, layout, call) == 0
    for f in ("paged_attention", "kv_append", "kv_read", "kv_pages"):
        assert getattr(lib, f"kunlun_{f}_f8_reason")(None, None) == b"shape"
    assert lib.kunlun_kv_cache_f8_reason(None) == b"shape"


# --- calls, with real memory ------------------------------------------------------------

def pools_of(m):
    """4 pages of 2 heads x 16 tokens x 64 codes, a scale for every 8 tokens."""
    return dict(k=m.part(8192), v=m.part(8192), k_scales=m.part(64), v_scales=m.part(64))


def attention_call():
    m = Memory()
    p = dict(y=m.part(2048), q=m.part(2048), **pools_of(m), table=m.part(24), lengths=m.part(8))
    return m, dict(p, device=0, cache=f8(), call=attend()), lambda kernel, a: kl.paged_attention_f8(
        kernel, a["device"], a["y"], a["q"], a["k"], a["v"], a["k_scales"], a["v_scales"], a["table"], a["lengths"],
        a["cache"], a["call"])


def append_call():
    m = Memory()
    rows = m.part(3 * 2048)
    pools = pools_of(m)
    p = dict(k_pool=pools["k"], v_pool=pools["v"], k_scales=pools["k_scales"], v_scales=pools["v_scales"],
             q_out=m.part(3 * 1024), q=rows, k=rows + 1024, v=rows + 1536, sequence=m.part(12), position=m.part(12),
             lengths=m.part(8), table=m.part(24), cosine=m.part(48 * 128), sine=m.part(48 * 128))
    return m, dict(p, device=0, cache=f8(), call=append()), lambda kernel, a: kl.kv_append_f8(
        kernel, a["device"], a["k_pool"], a["v_pool"], a["k_scales"], a["v_scales"], a["q_out"], a["q"], a["k"], a["v"],
        a["sequence"], a["position"], a["lengths"], a["table"], a["cosine"], a["sine"], a["cache"], a["call"])


def read_call():
    m = Memory()
    p = dict(k_out=m.part(1536), v_out=m.part(1536), **pools_of(m), sequence=m.part(12), position=m.part(12),
             lengths=m.part(8), table=m.part(24))
    return m, dict(p, device=0, cache=f8(), call=read()), lambda kernel, a: kl.kv_read_f8(
        kernel, a["device"], a["k_out"], a["v_out"], a["k"], a["v"], a["k_scales"], a["v_scales"], a["sequence"],
        a["position"], a["lengths"], a["table"], a["cache"], a["call"])


def pages_call(name):
    def make():
        m = Memory()
        p = dict(**pools_of(m), table=m.part(24), lengths=m.part(8), references=m.part(16), first=m.part(8),
                 second=m.part(8), table_out=m.part(24), references_out=m.part(16), used=m.part(4))
        a = dict(p, device=0, count=2, cache=f8(), pages=pages())

        def call(kernel, a):
            pools = (a["k"], a["v"], a["k_scales"], a["v_scales"])
            tables = (a["table"], a["lengths"], a["references"])
            if name == "kv_fork_f8":
                return kl.kv_fork_f8(kernel, a["device"], *pools, *tables, a["first"], a["second"], a["count"], a["cache"],
                                     a["pages"])
            if name == "kv_compact_f8":
                return kl.kv_compact_f8(kernel, a["device"], *pools, a["table_out"], a["references_out"], a["used"],
                                        *tables, a["cache"], a["pages"])
            return kl.kv_copy_pages_f8(kernel, a["device"], *pools, a["first"], a["second"], a["count"], a["cache"],
                                       a["pages"])
        return m, a, call
    return make


def in_f8(breaks):
    """The F16 cache's broken calls with its layouts as 8-bit ones."""
    return [{k: kl.KVCacheF8Layout(v, 8) if isinstance(v, kl.KVCacheLayout) else v for k, v in b.items()} for b in breaks]


SCALE_BREAKS = [dict(k_scales=None), dict(v_scales=None), dict(k_scales="+2"), dict(v_scales="+1"), dict(cache=f8(3)),
                dict(cache=f8(32))]
POOLS_APART = [dict(k_scales="v_scales+60"), dict(k_scales="k"), dict(v_scales="v+8188"), dict(k="v+16")]
CALLS = {
    "paged_attention_f8": (attention_call, in_f8(ATTENTION_BREAKS) + SCALE_BREAKS +
                           [dict(y="k_scales"), dict(y="v_scales-2044")]),
    "kv_append_f8": (append_call, in_f8(APPEND_BREAKS) + SCALE_BREAKS +
                     [dict(k_scales="v_scales+60"), dict(k_scales="k_pool"), dict(v_scales="q"), dict(k_scales="q_out+12"),
                      dict(v_scales="table-60"), dict(k_scales="cosine"), dict(k_scales="position")]),
    "kv_read_f8": (read_call, SCALE_BREAKS + [
        dict(device=-1), dict(device=8), dict(k_out=None), dict(v_out=None), dict(k=None), dict(v=None), dict(table=None),
        dict(sequence=None), dict(position=None), dict(position=None, sequence=None),
        dict(position=None, sequence=None, lengths=None), dict(k_out="+2"), dict(v_out="+1"), dict(k="+8"), dict(table="+2"),
        dict(sequence="+2"), dict(k_out="v_out"), dict(k_out="v_out+4"), dict(k_out="k"), dict(v_out="k_scales-1532"),
        dict(k_out="table"), dict(v_out="position-1532"), dict(v_out="sequence"),
        dict(v_out="k_out+256", call=read(k_stride=191, v_stride=191)),
        dict(v_out="k_out+508", call=read(k_stride=256, v_stride=256)),
        dict(v_out="k_out+512", call=read(k_stride=256, v_stride=257)), dict(call=read(tokens=0)),
        dict(call=read(k_stride=127)), dict(cache=f8(width=60))]),
    "kv_fork_f8": (pages_call("kv_fork_f8"), in_f8(TABLE_BREAKS + LIST_BREAKS + POOL_BREAKS) + SCALE_BREAKS + POOLS_APART +
                   [dict(second=None), dict(k="table-64"), dict(second="k+64"), dict(k_scales="table"), dict(v_scales="first")]),
    "kv_compact_f8": (pages_call("kv_compact_f8"), in_f8(TABLE_BREAKS + POOL_BREAKS) + SCALE_BREAKS + POOLS_APART +
                      [dict(table_out=None), dict(references_out=None), dict(used=None), dict(used="table"),
                       dict(table_out="table+4"), dict(references_out="references-4"), dict(table_out="references"),
                       dict(references_out="lengths"), dict(used="k"), dict(table_out="v+128"), dict(used="k_scales+4"),
                       dict(references_out="v_scales")]),
    "kv_copy_pages_f8": (pages_call("kv_copy_pages_f8"), [dict(first=None), dict(second=None), dict(count=0), dict(count=5),
                                                          dict(first="+2"), dict(second="v"), dict(second="k_scales")] +
                         in_f8(POOL_BREAKS) + SCALE_BREAKS + POOLS_APART),
}


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
    # the unbroken call is accepted (empty sequences, lists of sequence 0)
    if name in ("kv_fork_f8", "kv_copy_pages_f8"):
        args["count"] = 1
    assert call(kernel, args) is True
    assert kernel.route.startswith(name)
    assert gpu.kv_cache_status(0) == 0
