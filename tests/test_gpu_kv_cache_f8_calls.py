"""The 8-bit key-value cache: the longest lists, scales that something else has made, tokens in any order, and kernels that
ordinary sizes do not reach; against plain computations in 64 bits."""
import numpy as np
import pytest

import kunlunk200_lib_amd as kl
from kv_f8 import CacheF8, finish, upload

pytestmark = pytest.mark.gpu


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
