"""Sizes at the ends of 32-bit counting: what the page operations' loops could not count is refused, by name."""


def test_pages_and_sequences_that_loops_can_count(kl):
    def reason(pages, sequences):
        cache = kl.KVCacheLayout(pages, 1, 1, 8, 8, 8, 8)
        assert kl.kv_cache_reason(cache) == ""
        return kl.kv_pages_reason(cache, kl.KVPagesLayout(sequences, 1, 1, 0))
    assert reason(1 << 30, 1 << 30) == "" and reason(1, 1) == ""
    # steps of up to 2^21 pages past the last one stay below 2^31
    assert reason((1 << 30) + 1, 1) == reason(2 ** 31 - 1, 1) == "shape"
    assert reason(1, (1 << 30) + 1) == reason(1, 2 ** 31 - 1) == "shape"
