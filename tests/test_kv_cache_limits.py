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


def test_scale_that_has_no_base_2(kl):
    """Scores are kept in base 2: a scale whose product with log2(e) is not finite is refused like an infinite one."""
    cache = kl.KVCacheLayout(4, 16, 2, 64, 2048, 1024, 64)

    def reason(scale):
        call = kl.PagedAttentionLayout(2, 4, 40, 0, 3, 256, 256, scale, kl.InputType.f32)
        return kl.paged_attention_reason(cache, call)
    assert reason(2.3e38) == reason(-2.3e38) == reason(1e-45) == ""
    assert reason(2.4e38) == reason(-3.4e38) == "scale"
