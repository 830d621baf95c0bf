"""CPU: a paged cache's memory goes with the last reference to it, not with the collector's next pass."""
import gc
import weakref

import pytest

from tests.test_paged import _config


@pytest.mark.parametrize("form", ["bf16", "fp4"])
def test_a_cache_that_is_dropped_frees_its_pages(form):
    from pbs_attn_amd.patch.paged_cache import PagedKVCache
    gc.collect()
    gc.disable()
    try:
        cache = PagedKVCache(_config(), 2, 100, form=form, device="cpu")
        cache.lengths(5)
        held = [weakref.ref(x) for x in (cache, cache.page_table, cache.lengths(5), cache.layers[0].pages.k, cache.layers[2].pages.v)]
        del cache
        assert [x() for x in held] == [None] * 5
    finally:
        gc.enable()


def test_a_layer_by_itself_keeps_working():
    from pbs_attn_amd.patch.paged_cache import PagedKVCache
    layer = PagedKVCache(_config(), 2, 100, device="cpu").layers[1]
    with pytest.raises(ValueError, match="the cache holds 100"):
        layer.append(*[layer.pages.k.new_zeros(2, 2, 101, 128)] * 2)
