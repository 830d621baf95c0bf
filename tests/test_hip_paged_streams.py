"""GPU: a paged cache of a model that is used on one stream after another."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_lengths_belong_to_the_stream_that_filled_them(dev):
    from pbs_attn_amd.patch.paged_cache import PagedKVCache
    from tests.test_paged import _config
    cache = PagedKVCache(_config(), 2, 100, device=dev)
    side = torch.cuda.Stream()
    here = cache.lengths(3)
    with torch.cuda.stream(side):
        there = cache.lengths(3)
        assert cache.lengths(3) is there
    assert here.data_ptr() != there.data_ptr() and cache.lengths(3) is here
    torch.cuda.synchronize()
    assert here.tolist() == there.tolist() == [3, 3]


def test_steps_on_alternating_streams(dev):
    from pbs_attn_amd.patch.paged_cache import PagedKVCache
    from tests.test_paged import _config
    g = torch.Generator(device="cuda").manual_seed(0)
    steps = [[torch.randn(2, heads, S, 128, generator=g, device=dev).to(torch.bfloat16) for heads in (2, 2, 4)] for S in (50, 1, 1, 7, 1, 1)]

    def run(streams):
        cache, out = PagedKVCache(_config(num_hidden_layers=1), 2, 100, device=dev), []
        for i, (k, v, q) in enumerate(steps):
            stream = streams[i % len(streams)]
            stream.wait_stream(streams[i % len(streams) - 1])
            with torch.cuda.stream(stream):
                cache.layers[0].append(k, v)
                out.append(cache.layers[0].attention(q))
        torch.cuda.synchronize()
        return out
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    assert all(torch.equal(a, b) for a, b in zip(run([one]), run([one, two])))
