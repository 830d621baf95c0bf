"""CPU: taking tokens off a paged cache's end, as assisted decoding does, and what it refuses."""
import pytest
import torch

from tests import paged_cpu


def _ids(S, seed=0):
    return torch.randint(1, 101, (1, S), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("skip", [None, [1]])
def test_tokens_behind_a_crop_are_as_if_they_had_not_been(monkeypatch, skip):
    from pbs_attn_amd.patch.huggingface import get_paged_cache
    paged_cpu.use(monkeypatch)
    model, ids, other = paged_cpu.model(skip), _ids(40), _ids(9, 1)
    with torch.no_grad():
        straight, cache = get_paged_cache(model, 1, 60, page_size=32), get_paged_cache(model, 1, 60, page_size=32)
        for c in (straight, cache):
            model(ids[:, :30], past_key_values=c)
        model(other, past_key_values=cache)                       # past a page's end, and back
        assert cache.get_seq_length() == 39
        cache.crop(-9)
        assert [layer.length for layer in cache.layers] == [30, 30]
        want = model(ids[:, 30:], past_key_values=straight).logits
        assert torch.equal(model(ids[:, 30:], past_key_values=cache).logits, want)


def test_how_much_is_taken_off():
    from pbs_attn_amd.patch.paged_cache import PagedKVCache
    from tests.test_paged import _config
    cache = PagedKVCache(_config(), 1, 20, device="cpu")
    for n, left in ((-3, 9), (0, 12), (7, 7), (12, 12), (30, 12), (-12, 0), (-13, 0)):    # below zero: so many; else: what stays, 0 all
        for layer in cache.layers:
            layer.length = 12
            layer.crop(n)
        assert [layer.length for layer in cache.layers] == [left] * 3, n


def test_decoding_with_looked_up_tokens(monkeypatch):
    from pbs_attn_amd.patch.huggingface import get_paged_cache
    paged_cpu.use(monkeypatch)
    model = paged_cpu.model()
    ids = _ids(6).repeat(1, 4)                                    # (what follows a repeated piece is looked up)
    dropped = []
    from pbs_attn_amd.patch.paged_cache import _PagedLayer
    crop = _PagedLayer.crop
    monkeypatch.setattr(_PagedLayer, "crop", lambda self, n: (dropped.append(n), crop(self, n))[1])
    cache = get_paged_cache(model, 1, 64)
    with torch.no_grad():
        out = model.generate(ids, past_key_values=cache, max_new_tokens=10, do_sample=False, prompt_lookup_num_tokens=3, pad_token_id=0, eos_token_id=None)
    assert out.shape[1] >= 34 and dropped and cache.get_seq_length() == out.shape[1] - 1
    assert torch.equal(out[:, :24], ids)


def test_batches_are_not_reordered():
    from pbs_attn_amd.patch.paged_cache import PagedKVCache
    from tests.test_paged import _config
    cache = PagedKVCache(_config(), 2, 20, device="cpu")
    for call in (lambda: cache.batch_select_indices(torch.tensor([0])), lambda: cache.batch_repeat_interleave(2), lambda: cache.reorder_cache(torch.tensor([1, 0]))):
        with pytest.raises(NotImplementedError, match="reorder"):
            call()
