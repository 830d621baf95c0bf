"""CPU: masks that a paged cache's attention does not look at are refused where they hide or show anything else than it does."""
import pytest
import torch

from tests import paged_cpu


def _ids(B, S):
    return torch.randint(0, 101, (B, S), generator=torch.Generator().manual_seed(S))


@pytest.mark.parametrize("attention", ["sdpa", "eager"])
@pytest.mark.parametrize("skip", [None, [1]])
def test_padded_batches_are_refused(monkeypatch, attention, skip):
    from pbs_attn_amd.patch.huggingface import get_paged_cache
    paged_cpu.use(monkeypatch)
    model, plain = paged_cpu.model(skip, attn_implementation=attention), paged_cpu.model(patched=False, attn_implementation=attention)
    ids, ones, padded = _ids(2, 30), torch.ones(2, 30, dtype=torch.long), torch.ones(2, 30, dtype=torch.long)
    padded[1, :4] = 0
    cache = get_paged_cache(model, 2, 40)
    with torch.no_grad():
        with pytest.raises(ValueError, match="padding"):
            model(ids[:, :20], attention_mask=padded[:, :20], past_key_values=cache)
        assert [layer.length for layer in cache.layers] == [0, 0]       # refused before anything was stored
        want = plain(ids).logits
        got = [model(ids[:, :20], attention_mask=ones[:, :20], past_key_values=cache).logits]
        for first, last in ((20, 21), (21, 22), (22, 30)):              # single tokens, a later prompt
            with pytest.raises(ValueError, match="padding"):
                model(ids[:, first:last], attention_mask=padded[:, :last], past_key_values=cache)
            assert [layer.length for layer in cache.layers] == [first, first]
            got.append(model(ids[:, first:last], attention_mask=ones[:, :last], past_key_values=cache).logits)
        # (bf16 layers, two attentions: the bounds of the patched models' own tests)
        assert (torch.cat(got, 1).float() - want.float()).abs().max() < 0.15
        with pytest.raises(ValueError, match="padding"):                # a batch padded on the right
            cache.reset()
            model(ids[:, :20], attention_mask=padded.flip(1)[:, -20:], past_key_values=cache)
        # without a paged cache the patched model takes what it took
        assert model(ids, attention_mask=padded).logits.shape == want.shape


def test_the_first_patched_layer_looks(monkeypatch):
    """All layers of a step have the same mask: one of them reads it, whichever layers are skipped."""
    from pbs_attn_amd.patch import huggingface, paged_cache
    paged_cpu.use(monkeypatch)
    calls = []
    monkeypatch.setattr(paged_cache, "check_mask", lambda mask, past, new: calls.append((past, new)))
    for skip in (None, [0], [0, 1], [2]):
        model = paged_cpu.model(skip, layers=3, attn_implementation="eager")
        cache = huggingface.get_paged_cache(model, 1, 20)
        with torch.no_grad():
            model(_ids(1, 5), past_key_values=cache)
            model(_ids(1, 1), past_key_values=cache)
        assert calls == [(0, 5), (5, 1)], skip
        calls.clear()


def _causal(new, past, extra=0):
    return torch.arange(past + new + extra) <= past + torch.arange(new)[:, None]


@pytest.mark.parametrize("new,past", [(1, 0), (1, 9), (7, 0), (7, 30), (2100, 5)])      # (rows are looked at 1024 at a time)
def test_masks_that_say_what_the_cache_does(new, past):
    from pbs_attn_amd.patch.paged_cache import check_mask
    check_mask(None, past, new)
    check_mask(torch.ones(2, past + new, dtype=torch.long), past, new)
    check_mask(torch.ones(2, past + new, dtype=torch.bool), past, new)
    lowest = torch.finfo(torch.bfloat16).min
    for mask in (_causal(new, past), _causal(new, past, extra=3)):       # (columns behind the last token: a buffer's)
        check_mask(mask[None, None], past, new)
        for low in (lowest, -float("inf")):
            check_mask(torch.zeros(2, 1, *mask.shape, dtype=torch.bfloat16).masked_fill(~mask, low), past, new)


@pytest.mark.parametrize("new,past", [(1, 9), (7, 0), (7, 30), (2100, 5)])
def test_masks_that_say_something_else(new, past):
    from pbs_attn_amd.patch.paged_cache import check_mask
    n = past + new
    two = torch.ones(2, n, dtype=torch.long)
    two[1, 0] = 0
    right = _causal(new, past)[None, None].repeat(2, 1, 1, 1)
    bad = [two, two.bool(), torch.ones(2, n - 1, dtype=torch.long), right[..., :-1], right[:, :, :-1] if new > 1 else right[..., :0], "a mask", right[0]]
    for row, column in ((new - 1, 0), (new // 2, past // 2), (new - 1, n - 1), (0, 0)):
        other = right.clone()
        other[1, 0, row, column] = False
        bad.append(other)
        bad.append(torch.zeros(other.shape).masked_fill(~other, -1e9))
    if new > 1:
        bad.append(torch.ones_like(right))                               # every row sees every key
    bias = torch.zeros(right.shape).masked_fill(~right, -float("inf"))
    bias[0, 0, 0, 0] = -0.5                                              # neither hidden nor as it is
    bad.append(bias)
    for mask in bad:
        with pytest.raises(ValueError, match="padding"):
            check_mask(mask, past, new)
