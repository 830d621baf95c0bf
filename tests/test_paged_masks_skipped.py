"""CPU: a mask is refused by the first patched layer; layers ahead of it that are not patched have stored the call's tokens by then."""
import pytest
import torch

from tests import paged_cpu


@pytest.mark.parametrize("skip", [[0], [0, 1], [1]])
def test_a_refused_call_leaves_no_tokens(monkeypatch, skip):
    from pbs_attn_amd.patch.huggingface import get_paged_cache
    paged_cpu.use(monkeypatch)
    model = paged_cpu.model(skip, layers=3)
    ids = torch.randint(1, 101, (2, 12), generator=torch.Generator().manual_seed(0))
    mask = torch.ones(2, 12, dtype=torch.long)
    mask[0, :3] = 0
    cache, clean = get_paged_cache(model, 2, 12), get_paged_cache(model, 2, 12)
    with torch.no_grad():
        for first, last in ((0, 10), (10, 11), (11, 12)):
            with pytest.raises(ValueError, match="padding"):
                model(ids[:, first:last], attention_mask=mask[:, :last], past_key_values=cache)
            assert [layer.length for layer in cache.layers] == [first] * 3
            got, want = (model(ids[:, first:last], past_key_values=c).logits for c in (cache, clean))
            assert torch.equal(got, want)
