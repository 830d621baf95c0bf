"""GPU: decoding with looked-up tokens on a paged cache: several tokens are checked at once, and those that are not taken come off again."""
import pytest
import torch

from tests.test_hip_paged_model import _close, _patched

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["bf16", "fp4"])
def test_looked_up_tokens(dev, form):
    from pbs_attn.patch.huggingface import get_paged_cache
    from pbs_attn_amd.ttft import build_model
    model = build_model("llama31_8b", layers=2, device=dev)
    ids = torch.randint(1, 1000, (1, 50), generator=torch.Generator().manual_seed(1)).repeat(1, 8).to(dev)
    _patched(model)
    with torch.no_grad():
        cache = get_paged_cache(model, 1, 430, page_size=32, form=form)
        out = model.generate(ids, max_new_tokens=12, do_sample=False, prompt_lookup_num_tokens=4, past_key_values=cache, eos_token_id=None, pad_token_id=0)
        assert out.shape == (1, 412) and cache.get_seq_length() == 411 and torch.equal(out[:, :400], ids)
        # what the cache holds after all that is what it holds of the text
        after = model(out[:, -1:], past_key_values=cache).logits
        fresh = get_paged_cache(model, 1, 430, page_size=32, form=form)
        model(out[:, :400], past_key_values=fresh)
        for i in range(400, 412):
            want = model(out[:, i:i + 1], past_key_values=fresh).logits
    _close(after, want)
