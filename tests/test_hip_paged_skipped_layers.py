"""GPU: a later prompt on a paged cache where some layers keep the module's own attention."""
import pytest
import torch

from tests.test_hip_paged_model import _close, _patched

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("skip", [[0], [1]])
def test_a_later_prompt_with_layers_that_are_not_patched(dev, skip):
    from pbs_attn.patch.huggingface import get_paged_cache
    from pbs_attn_amd.ttft import build_model
    model = build_model("llama31_8b", layers=2, device=dev)
    ids = torch.randint(0, 1000, (2, 700), generator=torch.Generator().manual_seed(0)).to(dev)
    with torch.no_grad():
        ref = model(ids).logits
        _patched(model, skip)
        cache = get_paged_cache(model, 2, 700)
        _close(model(ids[:, :400], past_key_values=cache).logits, ref[:, :400])
        _close(model(ids[:, 400:401], past_key_values=cache).logits, ref[:, 400:401])
        _close(model(ids[:, 401:], past_key_values=cache).logits, ref[:, 401:])
        assert cache.get_seq_length() == 700
