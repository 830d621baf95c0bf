"""GPU: patched models on a paged cache in 8 bits: prompt, single tokens, a later prompt, looked-up tokens, layers that are not patched."""
import pytest
import torch

from tests import paged_fp8_plain, paged_plain
from tests.test_hip_paged_model import _close, _patched

pytestmark = pytest.mark.gpu


def test_what_the_cache_holds_of_a_prompt_and_what_follows(dev):
    """The first layer's keys and values do not depend on any attention: those of the 8-bit cache are the bf16 cache's in 8 bits, rounded as they come."""
    from pbs_attn.patch.huggingface import get_paged_cache
    from pbs_attn_amd.ttft import build_model
    model = build_model("qwen25_7b", layers=1, device=dev)
    ids = torch.randint(0, 1000, (2, 325), generator=torch.Generator().manual_seed(2)).to(dev)
    _patched(model)
    cuts = [0, 300, 301, 302, 325]
    held = []
    for form in ("bf16", "fp8"):
        cache = get_paged_cache(model, 2, 330, form=form)
        with torch.no_grad():
            for lo, hi in zip(cuts, cuts[1:]):
                assert model(ids[:, lo:hi], past_key_values=cache).logits.isfinite().all()
        plain = paged_plain if form == "bf16" else paged_fp8_plain
        held.append([plain.tokens_of(cache.layers[0].pages, cache.page_table[b].tolist(), 325) for b in range(2)])
    for b in range(2):
        for wide, narrow in zip(held[0][b], held[1][b]):
            assert torch.equal(narrow, paged_fp8_plain.held_after([wide[:, lo:hi] for lo, hi in zip(cuts, cuts[1:])]))


@pytest.mark.parametrize("skip", [None, [1]])
def test_generation(dev, skip):
    from pbs_attn.patch.huggingface import get_paged_cache
    from pbs_attn_amd.ttft import build_model
    model = build_model("llama31_8b", layers=2, device=dev)
    ids = torch.randint(0, 1000, (1, 700), generator=torch.Generator().manual_seed(1)).to(dev)
    _patched(model, skip)
    cache = get_paged_cache(model, 1, 720, page_size=32, form="fp8")
    with torch.no_grad():
        out = model.generate(ids, max_new_tokens=12, do_sample=False, past_key_values=cache, eos_token_id=None, pad_token_id=0)
    assert out.shape == (1, 712) and cache.get_seq_length() == 711


def test_looked_up_tokens(dev):
    """Tokens that come off again leave at most their share of a block's scale."""
    from pbs_attn.patch.huggingface import get_paged_cache
    from pbs_attn_amd.ttft import build_model
    model = build_model("llama31_8b", layers=2, device=dev)
    ids = torch.randint(1, 1000, (1, 50), generator=torch.Generator().manual_seed(1)).repeat(1, 8).to(dev)
    _patched(model)
    with torch.no_grad():
        cache = get_paged_cache(model, 1, 430, page_size=32, form="fp8")
        out = model.generate(ids, max_new_tokens=12, do_sample=False, prompt_lookup_num_tokens=4, past_key_values=cache, eos_token_id=None, pad_token_id=0)
        assert out.shape == (1, 412) and cache.get_seq_length() == 411 and torch.equal(out[:, :400], ids)
        after = model(out[:, -1:], past_key_values=cache).logits
        fresh = get_paged_cache(model, 1, 430, page_size=32, form="fp8")
        model(out[:, :400], past_key_values=fresh)
        for i in range(400, 412):
            want = model(out[:, i:i + 1], past_key_values=fresh).logits
    _close(after, want)


def test_a_layer_that_reads_its_cache_back(dev):
    from pbs_attn_amd.patch.paged_cache import PagedKVCache
    from tests.test_paged import _config
    g = torch.Generator(device="cuda").manual_seed(0)
    cache, pieces = PagedKVCache(_config(num_hidden_layers=1), 1, 100, form="fp8", device=dev), []
    for S in (50, 1, 1, 7, 30):
        pieces.append([torch.randn(1, 2, S, 128, generator=g, device=dev).to(torch.bfloat16) * S for _ in range(2)])
        got = cache.update(*pieces[-1], 0)
        for x, kv in zip(got, range(2)):
            assert torch.equal(x[0].double(), paged_fp8_plain.held_after([p[kv][0] for p in pieces]))
