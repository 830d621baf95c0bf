"""GPU: patched models on a paged cache: prompt, single tokens, a later prompt, layers that are not patched."""
import pytest
import torch

from tests.paged_plain import held_in_4_bits, tokens_of

pytestmark = pytest.mark.gpu


def _patched(model, skip_layers=None):
    from pbs_attn.patch.huggingface import apply_patch_with_prefill, get_permuted_block_sparse_attn_fwd
    apply_patch_with_prefill(model, get_permuted_block_sparse_attn_fwd(segment_size=256, threshold=1), skip_layers)


def _close(got, ref):
    # (the bounds of the patched prompt's own test: bf16 layers, two attention kernels with different summation orders)
    d = (got.float() - ref.float()).abs()
    assert d.max() < 0.15 and d.mean() < 0.02, (d.max(), d.mean())


@pytest.mark.parametrize("name,skip", [("llama31_8b", None), ("qwen25_7b", None), ("llama31_8b", [1])])
def test_prompt_tokens_and_a_later_prompt_on_a_paged_cache(dev, name, skip):
    """Every causal block selected: on the cache the patched model has to reproduce the unpatched one on the whole text."""
    from pbs_attn.patch.huggingface import get_paged_cache
    from pbs_attn_amd.ttft import build_model
    model = build_model(name, layers=2, device=dev)
    ids = torch.randint(0, 1000, (2, 1300), generator=torch.Generator().manual_seed(0)).to(dev)
    with torch.no_grad():
        ref = model(ids).logits
        _patched(model, skip)
        cache = get_paged_cache(model, 2, 1300)
        _close(model(ids[:, :1000], past_key_values=cache).logits, ref[:, :1000])
        for i in range(1000, 1004):
            assert cache.get_seq_length() == i
            _close(model(ids[:, i:i + 1], past_key_values=cache).logits, ref[:, i:i + 1])
        if skip is None:    # (an unpatched module's mask for several tokens on a filled cache is the module's own)
            _close(model(ids[:, 1004:], past_key_values=cache).logits, ref[:, 1004:])
            with pytest.raises(ValueError, match="the cache holds 1300"):
                model(ids[:, :1], past_key_values=cache)
        cache.reset()
        _close(model(ids[:, :1], past_key_values=cache).logits, ref[:, :1])   # a prompt of one token
        with pytest.raises(ValueError, match="a cache of 2 sequences"):
            model(ids[:1, :1], past_key_values=cache)


def test_generation_on_a_paged_cache(dev):
    from pbs_attn.patch.huggingface import get_paged_cache
    from pbs_attn_amd.ttft import build_model
    model = build_model("llama31_8b", layers=2, device=dev)
    ids = torch.randint(0, 1000, (1, 700), generator=torch.Generator().manual_seed(1)).to(dev)
    _patched(model)
    for form in ("bf16", "fp4"):
        cache = get_paged_cache(model, 1, 720, page_size=32, form=form)
        with torch.no_grad():
            out = model.generate(ids, max_new_tokens=12, do_sample=False, past_key_values=cache, eos_token_id=None, pad_token_id=0)
        assert out.shape == (1, 712) and cache.get_seq_length() == 711


def test_what_a_4_bit_cache_holds_of_a_prompt(dev):
    """The first layer's keys and values do not depend on any attention: those of a 4-bit cache are the bf16 cache's in 4 bits."""
    from pbs_attn.patch.huggingface import get_paged_cache
    from pbs_attn_amd.ttft import build_model
    model = build_model("qwen25_7b", layers=1, device=dev)
    ids = torch.randint(0, 1000, (2, 300), generator=torch.Generator().manual_seed(2)).to(dev)
    _patched(model)
    held = []
    for form in ("bf16", "fp4"):
        cache = get_paged_cache(model, 2, 301, form=form)
        with torch.no_grad():
            assert model(ids, past_key_values=cache).logits.isfinite().all()
            model(ids[:, :1], past_key_values=cache)
        held.append([tokens_of(cache.layers[0].pages, cache.page_table[b].tolist(), 301) for b in range(2)])
    for b in range(2):
        for wide, narrow in zip(held[0][b], held[1][b]):
            assert torch.equal(narrow, held_in_4_bits(wide.to(torch.bfloat16)))


def test_a_captured_step_keeps_lengths_of_its_own(dev):
    """The cache's lengths are the host's: a graph would replay those of its capture, so there the cache refuses."""
    from pbs_attn.patch.huggingface import get_paged_cache
    from pbs_attn_amd.ttft import build_model
    cache = get_paged_cache(build_model("llama31_8b", layers=1, device=dev), 1, 64)
    x = torch.zeros(1, 8, 1, 128, dtype=torch.bfloat16, device=dev)
    graph, y = torch.cuda.CUDAGraph(), torch.zeros(4, device=dev)
    with torch.cuda.graph(graph):
        y += 1
        for call in (lambda: cache.layers[0].append(x, x), lambda: cache.update(x, x, 0)):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    graph.replay()
    assert cache.get_seq_length() == 0 and not cache._lengths
    cache.update(x, x, 0)
    assert cache.get_seq_length() == 1 and y.tolist() == [1.0] * 4
