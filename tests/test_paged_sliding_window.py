"""CPU: a paged cache attends to all that is cached; a model with windows is refused."""
import pytest

from pbs_attn_amd.patch.paged_cache import PagedKVCache


def _qwen(**kw):
    from transformers import Qwen2Config
    return Qwen2Config(**{**dict(hidden_size=512, num_attention_heads=4, num_key_value_heads=2, num_hidden_layers=3), **kw})


def test_models_with_sliding_windows_are_refused():
    for config in (_qwen(use_sliding_window=True, max_window_layers=1), _qwen(layer_types=["full_attention", "chunked_attention", "full_attention"])):
        with pytest.raises(ValueError, match="attends to all"):
            PagedKVCache(config, 1, 64, device="cpu")
    for config in (_qwen(), _qwen(use_sliding_window=True, max_window_layers=3)):      # no layer has one
        assert len(PagedKVCache(config, 1, 64, device="cpu").layers) == 3


def test_a_configuration_without_layer_types():
    class Config:
        hidden_size, num_attention_heads, num_key_value_heads, num_hidden_layers = 512, 4, 2, 1
    assert len(PagedKVCache(Config, 1, 64, device="cpu").layers) == 1
    Config.use_sliding_window = True
    with pytest.raises(ValueError, match="attends to all"):
        PagedKVCache(Config, 1, 64, device="cpu")
