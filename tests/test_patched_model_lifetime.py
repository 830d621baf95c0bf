"""CPU: a patched model's weights go with the last reference to it, not with the collector's next pass, and patching leaves a module what it was otherwise."""
import copy
import gc
import weakref

import pytest
import torch

from tests.test_boundary import _oracle_prefill, _tiny

IDS = torch.randint(0, 97, (1, 40), generator=torch.Generator().manual_seed(2))


def _patch(model, **kw):
    from pbs_attn.patch.huggingface import apply_patch_with_prefill
    return apply_patch_with_prefill(model, _oracle_prefill(block_size=8, segment_size=16, threshold=1), **kw)


def _logits(model, ids=IDS):
    with torch.no_grad():
        return model(ids).logits


@pytest.mark.parametrize("kind", ["llama", "qwen2"])
@pytest.mark.parametrize("times", [1, 2])
@pytest.mark.parametrize("use", [None, "prompt", "generate", "back"])
def test_a_patched_model_that_is_dropped_frees_its_weights(kind, times, use):
    gc.collect()
    gc.disable()
    try:
        model = _tiny(kind)
        for _ in range(times):
            _patch(model)
        if use == "prompt":
            _logits(model)
        elif use == "generate":
            with torch.no_grad():
                model.generate(IDS, max_new_tokens=3, do_sample=False, eos_token_id=None, pad_token_id=0)
        elif use == "back":                     # taken back, which is the user's own cycle, and patched again
            for layer in model.model.layers:
                layer.self_attn.forward = layer.self_attn.original_forward
            _patch(model)
        held = [weakref.ref(x) for x in model.modules()] + [weakref.ref(x) for x in model.parameters()]
        del model
        if use == "back":
            layer = None
        assert [x() for x in held] == [None] * len(held)
    finally:
        gc.enable()


def test_a_module_is_still_what_it_was():
    model = _tiny("llama", layers=3)
    attn, other = model.model.layers[0].self_attn, model.model.layers[1].self_attn
    names, kind, keys = [n for n, _ in model.named_modules()], type(attn), list(model.state_dict())
    _patch(model, skip_layers=[1])
    assert type(other) is kind and isinstance(attn, kind) and type(attn).__name__ == kind.__name__ and type(attn).__module__ == kind.__module__
    assert [n for n, _ in model.named_modules()] == names and list(model.state_dict()) == keys
    assert attn.original_forward.__func__ is kind.forward and attn.original_forward.__self__ is attn


def test_a_copy_of_a_patched_model_has_its_own_weights():
    model = _patch(_tiny("llama"))
    want, twin = _logits(model), copy.deepcopy(model)
    with torch.no_grad():
        for p in model.parameters():
            p.zero_()
    assert torch.equal(_logits(twin), want) and not _logits(model).any()
    assert torch.equal(_logits(twin, IDS[:, :1]), _logits(_tiny("llama"), IDS[:, :1]))     # the module's own forward


def test_patched_again_and_taken_back():
    model = _tiny("llama")
    want, one = _logits(model), _logits(model, IDS[:, :1])
    for _ in range(3):
        _patch(model)
        assert torch.allclose(_logits(model), want, atol=2e-4) and torch.equal(_logits(model, IDS[:, :1]), one)
    for layer in model.model.layers:
        layer.self_attn.forward = layer.self_attn.original_forward
    assert torch.equal(_logits(model), want)
    _patch(model)
    assert torch.allclose(_logits(model), want, atol=2e-4) and torch.equal(_logits(model, IDS[:, :1]), one)


def test_a_forward_that_a_hook_has_put_in_its_place_is_the_original():
    model, calls = _tiny("llama"), []
    attn = model.model.layers[0].self_attn
    inner = attn.forward

    def hooked(*args, **kw):
        calls.append(1)
        return inner(*args, **kw)
    attn.forward = hooked
    want = _logits(model, IDS[:, :1])
    for _ in range(2):
        _patch(model)
        calls.clear()
        assert attn.original_forward is hooked and torch.equal(_logits(model, IDS[:, :1]), want) and len(calls) == 1


def test_a_class_that_another_tool_has_put_on_top_stays():
    """As sharding does: a class of the module's class and its own, made after the patch."""
    model = _tiny("llama")
    want, one = _logits(model), _logits(model, IDS[:, :1])
    _patch(model)
    for layer in model.model.layers:
        cls = type(layer.self_attn)
        layer.self_attn.__class__ = type("Sharded" + cls.__name__, (_Mixin, cls), {})
    for _ in range(2):
        _patch(model)
        assert all(isinstance(layer.self_attn, _Mixin) for layer in model.model.layers)
        assert torch.allclose(_logits(model), want, atol=2e-4) and torch.equal(_logits(model, IDS[:, :1]), one)


class _Mixin:
    pass
