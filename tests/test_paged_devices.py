"""CPU: a paged cache lies on one device, and a model that does not is refused before any of its layers runs."""
import pytest

from tests import paged_cpu


def test_a_model_on_several_devices_is_refused():
    from pbs_attn_amd.patch.huggingface import get_paged_cache
    model = paged_cpu.model()
    assert get_paged_cache(model, 1, 8).page_table.device.type == "cpu"
    model.model.layers[1].to("meta")
    with pytest.raises(ValueError, match="one device"):
        get_paged_cache(model, 1, 8)
