"""GPU: pages that share their memory with another tensor until one of them is written."""
import pytest
import torch

from pbs_attn_amd import ops
from pbs_attn_amd.paged import KVPages, alloc_pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["bf16", "fp4"])
def test_writing_to_a_lazy_copy_leaves_its_source(dev, form):
    pages = alloc_pages(2, 2, 32, form)
    tensors = [t for t in (pages.k, pages.v, pages.k_scale, pages.v_scale) if t is not None]
    for t in tensors:
        t.zero_()
    copy = KVPages(*[torch._lazy_clone(t) for t in tensors])
    x = torch.ones(1, 2, 5, 128, dtype=torch.bfloat16, device=dev)
    ops.paged_append(copy, torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev), x, x)
    assert not any(t.any() for t in tensors) and copy.k.any() and copy.v.any()
