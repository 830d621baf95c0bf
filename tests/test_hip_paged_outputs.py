"""GPU: the tensors that the native calls on a paged cache return are torch's own: of the mode, the pool and the stream that they are made in."""
import pytest
import torch

from pbs_attn_amd import _lib, ops
from pbs_attn_amd.paged import KVPages, alloc_pages

pytestmark = pytest.mark.gpu
FORMS = ["bf16", "fp8", "fp4"]


def _case(form, past=70):
    g = torch.Generator(device="cuda").manual_seed(0)
    x = [torch.randn(1, h, past + 1, 128, generator=g, device="cuda").to(torch.bfloat16) for h in (2, 2, 4)]
    pages, table, n = alloc_pages(3, 2, 64, form), torch.tensor([[2, 0]], dtype=torch.int32, device="cuda"), torch.tensor([past], dtype=torch.int32, device="cuda")
    ops.paged_append(pages, table, n * 0, x[0], x[1])
    return pages, table, n, x[2][:, :, -1:].contiguous(), x[0][:, :, -1:].contiguous()


def _calls(pages, table, n, q, k):
    assert _lib.paged_host() is not _lib._no_paged_host
    return [*_lib.paged_host().append(pages, table, n, k, k, q, None, None, None, True), _lib.paged_host().attn(q, pages, table, n, None, None, None),
            *_lib.paged_host().read(pages, table, n + 1, 71)]


@pytest.mark.parametrize("form", FORMS)
def test_outputs_are_ordinary_tensors(dev, form):
    case = _case(form)
    out = _calls(*case)
    for t in out:
        assert t.dtype == torch.bfloat16 and t.device == case[3].device and t.is_contiguous() and not t.requires_grad and not t.is_inference() and t.is_leaf
        t.record_stream(torch.cuda.current_stream())
        assert torch.equal(t + 0, t.clone()) and t.untyped_storage().nbytes() == t.numel() * 2
    with torch.inference_mode():
        assert all(t.is_inference() for t in _calls(*case))
    before = torch.cuda.memory_allocated()
    more = _calls(*case)
    assert torch.cuda.memory_allocated() > before
    del more
    assert torch.cuda.memory_allocated() == before
    assert (out[2].float().requires_grad_() * 2).requires_grad


@pytest.mark.parametrize("form", FORMS)
def test_inputs_whose_memory_is_not_torchs(dev, form):
    case = _case(form)
    want = _calls(*case)
    pages, table, n, q, k = case
    foreign = lambda t: torch.from_dlpack(t.view(torch.uint8).__dlpack__()).view(t.dtype).view(t.shape)  # noqa: E731
    tensors = [foreign(t) if t is not None else None for t in (pages.k, pages.v, pages.k_scale, pages.v_scale)]
    got = _calls(KVPages(*tensors), foreign(table), foreign(n), foreign(q), foreign(k))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_outputs_of_a_captured_call_are_the_graphs(dev):
    case = _case("fp8")
    want = _calls(*case)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _calls(*case)
    for _ in range(3):
        for t in out:
            t.zero_()
        spoil = [torch.full_like(t, 7) for t in out]      # (memory of the graph's pool is not given away)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and all((t == 7).all() for t in spoil)
