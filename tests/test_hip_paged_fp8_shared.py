"""GPU: a block of an 8-bit cache that two sequences share and one of them adds to: what the other reads before it and, by an event, behind it."""
import pytest
import torch

from pbs_attn_amd import ops
from pbs_attn_amd.paged import alloc_pages
from tests.paged_fp8_plain import check_append, clone, tokens_of
from tests.paged_plain import attention
from tests.test_hip_paged_fp8 import _garbage, _ints, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("up", [0.25, 64.0])         # the owner's tokens leave the block's exponent, or take it up
@pytest.mark.parametrize("shared,page", [(20, 32), (84, 64)])
def test_a_reader_of_the_owners_last_block(dev, up, shared, page):
    g = torch.Generator(device="cuda").manual_seed(shared)
    slots = shared // page + 1
    pages = _garbage(alloc_pages(slots + 1, 2, page, "fp8"))
    table = torch.randperm(slots + 1, generator=g, device="cuda")[:slots].int().view(1, -1)
    past, q = _ints(shared - 1), _randn(g, 1, 8, 1, 128)
    ops.paged_append(pages, table, _ints(0), _randn(g, 1, 2, shared, 128), _randn(g, 1, 2, shared, 128))
    k, v = _randn(g, 1, 2, 5, 128) * up, _randn(g, 1, 2, 5, 128) * up
    torch.cuda.synchronize()
    reader, written, read = torch.cuda.Stream(), torch.cuda.Event(), torch.cuda.Event()

    def look():
        with torch.cuda.stream(reader):
            out = ops.paged_attn(q, pages, table, past), *ops.paged_read(pages, table, past + 1, shared)
            read.record()
        return out

    def check(out, held):
        kk, vv = tokens_of(held, table[0].tolist(), shared)
        want, tol = attention(q[0], kk, vv, shared - 1, 1, 128 ** -0.5)
        assert ((out[0][0].double() - want).abs() <= tol).all()
        assert torch.equal(out[1][0].double(), kk) and torch.equal(out[2][0].double(), vv)

    before = clone(pages)
    torch.cuda.synchronize()
    first = look()
    read.wait()
    ops.paged_append(pages, table, _ints(shared), k, v)
    written.record()
    reader.wait_event(written)
    second = look()
    torch.cuda.synchronize()
    check(first, before)
    check(second, pages)
    check_append(before, pages, table[0].tolist(), shared, k[0], v[0])
    changed = not torch.equal(first[2], second[2])
    assert changed == (up > 1)
