"""GPU: calls of the C interface with one workspace, made for a model's largest call, and what lies behind it."""
import pytest
import torch

from pbs_attn_amd import _lib, ops
from tests.test_hip_paged import Filled

pytestmark = pytest.mark.gpu
GUARD = 1 << 16


def _call(f, q, past, new, max_len, ws, n):
    B, Hq, S, D = q.shape
    p, out = f.pages, torch.full_like(q, 7)
    pool, Hkv, size = p.k.shape[:3]
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    rc = _lib.load().pbs_paged_attn_fwd(
        q.data_ptr(), p.k.data_ptr(), p.v.data_ptr(), ptr(p.k_scale), ptr(p.v_scale), f.table.data_ptr(), past.data_ptr(), new.data_ptr(), out.data_ptr(),
        B, Hq, Hkv, S, D, pool, f.table.shape[1], size, p.bits, max_len, *q.stride()[:3], *out.stride()[:3], f.table.stride(0), D ** -0.5, ws.data_ptr(), n,
        torch.cuda.current_stream().cuda_stream)
    assert rc == 0, _lib.load().pbs_last_error()
    return out


@pytest.mark.parametrize("form", ["bf16", "fp8", "fp4"])
def test_one_workspace_for_all_calls_of_a_model(dev, form):
    past = [40000, 3, 2500, 1050, 700, 9000, 0, 130]
    big = {S: Filled(form, 28, 4, S, past, seed=S) for S in (1, 5, 9, 40)}
    bits = big[1].pages.bits
    size = lambda B, S, n: _lib.load().pbs_paged_attn_workspace_bytes(B, 28, 4, S, 128, bits, n)  # noqa: E731
    room = size(8, 40, 40040)
    ws = torch.empty(room + GUARD, dtype=torch.uint8, device=dev)
    for S, f in big.items():
        for B, bound in ((8, 40040), (8, 60000), (1, 40040)):
            if size(B, S, bound) <= room:
                ws.fill_(255)
                got = _call(f, f.q[:B], f.past[:B], f.new[:B], bound, ws, room)
                assert torch.equal(got, ops.paged_attn(f.q[:B], f.pages, f.table[:B], f.past[:B], f.new[:B], max_len=bound)), (S, B, bound)
                assert (ws[room:] == 255).all(), (S, B, bound)
        for i, n in enumerate(past):     # each sequence by itself, with its own bound
            ws.fill_(255)
            one = slice(i, i + 1)
            g = type("One", (), dict(pages=f.pages, table=f.table[one]))
            got = _call(g, f.q[one], f.past[one], f.new[one], n + S, ws, room)
            assert torch.equal(got, ops.paged_attn(f.q[one], f.pages, f.table[one], f.past[one], f.new[one], max_len=n + S)), (S, n)
            assert (ws[room:] == 255).all(), (S, n)
