"""GPU: attention over an 8-bit cache of values near the largest that it holds, whose average is finite, and of small ones; many sequences at once."""
import pytest
import torch

from pbs_attn_amd import ops
from pbs_attn_amd.paged import alloc_pages
from tests.paged_fp8_plain import tokens_of
from tests.paged_plain import attention
from tests.test_hip_paged_fp8 import Filled
from tests.test_hip_paged_large_values import LARGE, SIZES

pytestmark = pytest.mark.gpu


def _check(S, total, k, v, q, up=1.0):
    pages = alloc_pages((total + 63) // 64, 2, 64, "fp8")
    table = torch.arange((total + 63) // 64, dtype=torch.int32, device="cuda").flip(0).contiguous().view(1, -1)
    ops.paged_append(pages, table, torch.zeros(1, dtype=torch.int32, device="cuda"), k, v)
    past = torch.tensor([total - S], dtype=torch.int32, device="cuda")
    out = ops.paged_attn(q, pages, table, past, softmax_scale=1.0)
    kk, vv = tokens_of(pages, table[0].tolist(), total)
    want, tol = attention(q[0], kk, vv * up, total - S, S, 1.0)      # (exactly: float64, a power of two)
    assert out.isfinite().all() and ((out[0].double() * up - want).abs() <= tol).all()


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


@pytest.mark.parametrize("S,total", SIZES)
def test_a_large_value_of_a_key_that_weighs_more_than_those_before(dev, S, total):
    g = torch.Generator(device="cuda").manual_seed(S)
    k, v, q = _randn(g, 1, 2, total, 128) * 0.01, _randn(g, 1, 2, total, 128), _randn(g, 1, 8, S, 128) * 0.1
    k[..., 0], q[..., 0] = 0, 1
    at = (total - S) // 2 + 20
    k[:, :, at, 0] = 4
    v[:, :, at, :64], v[:, :, at, 64:] = LARGE, -LARGE
    _check(S, total, k, v, q)


@pytest.mark.parametrize("S,total", SIZES)
def test_large_values_everywhere(dev, S, total):
    g = torch.Generator(device="cuda").manual_seed(S)
    k, q = _randn(g, 1, 2, total, 128) * 0.1, _randn(g, 1, 8, S, 128)
    v = torch.full((1, 2, total, 128), LARGE, dtype=torch.bfloat16, device="cuda")
    v[..., 1::2] *= -1
    _check(S, total, k, v, q)
    v[:, :, :, 64:] *= torch.where(torch.rand(1, 2, total, 64, generator=g, device="cuda") < 0.5, -1, 1).to(torch.bfloat16)
    _check(S, total, k, v, q)


@pytest.mark.parametrize("down", [84, 100])
@pytest.mark.parametrize("S,total", SIZES)
def test_small_values(dev, down, S, total):
    g = torch.Generator(device="cuda").manual_seed(S)
    k, q = _randn(g, 1, 2, total, 128) * 0.1, _randn(g, 1, 8, S, 128)
    v = (_randn(g, 1, 2, total, 128).float() * 2.0 ** -down).to(torch.bfloat16)
    _check(S, total, k, v, q, 2.0 ** down)


@pytest.mark.parametrize("S,total", SIZES)
def test_queries_with_a_few_large_channels(dev, S, total):
    """The queries are two e4m3 numbers a channel, with one power of two a row: channels far below the row's largest, whose keys are as much larger."""
    g = torch.Generator(device="cuda").manual_seed(S)
    k, q = _randn(g, 1, 2, total, 128) * 0.05, _randn(g, 1, 8, S, 128)
    q[..., 3::16] *= 64
    k[..., 3::16] *= 0.015625
    _check(S, total, k, _randn(g, 1, 2, total, 128), q)


@pytest.mark.parametrize("B,S,past", [(65, 1, 300), (150, 3, 70), (300, 1, 1100), (600, 1, 40), (70, 20, 200)])
def test_many_sequences(dev, B, S, past):
    g = torch.Generator().manual_seed(B)
    f = Filled(8, 2, S, [int(torch.randint(0, past + 1, (1,), generator=g)) for _ in range(B - 1)] + [past], page=32, seed=B)
    f.check(f.attn())


@pytest.mark.parametrize("lens", [[20000, 3, 0, 700, 9000], [5] * 40 + [30000], [1000] * 17, [64, 31, 33000]])
@pytest.mark.parametrize("Hq,S", [(8, 1), (8, 6), (8, 14), (28, 5)])
def test_pieces_of_very_different_lengths(dev, lens, Hq, S):
    """Shares that begin and end anywhere in the line of all sequences' steps, in what a piece's beginning counts for among others."""
    f = Filled(Hq, 4 if Hq == 28 else 2, S, lens, page=64, seed=len(lens))
    f.check(f.attn())


@pytest.mark.parametrize("Hq,Hkv,S,page", [(8, 2, 1, 64), (8, 2, 1, 32), (28, 4, 5, 128), (28, 4, 9, 32), (8, 2, 40, 32)])
def test_shares_of_hundreds_of_steps(dev, Hq, Hkv, S, page):
    """Many sequences that list the pages of one long one: a workgroup goes through more steps than it looks up pages for at once."""
    n, B = 70000, 160
    g = torch.Generator(device="cuda").manual_seed(S)
    slots = (n + page - 1) // page
    pages = alloc_pages(slots + 1, Hkv, page, "fp8")
    row = torch.randperm(slots + 1, generator=g, device="cuda")[:slots].int().view(1, -1)
    ops.paged_append(pages, row, torch.zeros(1, dtype=torch.int32, device="cuda"), _randn(g, 1, Hkv, n, 128), _randn(g, 1, Hkv, n, 128))
    q = _randn(g, B, Hq, S, 128)
    past = torch.full((B,), n - S, dtype=torch.int32, device="cuda")
    past[1::3] -= 20000
    out = ops.paged_attn(q, pages, row.expand(B, -1).contiguous(), past)
    k, v = tokens_of(pages, row[0].tolist(), n)
    for b in (0, 1, 77, 158, 159):
        m = int(past[b])
        want, tol = attention(q[b], k[:, :m + S], v[:, :m + S], m, S, 128 ** -0.5)
        assert ((out[b].double() - want).abs() <= tol).all(), b
