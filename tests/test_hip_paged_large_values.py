"""GPU: attention over values near the largest that bf16 and 4 bits hold, whose average is finite, and over small ones."""
import pytest
import torch

from pbs_attn_amd import ops
from pbs_attn_amd.paged import alloc_pages
from tests.paged_plain import attention, tokens_of

pytestmark = pytest.mark.gpu
LARGE = 6.0 * 2.0 ** 125      # the largest that both forms hold exactly


def _check(form, S, total, k, v, q, up=1.0):
    pages = alloc_pages((total + 63) // 64, 2, 64, form)
    table = torch.arange((total + 63) // 64, dtype=torch.int32, device="cuda").flip(0).contiguous().view(1, -1)
    ops.paged_append(pages, table, torch.zeros(1, dtype=torch.int32, device="cuda"), k, v)
    past = torch.tensor([total - S], dtype=torch.int32, device="cuda")
    out = ops.paged_attn(q, pages, table, past, softmax_scale=1.0)
    kk, vv = tokens_of(pages, table[0].tolist(), total)
    want, tol = attention(q[0], kk, vv * up, total - S, S, 1.0)      # (exactly: float64, a power of two)
    assert out.isfinite().all() and ((out[0].double() * up - want).abs() <= tol).all()


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


SIZES = [(1, 70), (1, 5000), (3, 700), (5, 5000), (9, 1500), (15, 3000), (20, 100), (20, 5000), (75, 200), (75, 5000)]   # 4 .. 300 rows, cut and whole


@pytest.mark.parametrize("form", ["bf16", "fp4"])
@pytest.mark.parametrize("S,total", SIZES)
def test_a_large_value_of_a_key_that_weighs_more_than_those_before(dev, form, S, total):
    """One logit a little above all others, in the middle: its weight is more than the first one's."""
    g = torch.Generator(device="cuda").manual_seed(S)
    k, v, q = _randn(g, 1, 2, total, 128) * 0.01, _randn(g, 1, 2, total, 128), _randn(g, 1, 8, S, 128) * 0.1
    k[..., 0], q[..., 0] = 0, 1
    at = (total - S) // 2 + 20
    k[:, :, at, 0] = 4
    v[:, :, at, :64], v[:, :, at, 64:] = LARGE, -LARGE
    _check(form, S, total, k, v, q)


@pytest.mark.parametrize("form", ["bf16", "fp4"])
@pytest.mark.parametrize("S,total", SIZES)
def test_large_values_everywhere(dev, form, S, total):
    """All values of a channel alike (their sum is past the range of fp32, their average is not), or of any sign."""
    g = torch.Generator(device="cuda").manual_seed(S)
    k, q = _randn(g, 1, 2, total, 128) * 0.1, _randn(g, 1, 8, S, 128)
    v = torch.full((1, 2, total, 128), LARGE, dtype=torch.bfloat16, device="cuda")
    v[..., 1::2] *= -1
    _check(form, S, total, k, v, q)
    v[:, :, :, 64:] *= torch.where(torch.rand(1, 2, total, 64, generator=g, device="cuda") < 0.5, -1, 1).to(torch.bfloat16)
    _check(form, S, total, k, v, q)


@pytest.mark.parametrize("form", ["bf16", "fp4"])
@pytest.mark.parametrize("S,total", SIZES)
def test_small_values(dev, form, S, total):
    """Values about 2^-84 keep their relative accuracy."""
    g = torch.Generator(device="cuda").manual_seed(S)
    k, q = _randn(g, 1, 2, total, 128) * 0.1, _randn(g, 1, 8, S, 128)
    v = (_randn(g, 1, 2, total, 128).float() * 2.0 ** -84).to(torch.bfloat16)
    _check(form, S, total, k, v, q, 2.0 ** 84)


@pytest.mark.parametrize("form,down", [("bf16", 109), ("bf16", 104), ("fp4", 99)])      # (4 bits: groups of less than 2^-100 are not held exactly)
@pytest.mark.parametrize("S,total", SIZES)
def test_the_smallest_values(dev, form, down, S, total):
    g = torch.Generator(device="cuda").manual_seed(S)
    k, q = _randn(g, 1, 2, total, 128) * 0.1, _randn(g, 1, 8, S, 128)
    v = (_randn(g, 1, 2, total, 128).float() * 2.0 ** -down).to(torch.bfloat16)
    _check(form, S, total, k, v, q, 2.0 ** down)
