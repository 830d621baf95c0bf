"""GPU: attention over an 8-bit cache by workgroups of eight waves that share the steps of a few long sequences: one sequence and several, a few steps a
share and hundreds, pages that are not there."""
import pytest
import torch

from pbs_attn_amd import ops
from pbs_attn_amd.paged import alloc_pages
from tests.paged_fp8_plain import tokens_of
from tests.paged_plain import attention
from tests.test_hip_paged_fp8 import Filled, _garbage, _ints, _randn


pytestmark = pytest.mark.gpu
# (a call is cut for eight waves where at most 128 heads' rows, 16 at most each, have 512 steps of 512 keys or more among them)


def _check_missing(f, gone, S, max_len=None):
    """Pages `gone` (slots of each sequence's row) are taken out of the table: their tokens count as not there."""
    size, table = f.pages.page_size, f.table.clone()
    for b, slots in gone.items():
        table[b, slots] = torch.tensor([-1, f.pages.k.shape[0], 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda").repeat(len(slots))[:len(slots)]
    out = ops.paged_attn(f.q, f.pages, table, f.past, f.new, max_len=max_len)
    for b, (past, new) in enumerate(zip(f.past_list, f.new_list)):
        n = past + new
        there = torch.ones(n, dtype=torch.bool, device="cuda")
        for slot in gone.get(b, []):
            there[slot * size:(slot + 1) * size] = False
        k, v = tokens_of(f.pages, f.table[b].tolist(), n)
        want, tol = attention(f.q[b], k, v, past, new, 128 ** -0.5, there)
        assert ((out[b].double() - want).abs() <= tol).all(), b


@pytest.mark.parametrize("Hq,Hkv,S,past,page", [
    (32, 8, 1, [40000], 64),                       # one sequence
    (32, 8, 1, [131071], 128),
    (28, 4, 2, [70001], 32),
    (16, 16, 1, [17000], 256),
    (32, 8, 4, [32768], 64),                       # 16 rows
    (32, 8, 1, [40000, 0, 33, 20000], 64),         # beside short and empty ones
    (8, 2, 1, [9000] * 20 + [5, 16000], 64),
    (8, 1, 2, [30000, 1, 61000, 31, 0, 512, 511], 64),
])
def test_long_sequences(dev, Hq, Hkv, S, past, page):
    f = Filled(Hq, Hkv, S, past, page=page, seed=len(past))
    out = f.attn()
    f.check(out)
    assert all(torch.equal(f.attn(), out) for _ in range(2))


@pytest.mark.parametrize("S", [1, 4])
def test_a_sequence_without_a_new_token_and_missing_pages(dev, S):
    f = Filled(32, 8, S, [40000, 39000, 900], [S, 0, 1], page=64)
    f.check(f.attn())
    last = (40000 + S - 1) // 64
    # single pages, runs over the steps of a wave and of a whole workgroup, the first and the last
    _check_missing(f, {0: [3, 100, 101, *range(200, 230), 500], 2: [0, 14]}, S)
    _check_missing(f, {0: [0, 1, last]}, S)
    _check_missing(f, {0: list(range(1, last)), 2: list(range(15))}, S)


@pytest.mark.parametrize("Hq,Hkv,S,page,B,n", [(8, 2, 1, 64, 60, 70000), (28, 4, 1, 32, 30, 70000), (8, 1, 2, 128, 120, 70001), (4, 1, 1, 32, 100, 131072)])
def test_shares_of_many_steps(dev, Hq, Hkv, S, page, B, n):
    """Sequences that list the pages of one long one: a workgroup's waves look pages up more than once, in the middle of a unit and at its end."""
    g = torch.Generator(device="cuda").manual_seed(B)
    slots = (n + page - 1) // page
    pages = _garbage(alloc_pages(slots + 1, Hkv, page, "fp8"))
    row = torch.randperm(slots + 1, generator=g, device="cuda")[:slots].int().view(1, -1)
    ops.paged_append(pages, row, _ints(0), _randn(g, 1, Hkv, n, 128), _randn(g, 1, Hkv, n, 128))
    q = _randn(g, B, Hq, S, 128)
    past = torch.full((B,), n - S, dtype=torch.int32, device="cuda")
    past[1::3] -= 20000
    out = ops.paged_attn(q, pages, row.expand(B, -1).contiguous(), past)
    k, v = tokens_of(pages, row[0].tolist(), n)
    for b in (0, 1, 2, B // 2, B - 2, B - 1):
        m = int(past[b])
        want, tol = attention(q[b], k[:, :m + S], v[:, :m + S], m, S, 128 ** -0.5)
        assert ((out[b].double() - want).abs() <= tol).all(), b
