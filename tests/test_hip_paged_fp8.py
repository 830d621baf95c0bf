"""GPU: the paged cache in 8 bits against plain float64: what is written, what is read back, the attention over it."""
import pytest
import torch

from pbs_attn_amd import ops
from pbs_attn_amd.paged import KVPages, alloc_pages
from tests.paged_fp8_plain import block_of, check_append, check_untouched, clone, code_values, tokens_of
from tests.paged_plain import attention, rotated

pytestmark = pytest.mark.gpu


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def _tokens(g, *shape):
    """Rows whose sizes differ by powers of two, so that a block's scale grows with them."""
    return (torch.randn(shape, generator=g, device="cuda") * torch.randn(shape[:-1] + (1,), generator=g, device="cuda").exp2()).to(torch.bfloat16)


def _garbage(pages):
    """What an earlier owner may have left in the pages: NaNs, and scales that are none."""
    for t in (pages.k, pages.v, pages.k_scale, pages.v_scale):
        t.view(torch.uint8).fill_(255)
    return pages


def _table(g, B, slots, pool):
    return torch.randperm(pool, generator=g, device="cuda")[:B * slots].view(B, slots).int()


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Filled:
    """A cache of B sequences with `past` tokens each, written by ops.paged_append, and the new tokens' Q, K and V appended."""

    def __init__(self, Hq, Hkv, S, past, new=None, page=64, seed=0, spare=3, slots=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        B = len(past)
        new = [S] * B if new is None else new
        slots = slots or max(1, max((p + n + page - 1) // page for p, n in zip(past, new)))
        self.pages = _garbage(alloc_pages(B * slots + spare, Hkv, page, "fp8"))
        self.table = _table(g, B, slots, B * slots + spare)
        self.past, self.new, self.past_list, self.new_list = _ints(*past), _ints(*new), past, new
        self.q = _randn(g, B, Hq, S, 128)
        longest = max(past)
        if longest:
            ops.paged_append(self.pages, self.table, _ints(*[0] * B), _randn(g, B, Hkv, longest, 128), _randn(g, B, Hkv, longest, 128), new_lens=self.past)
        ops.paged_append(self.pages, self.table, self.past, _randn(g, B, Hkv, S, 128), _randn(g, B, Hkv, S, 128), new_lens=self.new)

    def check(self, out, q=None, scale=128 ** -0.5):
        q = self.q if q is None else q
        assert out.shape == q.shape and out.dtype == torch.bfloat16
        for b, (past, new) in enumerate(zip(self.past_list, self.new_list)):
            k, v = tokens_of(self.pages, self.table[b].tolist(), past + new)
            want, tol = attention(q[b], k, v, past, new, scale)
            over = (out[b].double() - want).abs() > tol
            assert not over.any(), (b, past, new, int(over.sum()), ((out[b].double() - want).abs() / tol.clamp_min(1e-30)).max().item())

    def attn(self, **kw):
        return ops.paged_attn(self.q, self.pages, self.table, self.past, self.new, **kw)


# ---- writing -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("B,Hq,Hkv,S,past,new,page", [
    (1, 4, 1, 1, [0], [1], 32),
    (1, 32, 8, 1, [777], [1], 64),
    (3, 8, 2, 1, [31, 32, 0], [1, 1, 0], 32),           # around a block's border; one sequence without a new token
    (2, 28, 4, 33, [5, 64], [33, 20], 64),
    (3, 5, 5, 100, [0, 1, 250], [100, 0, 77], 256),
    (1, 7, 1, 300, [127], [300], 128),
    (1, 2, 2, 9, [3], [9], 64),                          # inside a block, from the middle of one group of eight to the middle of another
    (2, 4, 2, 40, [24, 31], [1, 40], 32),
])
def test_append_writes_what_its_layout_says(dev, B, Hq, Hkv, S, past, new, page):
    g = torch.Generator(device="cuda").manual_seed(S)
    slots = max((p + n + page - 1) // page for p, n in zip(past, new)) or 1
    pages = _garbage(alloc_pages(B * slots + 2, Hkv, page, "fp8"))
    table = _table(g, B, slots, B * slots + 2)
    if max(past):
        x, y = _tokens(g, B, Hkv, max(past), 128), _tokens(g, B, Hkv, max(past), 128)
        before = clone(pages)
        ops.paged_append(pages, table, _ints(*[0] * B), x, y, new_lens=_ints(*past))
        for b in range(B):
            check_append(before, pages, table[b].tolist(), 0, x[b, :, :past[b]], y[b, :, :past[b]])
    before = clone(pages)
    q, k, v = (_tokens(g, B, S, H, 128).transpose(1, 2) for H in (Hq, Hkv, Hkv))   # as projections leave them
    angle = torch.rand(B, S, 64, generator=g, device="cuda").repeat(1, 1, 2) * 6.28
    cos, sin = angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)
    q_rot, k_rot = ops.paged_append(pages, table, _ints(*past), k, v, q=q, cos=cos, sin=sin, new_lens=_ints(*new), want_k=True)
    for got, x in ((q_rot, q), (k_rot, k)):
        want, tol = rotated(x, cos, sin)
        assert got.is_contiguous() and ((got.double() - want).abs() <= tol).all()
    touched = set()
    for b in range(B):
        if new[b]:
            touched |= check_append(before, pages, table[b].tolist(), past[b], k_rot[b, :, :new[b]], v[b, :, :new[b]])
    check_untouched(before, pages, touched)


@pytest.mark.parametrize("size", [lambda i: 1.5 ** i, lambda i: 1.5 ** -i, lambda i: 2.0 ** (7 * i - 60), lambda i: 0.0 if i < 9 else 1.0, lambda i: float(i % 3)])
def test_tokens_one_by_one(dev, size):
    """A block's scale follows its tokens up, never down, and starts anew with the next block; what was there is rounded once more."""
    g = torch.Generator(device="cuda").manual_seed(11)
    pages, table = _garbage(alloc_pages(3, 2, 32, "fp8")), _ints(2, 0, 1).view(1, 3)
    past = 0
    for i, n in enumerate([1, 1, 2, 1, 7, 1, 1, 17, 1, 1, 1, 13, 1, 1]):
        k, v = (_randn(g, 1, 2, n, 128) * size(i) for _ in range(2))
        before = clone(pages)
        ops.paged_append(pages, table, _ints(past), k, v)
        check_untouched(before, pages, check_append(before, pages, table[0].tolist(), past, k[0], v[0]))
        past += n


def test_append_without_rotation_or_queries(dev):
    g = torch.Generator(device="cuda").manual_seed(3)
    pages = _garbage(alloc_pages(4, 2, 64, "fp8"))
    k, v = _randn(g, 1, 2, 50, 128), _randn(g, 1, 2, 50, 128)
    before = clone(pages)
    assert ops.paged_append(pages, _ints(2, 1).view(1, 2), _ints(64), k, v) == (None, None)
    check_untouched(before, pages, check_append(before, pages, [2, 1], 64, k[0], v[0]))
    q, k_rot = ops.paged_append(pages, _ints(2, 1).view(1, 2), _ints(64), k, v, q=k, want_k=True)
    assert torch.equal(q, k) and torch.equal(k_rot, k)


def test_append_takes_strided_rows_and_broadcast_cosines(dev):
    g = torch.Generator(device="cuda").manual_seed(4)
    wide = _randn(g, 2, 70, 3 * 4 * 128 + 8)           # one projection for Q, K and V, rows padded
    q, k, v = (wide[..., i * 512:i * 512 + 512].unflatten(-1, (4, 128)).transpose(1, 2) for i in range(3))
    angle = torch.rand(1, 70, 128, generator=g, device="cuda") * 6.28
    cos, sin = angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)
    pages = _garbage(alloc_pages(6, 4, 64, "fp8"))
    table = torch.tensor([[0, 1, 9], [3, 4, 9]], dtype=torch.int32, device="cuda")[:, :2]   # rows further apart than they are long
    before = clone(pages)
    q_rot, k_rot = ops.paged_append(pages, table, _ints(0, 32), k, v, q=q, cos=cos, sin=sin, want_k=True)
    for got, x in ((q_rot, q), (k_rot, k)):
        want, tol = rotated(x, cos.expand(2, -1, -1), sin.expand(2, -1, -1))
        assert ((got.double() - want).abs() <= tol).all()
    check_append(before, pages, [0, 1], 0, k_rot[0], v[0])
    check_append(before, pages, [3, 4], 32, k_rot[1], v[1])
    odd = _randn(g, 2, 4, 70, 129)[..., :128]          # rows off their 16 bytes are copied first
    before = clone(pages)
    q2, k2 = ops.paged_append(pages, table, _ints(0, 32), odd, odd, q=odd, cos=cos, sin=sin, want_k=True)
    assert torch.equal(q2, k2)
    check_append(before, pages, [3, 4], 32, k2[1], odd[1])


def _edges():
    """Blocks (32, 128) at the edges of the format: every code and the ties between them at several scales, the largest and smallest magnitudes, zeros,
    infinities and NaN."""
    level = code_values()[:127]
    ties = torch.cat((level, (level[1:] + level[:-1]) / 2)).float()
    blocks = []
    for scale in (1.0, 2.0 ** -100, 2.0 ** 119, 2.0 ** -7):
        x = torch.zeros(32 * 128)
        x[0], x[1:254], x[300:553] = 448.0, ties, -ties
        blocks.append(x * scale)
    for top in (448.0, 450.0, 446.0, 512.0, 256.0, 1.75 * 2.0 ** 127, 1.99 * 2.0 ** 127, 2.0 ** -92, 2.0 ** -110, 2.0 ** -133):
        x = torch.linspace(-1, 1, 32 * 128) * min(top, 2.0 ** 126)
        x[77] = top
        blocks.append(x)
    blocks += [torch.zeros(32 * 128), -torch.zeros(32 * 128)]
    for bad in (float("inf"), -float("inf"), float("nan")):
        x = torch.linspace(-3, 3, 32 * 128)
        x[5], x[2000] = bad, bad
        blocks.append(x)
    blocks.append(torch.full((32 * 128,), float("inf")))
    return torch.stack(blocks).view(-1, 128).to(torch.bfloat16).cuda()


def test_values_at_the_edges_of_the_format(dev):
    x = _edges()[None, None]
    n = x.shape[2]
    pages, table = _garbage(alloc_pages((n + 63) // 64, 1, 64, "fp8")), torch.arange((n + 63) // 64, dtype=torch.int32, device="cuda").view(1, -1)
    v = x.flip(2).contiguous()
    before = clone(pages)
    ops.paged_append(pages, table, _ints(0), x, v)
    check_append(before, pages, table[0].tolist(), 0, x[0], v[0])
    kk, vv = tokens_of(pages, table[0].tolist(), n)
    k, v = ops.paged_read(pages, table, _ints(n), n)
    for got, want in ((k, kk), (v, vv)):
        assert torch.equal(got[0].isnan(), want.isnan()) and torch.equal(got[0].double().nan_to_num(0), want.nan_to_num(0))


def test_blocks_at_the_edges_that_other_tokens_join(dev):
    """Each of those blocks short of its last token, which then joins it, larger and smaller."""
    x = _edges().view(1, -1, 32, 128)      # a block a head
    H = x.shape[1]
    for last in (2.0 ** 127, 1.0, 2.0 ** -120, 3.0 * 2.0 ** 14, float("nan")):
        pages, table = _garbage(alloc_pages(1, H, 32, "fp8")), _ints(0).view(1, 1)
        before = clone(pages)
        ops.paged_append(pages, table, _ints(0), x[:, :, :31], x[:, :, :31])
        check_append(before, pages, [0], 0, x[0, :, :31], x[0, :, :31])
        y = torch.full((1, H, 1, 128), last, dtype=torch.bfloat16, device="cuda")
        before = clone(pages)
        ops.paged_append(pages, table, _ints(31), y, y)
        check_append(before, pages, [0], 31, y[0], y[0])


# ---- reading -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("page", [32, 64, 128, 256])
def test_read_gives_the_tokens_and_zeros_behind_them(dev, page):
    f = Filled(3, 3, 5, [0, 28, 300, 64], page=page)
    lens = f.past + f.new
    for max_len in (1, 31, 70, 305, 333):
        k, v = ops.paged_read(f.pages, f.table, lens, max_len)
        assert k.shape == v.shape == (4, 3, max_len, 128)
        for b, n in enumerate(lens.tolist()):
            n = min(n, max_len)
            kk, vv = tokens_of(f.pages, f.table[b].tolist(), n)
            assert torch.equal(k[b, :, :n].double(), kk) and torch.equal(v[b, :, :n].double(), vv)
            assert not k[b, :, n:].any() and not v[b, :, n:].any()
    k, v = ops.paged_read(f.pages, f.table, _ints(0, -5, 2 ** 31 - 1, 2 ** 31 - 1), 40)     # no tokens; lengths that no cache has
    assert not k[:2].any() and not v[:2].any() and k[2].isfinite().all()


# ---- attention -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("Hq,Hkv,S,past,new,page", [
    (4, 1, 1, [0], None, 32),                            # one key
    (32, 8, 1, [1003], None, 64),
    (8, 2, 1, [30, 31, 32, 33, 0, 127, 128], None, 32),  # around the tiles' borders
    (28, 4, 1, [500, 3, 0, 77], [1, 0, 0, 1], 64),       # sequences without a new token, one of them empty
    (16, 16, 1, [90, 1000], None, 128),                  # one query head a KV head
    (32, 1, 1, [700], None, 64),                         # one KV head for all: more rows than a tile of the matrix instruction has
    (5, 1, 3, [61], None, 32),                           # 15 rows
    (28, 4, 5, [100, 40], [5, 2], 64),                   # 35 rows: drafted tokens
    (20, 4, 2, [5000], None, 256),
    (28, 4, 3, [90, 300], [3, 1], 128),                  # 21 rows
    (28, 4, 7, [2, 400], [4, 7], 32),                    # 49 rows
    (8, 1, 8, [600], None, 64),                          # 64 rows
    (8, 2, 33, [0, 200], [33, 30], 64),                  # prompts: rows that see few keys beside rows that see many
    (6, 2, 100, [1500, 0], [64, 100], 128),
    (4, 4, 257, [300], None, 64),
    (28, 4, 140, [700, 64], [140, 31], 32),
])
def test_attention_over_the_pages(dev, Hq, Hkv, S, past, new, page):
    f = Filled(Hq, Hkv, S, past, new, page)
    f.check(f.attn())
    if S > 1:
        for b, n in enumerate(f.new_list):
            assert not f.attn()[b, :, n:].any()
    # a bound on the lengths changes how the work is cut, not what comes out
    f.check(f.attn(max_len=max(p + n for p, n in zip(f.past_list, f.new_list))))


@pytest.mark.parametrize("B,Hq,Hkv,S,past", [(1, 8, 2, 1, 40000), (2, 4, 1, 3, 33333), (40, 28, 4, 1, 900), (1, 32, 8, 200, 5000), (300, 8, 2, 1, 400),
                                             # every number of row tiles, a few long sequences beside short ones
                                             (3, 28, 4, 3, 6000), (3, 28, 4, 5, 6000), (3, 28, 4, 9, 6000), (1, 28, 4, 9, 20000), (5, 28, 4, 20, 3000)])
def test_attention_over_long_caches_and_many_sequences(dev, B, Hq, Hkv, S, past):
    g = torch.Generator().manual_seed(B)
    pasts = [past] + [int(torch.randint(0, past, (1,), generator=g)) for _ in range(B - 1)]
    f = Filled(Hq, Hkv, S, pasts, page=64, seed=B)
    f.check(f.attn())
    f.check(f.attn(max_len=past + S, softmax_scale=0.02), scale=0.02)


def test_attention_where_few_keys_weigh(dev):
    """Logits of hundreds: the largest exponent grows from tile to tile, most weights vanish."""
    f = Filled(8, 2, 2, [700, 64], page=64)
    f.q = f.q * 16
    f.check(f.attn())


@pytest.mark.parametrize("S", [2, 9, 40])
def test_attention_over_blocks_of_different_scales(dev, S):
    g = torch.Generator(device="cuda").manual_seed(S)
    n = 900
    pages, table = _garbage(alloc_pages(20, 2, 64, "fp8")), _table(g, 1, 15, 20)
    up = torch.randint(-6, 7, (1, 2, n // 32 + 1, 1), generator=g, device="cuda").repeat_interleave(32, 2)[:, :, :n].float().exp2()
    k, v = (_randn(g, 1, 2, n, 128) * 0.1 * up).to(torch.bfloat16), (_randn(g, 1, 2, n, 128) * up.flip(2)).to(torch.bfloat16)
    ops.paged_append(pages, table, _ints(0), k, v)
    q = _randn(g, 1, 8, S, 128)
    out = ops.paged_attn(q, pages, table, _ints(n - S))
    want, tol = attention(q[0], *tokens_of(pages, table[0].tolist(), n), n - S, S, 128 ** -0.5)
    assert ((out[0].double() - want).abs() <= tol).all()


def test_attention_reads_queries_where_they_are(dev):
    f = Filled(8, 2, 3, [100, 37], page=64)
    q = f.q.transpose(1, 2).contiguous().transpose(1, 2)          # token-major
    assert torch.equal(ops.paged_attn(q, f.pages, f.table, f.past, f.new), f.attn())
    odd = torch.zeros(2, 8, 3, 129, dtype=torch.bfloat16, device="cuda")[..., 1:]
    odd.copy_(f.q)
    assert torch.equal(ops.paged_attn(odd, f.pages, f.table, f.past, f.new), f.attn())
    wide = torch.full((2, f.table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")   # a longer table; what is not reached is not read
    wide[:, :f.table.shape[1]] = f.table
    f.check(ops.paged_attn(f.q, f.pages, wide, f.past, f.new))
    assert torch.equal(ops.paged_attn(f.q, f.pages, f.table, f.past), f.attn())


@pytest.mark.parametrize("S", [2, 12, 40])
def test_pages_outside_the_pool_and_behind_the_table(dev, S):
    f = Filled(8, 2, S, [300, 10], page=64, slots=6)
    assert 0 not in f.table[0].tolist() or f.pages.k.shape[0] > 12
    f.pages.k_scale[f.table.new_tensor([i for i in range(f.pages.k.shape[0]) if i not in f.table.flatten().tolist()]).long()] = 255
    table = f.table.clone()
    table[0, 1], table[0, 3] = -1, f.pages.k.shape[0]              # tokens 64..127 and 192..255 of the first sequence are not there
    out = ops.paged_attn(f.q, f.pages, table, f.past, f.new)
    there = torch.ones(300 + S, dtype=torch.bool, device="cuda")
    there[64:128] = there[192:256] = False
    k, v = tokens_of(f.pages, f.table[0].tolist(), 300 + S)
    want, tol = attention(f.q[0], k, v, 300, S, 128 ** -0.5, there)
    assert ((out[0].double() - want).abs() <= tol).all()
    assert torch.equal(out[1], f.attn()[1])
    k, v = ops.paged_read(f.pages, table, f.past + f.new, 302)
    assert not k[0, :, 64:128].any() and not v[0, :, 192:256].any() and k[0, :, 128:192].any()
    all_bad = torch.full_like(table, 1 << 30)
    assert not ops.paged_attn(f.q, f.pages, all_bad, f.past, f.new).any()
    # writing: nothing happens to any page
    before = clone(f.pages)
    x = torch.ones(2, 2, 2, 128, dtype=torch.bfloat16, device="cuda")
    for t in (all_bad, f.table[:, :2].contiguous()):
        ops.paged_append(f.pages, t, _ints(300, 2 ** 31 - 1), x, x)
        check_untouched(before, f.pages, set())


@pytest.mark.parametrize("S", [1, 3, 20])
@pytest.mark.parametrize("past", [40, 1500])
def test_the_first_page_of_the_pool_may_hold_anything(dev, S, past):
    """A tile that is not there is read as the pool's first one: NaN codes and a scale that is none reach nothing."""
    g = torch.Generator(device="cuda").manual_seed(S)
    n = past + S
    pages, slots = _garbage(alloc_pages(n // 32 + 3, 2, 32, "fp8")), n // 32 + 1
    table = torch.arange(1, slots + 1, dtype=torch.int32, device="cuda").view(1, -1)
    ops.paged_append(pages, table, _ints(0), _randn(g, 1, 2, n, 128), _randn(g, 1, 2, n, 128))
    q, there = _randn(g, 1, 8, S, 128), torch.ones(n, dtype=torch.bool, device="cuda")
    k, v = tokens_of(pages, table[0].tolist(), n)
    table[0, 0], there[:32] = -7, False
    out = ops.paged_attn(q, pages, table, _ints(past))
    want, tol = attention(q[0], k, v, past, S, 128 ** -0.5, there)
    assert ((out[0].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("S", [1, 20])
def test_sequences_that_share_their_first_pages(dev, S):
    """Three sequences behind the same 128 tokens, written once: each appends to pages of its own."""
    g = torch.Generator(device="cuda").manual_seed(S)
    pages = _garbage(alloc_pages(9, 2, 64, "fp8"))
    table = torch.tensor([[4, 7, 0], [4, 7, 2], [4, 7, 8]], dtype=torch.int32, device="cuda")
    ops.paged_append(pages, table[:1], _ints(0), _randn(g, 1, 2, 128, 128), _randn(g, 1, 2, 128, 128))
    k, v, q = _randn(g, 3, 2, S, 128), _randn(g, 3, 2, S, 128), _randn(g, 3, 8, S, 128)
    ops.paged_append(pages, table, _ints(128, 128, 128), k, v)
    out = ops.paged_attn(q, pages, table, _ints(128, 128, 128))
    for b in range(3):
        kk, vv = tokens_of(pages, table[b].tolist(), 128 + S)
        want, tol = attention(q[b], kk, vv, 128, S, 128 ** -0.5)
        assert ((out[b].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("S", [1, 20])
@pytest.mark.parametrize("past", [40, 3000])
def test_infinities_and_nans_reach_the_rows_that_see_them(dev, S, past):
    f = Filled(8, 2, S, [past, past])
    clean = f.attn()
    f.q[0, 3, 0, 17] = float("nan")                 # one query row
    out = f.attn()
    assert out[0, 3, 0].isnan().all()
    out[0, 3, 0] = clean[0, 3, 0]
    assert torch.equal(out, clean)
    f.q[0, 3, 0, 17] = 0.5
    k = torch.zeros(2, 2, 1, 128, dtype=torch.bfloat16, device="cuda")
    k[1, 0, 0, 5] = float("inf")
    last = f.past + S - 1                           # the last token's key, which only the last query sees: head 0 of the second sequence
    v = ops.paged_read(f.pages, f.table, f.past + S, past + S)[1][:, :, -1:].contiguous()
    before = f.attn()
    ops.paged_append(f.pages, f.table, last, k, v)
    out = f.attn()
    assert torch.equal(out[:, :, :-1], before[:, :, :-1]) and out[0].isfinite().all() and out[1, 4:].isfinite().all()
    assert out[1, :4, -1].isnan().all()             # (held as NaN)


@pytest.mark.parametrize("S,past", [(2, 0), (4, 40), (7, 3000), (11, 40), (11, 3000), (16, 40), (16, 3000), (40, 0), (40, 3000), (75, 1030)])   # 8 .. 300 rows
def test_values_that_are_not_finite_reach_no_earlier_row(dev, S, past):
    """Infinities and NaN among the new tokens' values: rows before them keep their bits, rows from them on get NaN in their channels, no other channel does."""
    f = Filled(8, 2, S, [past, past])
    clean = f.attn()
    k, v = (x[:, :, past:].contiguous() for x in ops.paged_read(f.pages, f.table, f.past + S, past + S))
    t = S // 2
    v[1, 0, t, 5], v[1, 0, t, 38], v[1, 0, t, 71] = float("inf"), -float("inf"), float("nan")
    v[1, 0, S - 1, 38] = float("inf")
    ops.paged_append(f.pages, f.table, f.past, k, v)
    now = [x[:, :, past:] for x in ops.paged_read(f.pages, f.table, f.past + S, past + S)]
    assert torch.equal(now[0], k) and torch.equal(now[1].isnan(), ~v.isfinite()) and torch.equal(now[1].nan_to_num(0), torch.where(v.isfinite(), v, 0))
    out = f.attn()
    assert out[1, :4, t:][..., [5, 38, 71]].isnan().all()
    for c in (5, 38, 71):
        out[1, :4, t:, c] = clean[1, :4, t:, c]
    assert torch.equal(out, clean)


def test_pools_past_4_gib(dev):
    """Byte offsets past 32 bits: the pages used are the last of a pool of 18000 pages of a quarter of a megabyte."""
    pages = alloc_pages(18000, 8, 256, "fp8")
    assert pages.k.numel() > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v, q = _randn(g, 1, 8, 300, 128), _randn(g, 1, 8, 300, 128), _randn(g, 1, 8, 300, 128)
    table = _ints(17999, 17500).view(1, 2)
    ops.paged_append(pages, table, _ints(0), k, v)
    small = alloc_pages(2, 8, 256, "fp8")
    ops.paged_append(small, _ints(0, 1).view(1, 2), _ints(0), k, v)
    kk, vv = tokens_of(small, [0, 1], 300)
    got_k, got_v = ops.paged_read(pages, table, _ints(300), 300)
    assert torch.equal(got_k[0].double(), kk) and torch.equal(got_v[0].double(), vv)
    for S in (1, 30, 100):
        out = ops.paged_attn(q[:, :, :S].contiguous(), pages, table, _ints(300 - S))
        want, tol = attention(q[0, :, :S], kk, vv, 300 - S, S, 128 ** -0.5)
        assert ((out[0].double() - want).abs() <= tol).all()


def test_equal_calls_give_equal_bits(dev):
    for S in (1, 2, 9, 40):
        f = Filled(28, 4, S, [5000, 33, 1200], page=64)
        first = f.attn()
        assert all(torch.equal(f.attn(), first) for _ in range(3))


def test_a_step_on_another_stream_and_two_at_once(dev):
    f, h = Filled(8, 2, 1, [3000, 70], page=64), Filled(8, 2, 1, [2000, 900], page=64, seed=5)
    want = f.attn(), h.attn()
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(one):
            a = f.attn()
        with torch.cuda.stream(two):
            b = h.attn()
        torch.cuda.synchronize()
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])


@pytest.mark.parametrize("S", [1, 9, 40])     # a wave's rows (one row tile; three), and rows through LDS
def test_a_captured_decoding_step(dev, S):
    """Append, attention and reading back in a graph: replayed while the lengths grow, with eager work on the same pages between the replays."""
    g = torch.Generator(device="cuda").manual_seed(9)
    B, Hq, Hkv, page, steps = 2, 8, 2, 32, 6
    pages = _garbage(alloc_pages(120, Hkv, page, "fp8"))
    table = _table(g, B, 55, 120)          # (room for more tokens than a single workgroup takes)
    past = _ints(60, 200)
    ops.paged_append(pages, table, _ints(0, 0), _randn(g, B, Hkv, 200, 128), _randn(g, B, Hkv, 200, 128), new_lens=past)
    q, k, v = _randn(g, B, Hq, S, 128), _randn(g, B, Hkv, S, 128), _randn(g, B, Hkv, S, 128)
    angle = torch.rand(B, S, 128, generator=g, device="cuda")
    cos, sin = angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)

    def step():
        q_rot, _ = ops.paged_append(pages, table, past, k, v, q=q, cos=cos, sin=sin)
        return q_rot, ops.paged_attn(q_rot, pages, table, past), *ops.paged_read(pages, table, past + S, 500)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q_rot, *out = step()
    for i in range(steps):
        for t in (q, k, v):
            t.copy_(_tokens(g, *t.shape))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        eager = step()[1:]                 # (the same tokens again: no scale grows, nothing is rounded anew)
        assert all(torch.equal(a, b) for a, b in zip(eager, got))
        for b, n in enumerate(past.tolist()):
            kk, vv = tokens_of(pages, table[b].tolist(), n + S)
            want, tol = attention(q_rot[b], kk, vv, n, S, 128 ** -0.5)
            assert ((got[0][b].double() - want).abs() <= tol).all(), (i, b)
            assert torch.equal(got[1][b, :, :n + S].double(), kk) and torch.equal(got[2][b, :, :n + S].double(), vv)
        past += S


def test_calls_without_the_native_module_give_the_same_bits(dev, monkeypatch):
    from pbs_attn_amd import _lib
    f = Filled(8, 2, 3, [700, 64], page=64)
    assert _lib.paged_host() is not _lib._no_paged_host
    assert _lib.paged_host().pages_ok(f.pages.k, f.pages.v, f.pages.k_scale, f.pages.v_scale) is True
    assert _lib.paged_host().read(f.pages, f.table, f.past, 700) is not None
    want, read = f.attn(softmax_scale=0.1, max_len=703), ops.paged_read(f.pages, f.table, f.past, 700)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, q, cos = _randn(g, 2, 2, 3, 128), _randn(g, 2, 8, 3, 128), _randn(g, 1, 3, 128)
    rotated_natively = ops.paged_append(f.pages, f.table, f.past, k, k, q=q, cos=cos, sin=cos, want_k=True)
    stored = ops.paged_read(f.pages, f.table, f.past + 3, 703)
    monkeypatch.setattr(_lib, "_paged_host", _lib._no_paged_host)
    again = ops.paged_append(f.pages, f.table, f.past, k, k, q=q, cos=cos, sin=cos, want_k=True)
    assert all(torch.equal(a, b) for a, b in zip(again, rotated_natively))
    assert all(torch.equal(a.nan_to_num(9), b.nan_to_num(9)) for a, b in zip(ops.paged_read(f.pages, f.table, f.past + 3, 703), stored))
    f2 = Filled(8, 2, 3, [700, 64], page=64)
    assert torch.equal(f2.attn(softmax_scale=0.1, max_len=703), want)
    assert all(torch.equal(a, b) for a, b in zip(ops.paged_read(f2.pages, f2.table, f2.past, 700), read))


def test_native_calls_refuse_what_the_general_path_refuses(dev):
    f = Filled(8, 2, 1, [70], page=64)
    p = f.pages
    for bad in [(p.k, p.v, None, None), (p.k, p.v, p.k_scale, None), (p.k, p.v.view(torch.uint8), p.k_scale, p.v_scale), (p.k.view(torch.uint8), p.v, p.k_scale, p.v_scale),
                (p.k, p.v, p.k_scale[:1], p.v_scale), (p.k, p.v, p.k_scale, p.v_scale[..., :1]), (p.k, p.v[:, :1], p.k_scale, p.v_scale),
                (p.k.view(torch.float8_e5m2), p.v.view(torch.float8_e5m2), p.k_scale, p.v_scale), (p.k, p.v, p.k_scale.cpu(), p.v_scale)]:
        with pytest.raises(ValueError):
            KVPages(*bad)
    p.v_scale = p.v_scale[:1]
    with pytest.raises(ValueError, match="pages are either"):
        ops.paged_attn(f.q, p, f.table, f.past)


def test_writing_to_a_lazy_copy_leaves_its_source(dev):
    pages = alloc_pages(2, 2, 32, "fp8")
    tensors = [pages.k, pages.v, pages.k_scale, pages.v_scale]
    for t in tensors:
        t.view(torch.uint8).zero_()
    copy = KVPages(*[torch._lazy_clone(t) for t in tensors])
    x = torch.ones(1, 2, 5, 128, dtype=torch.bfloat16, device=dev)
    ops.paged_append(copy, torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev), x, x)
    assert not any(t.view(torch.uint8).any() for t in tensors) and copy.k.view(torch.uint8).any() and copy.v.view(torch.uint8).any()
    assert block_of(copy, 0, 0, 0)[2].tolist() == [-8.0, -8.0]      # 1 is 256 of 2^-8
