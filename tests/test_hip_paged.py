"""GPU: the paged cache against plain float64: what is written, what is read back, the attention over it."""
import pytest
import torch

from pbs_attn_amd import ops
from pbs_attn_amd.paged import KVPages, alloc_pages
from tests.paged_plain import attention, held_in_4_bits, rotated, tokens_in_page, tokens_of

pytestmark = pytest.mark.gpu
FORMS = ["bf16", "fp4"]


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def _garbage(pages):
    """What an earlier owner may have left in the pages: NaNs."""
    for t in (pages.k, pages.v, pages.k_scale, pages.v_scale):
        if t is not None:
            t.fill_(float("nan") if t.dtype == torch.bfloat16 else 255)
    return pages


def _table(g, B, slots, pool, device="cuda"):
    return torch.randperm(pool, generator=g, device=device)[:B * slots].view(B, slots).int()


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Filled:
    """A cache of B sequences with `past` tokens each, written by ops.paged_append, and the new tokens' Q, K and V appended."""

    def __init__(self, form, Hq, Hkv, S, past, new=None, page=64, seed=0, spare=3, slots=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        B = len(past)
        new = [S] * B if new is None else new
        slots = slots or max(1, max((p + n + page - 1) // page for p, n in zip(past, new)))
        self.pages = _garbage(alloc_pages(B * slots + spare, Hkv, page, form))
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

@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("B,Hq,Hkv,S,past,new,page", [
    (1, 4, 1, 1, [0], [1], 32),
    (1, 32, 8, 1, [777], [1], 64),
    (3, 8, 2, 1, [31, 32, 0], [1, 1, 0], 32),           # around a tile's border; one sequence without a new token
    (2, 28, 4, 33, [5, 64], [33, 20], 64),
    (3, 5, 5, 100, [0, 1, 250], [100, 0, 77], 256),
    (1, 7, 1, 300, [127], [300], 128),
    (1, 2, 2, 9, [3], [9], 64),                          # inside a tile, from the middle of one group of eight to the middle of another
])
def test_append_writes_what_its_layout_says(dev, form, B, Hq, Hkv, S, past, new, page):
    g = torch.Generator(device="cuda").manual_seed(S)
    slots = max((p + n + page - 1) // page for p, n in zip(past, new)) or 1
    pages = _garbage(alloc_pages(B * slots + 2, Hkv, page, form))
    before = [None if t is None else t.clone() for t in (pages.k, pages.v, pages.k_scale, pages.v_scale)]
    table = _table(g, B, slots, B * slots + 2)
    q, k, v = (_randn(g, B, S, H, 128).transpose(1, 2) for H in (Hq, Hkv, Hkv))   # as projections leave them
    angle = torch.rand(B, S, 64, generator=g, device="cuda").repeat(1, 1, 2) * 6.28
    cos, sin = angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)
    q_rot, k_rot = ops.paged_append(pages, table, _ints(*past), k, v, q=q, cos=cos, sin=sin, new_lens=_ints(*new), want_k=True)
    for got, x in ((q_rot, q), (k_rot, k)):
        want, tol = rotated(x, cos, sin)
        assert got.is_contiguous() and ((got.double() - want).abs() <= tol).all()
    touched = torch.zeros(pages.k.shape[0], pages.k.shape[2], dtype=torch.bool)
    for b in range(B):
        kk, vv = tokens_of(pages, table[b].tolist(), past[b] + new[b])
        want_k, want_v = k_rot[b, :, :new[b]], v[b, :, :new[b]]
        want_k, want_v = (want_k.double(), want_v.double()) if form == "bf16" else (held_in_4_bits(want_k), held_in_4_bits(want_v))
        assert torch.equal(kk[:, past[b]:], want_k) and torch.equal(vv[:, past[b]:], want_v)
        for t in range(past[b], past[b] + new[b]):
            touched[table[b, t // page], t % page] = True
    # nothing else was touched: the tokens before, behind and of other pages are what they were
    for index in range(pages.k.shape[0]):
        at = (~touched[index]).nonzero().flatten().cuda()
        for now, then in zip(tokens_in_page(pages, index, at), tokens_in_page(KVPages(*before), index, at)):
            assert torch.equal(now.nan_to_num(1e9), then.nan_to_num(1e9))


def test_append_without_rotation_or_queries(dev):
    g = torch.Generator(device="cuda").manual_seed(3)
    pages = alloc_pages(4, 2, 64, "bf16")
    k, v = _randn(g, 1, 2, 50, 128), _randn(g, 1, 2, 50, 128)
    assert ops.paged_append(pages, _ints(2, 1).view(1, 2), _ints(40), k, v) == (None, None)
    kk, vv = tokens_of(pages, [2, 1], 90)
    assert torch.equal(kk[:, 40:], k[0].double()) and torch.equal(vv[:, 40:], v[0].double())
    q, k_rot = ops.paged_append(pages, _ints(2, 1).view(1, 2), _ints(40), k, v, q=k, want_k=True)
    assert torch.equal(q, k) and torch.equal(k_rot, k)


def test_append_takes_strided_rows_and_broadcast_cosines(dev):
    g = torch.Generator(device="cuda").manual_seed(4)
    wide = _randn(g, 2, 70, 3 * 4 * 128 + 8)           # one projection for Q, K and V, rows padded
    q, k, v = (wide[..., i * 512:i * 512 + 512].unflatten(-1, (4, 128)).transpose(1, 2) for i in range(3))
    angle = torch.rand(1, 70, 128, generator=g, device="cuda") * 6.28
    cos, sin = angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)
    pages = alloc_pages(6, 4, 64, "bf16")
    table = torch.tensor([[0, 1, 9], [3, 4, 9]], dtype=torch.int32, device="cuda")[:, :2]   # rows further apart than they are long
    q_rot, k_rot = ops.paged_append(pages, table, _ints(0, 11), k, v, q=q, cos=cos, sin=sin, want_k=True)
    for got, x in ((q_rot, q), (k_rot, k)):
        want, tol = rotated(x, cos.expand(2, -1, -1), sin.expand(2, -1, -1))
        assert ((got.double() - want).abs() <= tol).all()
    odd = _randn(g, 2, 4, 70, 129)[..., :128]          # rows off their 16 bytes are copied first
    q2, k2 = ops.paged_append(pages, table, _ints(0, 11), odd, v, q=odd, cos=cos, sin=sin, want_k=True)
    assert torch.equal(q2, k2)
    kk, _ = tokens_of(pages, [3, 4], 81)
    assert torch.equal(kk[:, 11:], k2[1].double())


def test_4_bit_groups_at_the_edges_of_the_format(dev):
    """Zeros, signed zeros, ties of every level, the largest and smallest magnitudes, infinities and NaN, each in a group of its own."""
    tie = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 4.0])
    rows = []
    for scale in (1.0, 2.0 ** -100, 2.0 ** 124, 2.0 ** -7):
        rows.append(torch.cat((tie, tie)) * scale)
    for top in (7.0, 7.03125, 6.96875, 4.0, 8.0, 3.5, 1.75 * 2.0 ** 127, 1.99 * 2.0 ** 127, 2.0 ** -102, 2.0 ** -110, 2.0 ** -133):
        rows.append(torch.cat((torch.tensor([top]), torch.linspace(-1, 1, 31) * min(top, 2.0 ** 126))))
    rows += [torch.zeros(32), -torch.zeros(32)]
    for bad in (float("inf"), -float("inf"), float("nan")):
        rows.append(torch.cat((torch.ones(5), torch.tensor([bad]), torch.ones(26))))
    while len(rows) % 4:
        rows.append(torch.randn(32, generator=torch.Generator().manual_seed(1)))
    x = torch.stack(rows).view(1, 1, -1, 128).to(torch.bfloat16).cuda()
    n = x.shape[2]
    pages = alloc_pages(1, 1, 32, "fp4")
    ops.paged_append(pages, _ints(0).view(1, 1), _ints(3), x, x.flip(2))
    k, v = tokens_of(pages, [0], n + 3)
    want = held_in_4_bits(x[0])
    for got, w in ((k[:, 3:], want), (v[:, 3:], want.flip(1))):
        assert torch.equal(got.isnan(), w.isnan()) and torch.equal(got.nan_to_num(0), w.nan_to_num(0))
    k, v = ops.paged_read(pages, _ints(0).view(1, 1), _ints(n + 3), n + 3)
    assert torch.equal(k[0, :, 3:].isnan(), want.isnan()) and torch.equal(k[0, :, 3:].double().nan_to_num(0), want.nan_to_num(0))
    assert torch.equal(v[0, :, 3:].isnan(), want.flip(1).isnan()) and torch.equal(v[0, :, 3:].double().nan_to_num(0), want.flip(1).nan_to_num(0))


# ---- reading -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("page", [32, 64, 128, 256])
def test_read_gives_the_tokens_and_zeros_behind_them(dev, form, page):
    f = Filled(form, 3, 3, 5, [0, 28, 300, 64], page=page)
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

@pytest.mark.parametrize("form", FORMS)
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
def test_attention_over_the_pages(dev, form, Hq, Hkv, S, past, new, page):
    f = Filled(form, Hq, Hkv, S, past, new, page)
    f.check(f.attn())
    if S > 1:
        for b, n in enumerate(f.new_list):
            assert not f.attn()[b, :, n:].any()
    # a bound on the lengths changes how the work is cut, not what comes out
    f.check(f.attn(max_len=max(p + n for p, n in zip(f.past_list, f.new_list))))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("B,Hq,Hkv,S,past", [(1, 8, 2, 1, 40000), (2, 4, 1, 3, 33333), (40, 28, 4, 1, 900), (1, 32, 8, 200, 5000),
                                             # every number of row tiles, a few long sequences beside short ones
                                             (3, 28, 4, 3, 6000), (3, 28, 4, 5, 6000), (3, 28, 4, 9, 6000), (1, 28, 4, 9, 20000), (5, 28, 4, 20, 3000)])
def test_attention_over_long_caches_and_many_sequences(dev, form, B, Hq, Hkv, S, past):
    g = torch.Generator().manual_seed(B)
    pasts = [past] + [int(torch.randint(0, past, (1,), generator=g)) for _ in range(B - 1)]
    f = Filled(form, Hq, Hkv, S, pasts, page=64, seed=B)
    f.check(f.attn())
    f.check(f.attn(max_len=past + S, softmax_scale=0.02), scale=0.02)


@pytest.mark.parametrize("form", FORMS)
def test_attention_where_few_keys_weigh(dev, form):
    """Logits of hundreds: the largest exponent grows from tile to tile, most weights vanish."""
    f = Filled(form, 8, 2, 2, [700, 64], page=64)
    f.q = f.q * 16
    f.check(f.attn())


@pytest.mark.parametrize("form", FORMS)
def test_attention_reads_queries_where_they_are(dev, form):
    f = Filled(form, 8, 2, 3, [100, 37], page=64)
    q = f.q.transpose(1, 2).contiguous().transpose(1, 2)          # token-major
    assert torch.equal(ops.paged_attn(q, f.pages, f.table, f.past, f.new), f.attn())
    odd = torch.zeros(2, 8, 3, 129, dtype=torch.bfloat16, device="cuda")[..., 1:]
    odd.copy_(f.q)
    assert torch.equal(ops.paged_attn(odd, f.pages, f.table, f.past, f.new), f.attn())
    wide = torch.full((2, f.table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")   # a longer table; what is not reached is not read
    wide[:, :f.table.shape[1]] = f.table
    f.check(ops.paged_attn(f.q, f.pages, wide, f.past, f.new))
    assert torch.equal(ops.paged_attn(f.q, f.pages, f.table, f.past), f.attn())


@pytest.mark.parametrize("form", FORMS)
def test_pages_outside_the_pool_and_behind_the_table(dev, form):
    f = Filled(form, 8, 2, 2, [300, 10], page=64, slots=5)
    table = f.table.clone()
    table[0, 1], table[0, 3] = -1, f.pages.k.shape[0]              # tokens 64..127 and 192..255 of the first sequence are not there
    out = ops.paged_attn(f.q, f.pages, table, f.past, f.new)
    there = torch.ones(302, dtype=torch.bool, device="cuda")
    there[64:128] = there[192:256] = False
    k, v = tokens_of(f.pages, f.table[0].tolist(), 302)
    want, tol = attention(f.q[0], k, v, 300, 2, 128 ** -0.5, there)
    assert ((out[0].double() - want).abs() <= tol).all()
    assert torch.equal(out[1], f.attn()[1])
    k, v = ops.paged_read(f.pages, table, f.past + f.new, 302)
    assert not k[0, :, 64:128].any() and not v[0, :, 192:256].any() and k[0, :, 128:192].any()
    all_bad = torch.full_like(table, 1 << 30)
    assert not ops.paged_attn(f.q, f.pages, all_bad, f.past, f.new).any()
    # lengths past the end of the table: the tokens there do not exist
    short = f.table[:, :2].contiguous()
    out = ops.paged_attn(f.q, f.pages, short, f.past, f.new)
    k, v = tokens_of(f.pages, f.table[0].tolist(), 128)
    want, tol = attention(f.q[0], k, v, 126, 2, 128 ** -0.5)
    want[:, 0], tol[:, 0] = attention(f.q[0], k, v, 127, 1, 128 ** -0.5)[0][:, 0], tol[:, 1]    # both rows see all 128
    assert ((out[0].double() - want).abs() <= tol.amax(1, keepdim=True)).all()
    # writing: nothing happens to any page
    for t in (all_bad, short):
        before = [x.clone() for x in (f.pages.k, f.pages.v)]
        x = torch.ones(2, 2, 2, 128, dtype=torch.bfloat16, device="cuda")
        ops.paged_append(f.pages, t, _ints(300, 2 ** 31 - 1), x, x)
        assert torch.equal(f.pages.k.view(torch.uint8), before[0].view(torch.uint8)) and torch.equal(f.pages.v.view(torch.uint8), before[1].view(torch.uint8))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("S", [1, 20])
def test_sequences_that_share_their_first_pages(dev, form, S):
    """Three sequences behind the same 128 tokens, written once: each appends to pages of its own."""
    g = torch.Generator(device="cuda").manual_seed(S)
    pages = _garbage(alloc_pages(9, 2, 64, form))
    table = torch.tensor([[4, 7, 0], [4, 7, 2], [4, 7, 8]], dtype=torch.int32, device="cuda")
    ops.paged_append(pages, table[:1], _ints(0), _randn(g, 1, 2, 128, 128), _randn(g, 1, 2, 128, 128))
    k, v, q = _randn(g, 3, 2, S, 128), _randn(g, 3, 2, S, 128), _randn(g, 3, 8, S, 128)
    ops.paged_append(pages, table, _ints(128, 128, 128), k, v)
    out = ops.paged_attn(q, pages, table, _ints(128, 128, 128))
    for b in range(3):
        kk, vv = tokens_of(pages, table[b].tolist(), 128 + S)
        want, tol = attention(q[b], kk, vv, 128, S, 128 ** -0.5)
        assert ((out[b].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("S", [1, 20])
@pytest.mark.parametrize("past", [40, 3000])
def test_infinities_and_nans_reach_the_rows_that_see_them(dev, form, S, past):
    f = Filled(form, 8, 2, S, [past, past])
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
    if form == "fp4":                               # (the group is held as NaN)
        assert out[1, :4, -1].isnan().all()
    else:
        want = torch.where(f.q[1, :4, -1, 5:6] > 0, float("nan"), 0.0).expand(4, 128)   # weight exp(inf - inf), or exp(-inf)
        assert torch.equal(out[1, :4, -1].isnan(), want.isnan())


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("S,past", [(2, 0), (4, 40), (7, 3000), (11, 40), (11, 3000), (16, 40), (16, 3000), (40, 0), (40, 3000), (75, 1030)])   # 8 .. 300 rows
def test_values_that_are_not_finite_reach_no_earlier_row(dev, form, S, past):
    """Infinities and NaN among the new tokens' values: rows before them keep their bits, rows from them on get them."""
    f = Filled(form, 8, 2, S, [past, past])
    clean = f.attn()
    k, v = (x[:, :, past:].contiguous() for x in ops.paged_read(f.pages, f.table, f.past + S, past + S))
    t = S // 2
    v[1, 0, t, 5], v[1, 0, t, 38], v[1, 0, t, 71] = float("inf"), -float("inf"), float("nan")
    v[1, 0, S - 1, 38] = float("inf")
    ops.paged_append(f.pages, f.table, f.past, k, v)
    out = f.attn()
    if form == "bf16":
        seen, last = out[1, :4, t:S - 1] if t < S - 1 else None, out[1, :4, S - 1]
        if seen is not None:
            assert (seen[..., 5] == float("inf")).all() and (seen[..., 38] == -float("inf")).all() and seen[..., 71].isnan().all()
        assert (last[..., 5] == float("inf")).all() and last[..., 71].isnan().all()
        assert last[..., 38].isnan().all() if t < S - 1 else (last[..., 38] == float("inf")).all()
        touched = [5, 38, 71]
    else:                                           # (groups of 32 channels are held as NaN)
        seen = out[1, :4, t:]
        assert seen[..., :96].isnan().all()
        touched = range(96)
    for c in touched:
        out[1, :4, t:, c] = clean[1, :4, t:, c]
    assert torch.equal(out, clean)


def test_pools_past_4_gib(dev):
    """Byte offsets past 32 bits, element offsets past 31: the pages used are the last of a pool of 9000 pages of half a megabyte."""
    pages = alloc_pages(9000, 8, 256, "bf16")
    assert pages.k.numel() * 2 > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v, q = _randn(g, 1, 8, 300, 128), _randn(g, 1, 8, 300, 128), _randn(g, 1, 8, 300, 128)
    table = _ints(8999, 8500).view(1, 2)
    ops.paged_append(pages, table, _ints(100), k[:, :, 100:], v[:, :, 100:])
    ops.paged_append(pages, table, _ints(0), k[:, :, :100], v[:, :, :100])
    kk, vv = ops.paged_read(pages, table, _ints(300), 300)
    assert torch.equal(kk, k) and torch.equal(vv, v)
    out = ops.paged_attn(q[:, :, :1].contiguous(), pages, table, _ints(299))
    want, tol = attention(q[0, :, :1], k[0].double(), v[0].double(), 299, 1, 128 ** -0.5)
    assert ((out[0].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("form", FORMS)
def test_equal_calls_give_equal_bits(dev, form):
    f = Filled(form, 28, 4, 2, [5000, 33, 1200], page=64)
    first = f.attn()
    assert all(torch.equal(f.attn(), first) for _ in range(3))


@pytest.mark.parametrize("form", FORMS)
def test_a_step_on_another_stream_and_two_at_once(dev, form):
    f, h = Filled(form, 8, 2, 1, [3000, 70], page=64), Filled(form, 8, 2, 1, [2000, 900], page=64, seed=5)
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


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("S", [1, 9, 40])     # a wave's rows (one row tile; three), and rows through LDS
def test_a_captured_decoding_step(dev, form, S):
    """Append and attention in a graph: replayed while the lengths grow, with eager work on the same pages between the replays."""
    g = torch.Generator(device="cuda").manual_seed(9)
    B, Hq, Hkv, page, steps = 2, 8, 2, 32, 6
    pages = _garbage(alloc_pages(120, Hkv, page, form))
    table = _table(g, B, 55, 120)          # (room for more tokens than a single workgroup takes)
    past = _ints(60, 200)
    ops.paged_append(pages, table, _ints(0, 0), _randn(g, B, Hkv, 200, 128), _randn(g, B, Hkv, 200, 128), new_lens=past)
    q, k, v = _randn(g, B, Hq, S, 128), _randn(g, B, Hkv, S, 128), _randn(g, B, Hkv, S, 128)
    angle = torch.rand(B, S, 128, generator=g, device="cuda")
    cos, sin = angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)

    def step():
        q_rot, _ = ops.paged_append(pages, table, past, k, v, q=q, cos=cos, sin=sin)
        return q_rot, ops.paged_attn(q_rot, pages, table, past)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q_rot, out = step()
    for i in range(steps):
        for t in (q, k, v):
            t.copy_(_randn(g, *t.shape))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        eager = step()[1]
        assert torch.equal(eager, got)
        for b, n in enumerate(past.tolist()):
            kk, vv = tokens_of(pages, table[b].tolist(), n + S)
            want, tol = attention(q_rot[b], kk, vv, n, S, 128 ** -0.5)
            assert ((got[b].double() - want).abs() <= tol).all(), (i, b)
        past += S


@pytest.mark.parametrize("form", FORMS)
def test_calls_without_the_native_module_give_the_same_bits(dev, form, monkeypatch):
    from pbs_attn_amd import _lib
    f = Filled(form, 8, 2, 3, [700, 64], page=64)
    assert _lib.paged_host() is not _lib._no_paged_host
    want, read = f.attn(softmax_scale=0.1, max_len=703), ops.paged_read(f.pages, f.table, f.past, 700)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, q, cos = _randn(g, 2, 2, 3, 128), _randn(g, 2, 8, 3, 128), _randn(g, 1, 3, 128)
    rotated_natively = ops.paged_append(f.pages, f.table, f.past, k, k, q=q, cos=cos, sin=cos, want_k=True)
    stored = ops.paged_read(f.pages, f.table, f.past + 3, 703)
    monkeypatch.setattr(_lib, "_paged_host", _lib._no_paged_host)
    again = ops.paged_append(f.pages, f.table, f.past, k, k, q=q, cos=cos, sin=cos, want_k=True)
    assert all(torch.equal(a, b) for a, b in zip(again, rotated_natively))
    assert all(torch.equal(a.nan_to_num(9), b.nan_to_num(9)) for a, b in zip(ops.paged_read(f.pages, f.table, f.past + 3, 703), stored))
    f2 = Filled(form, 8, 2, 3, [700, 64], page=64)
    assert torch.equal(f2.attn(softmax_scale=0.1, max_len=703), want)
    assert all(torch.equal(a, b) for a, b in zip(ops.paged_read(f2.pages, f2.table, f2.past, 700), read))


def test_native_calls_refuse_what_the_general_path_refuses(dev):
    """The same messages, as the native call hands over what is not plain."""
    f = Filled("bf16", 8, 2, 1, [70], page=64)
    k = torch.zeros(1, 2, 1, 128, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="pages of 2 heads"):
        ops.paged_append(f.pages, f.table, f.past, k[:, :1], k[:, :1])
    with pytest.raises(ValueError, match="page_table"):
        ops.paged_attn(f.q, f.pages, f.table.long(), f.past)
    with pytest.raises(ValueError, match="lengths"):
        ops.paged_attn(f.q, f.pages, f.table, f.past.long())
    with pytest.raises(ValueError, match="lengths"):
        ops.paged_read(f.pages, f.table, f.past.cpu().repeat(2), 5)
    with pytest.raises(ValueError, match="tensors on cpu"):
        ops.paged_read(f.pages, f.table, f.past.cpu(), 5)
    with pytest.raises(ValueError, match="max_len"):
        ops.paged_read(f.pages, f.table, f.past, 0)
    from pbs_attn_amd._lib import PbsHipError
    with pytest.raises(PbsHipError, match="softmax_scale"):
        ops.paged_attn(f.q, f.pages, f.table, f.past, softmax_scale=-1.0)
    with pytest.raises(PbsHipError, match="max_len"):
        ops.paged_attn(f.q, f.pages, f.table, f.past, max_len=0)
    with pytest.raises(PbsHipError, match="bf16 only"):
        ops.paged_attn(f.q.float(), f.pages, f.table, f.past)
    with pytest.raises(AssertionError):
        ops.paged_attn(f.q[:, :7], f.pages, f.table, f.past)
    f.pages.v = f.pages.v[:1]
    with pytest.raises(ValueError, match="pages are either"):
        ops.paged_attn(f.q, f.pages, f.table, f.past)
