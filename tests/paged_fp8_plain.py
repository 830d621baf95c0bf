"""A paged cache in 8 bits in plain float64, for the tests: what the pages hold, value by value, and what writing into them has to leave."""
import math

import torch

from pbs_attn_amd.paged import KVPages
from tests.paged_plain import two_to

BLOCK = 32


def code_values():
    """The 256 numbers of e4m3: sign, four bits of exponent (bias 7), three of fraction; all ones: NaN."""
    out = []
    for code in range(256):
        e, m = code >> 3 & 15, code & 7
        x = math.nan if code & 127 == 127 else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out.append(-x if code & 128 else x)
    return torch.tensor(out, dtype=torch.float64)


def rounded(y):
    """float64 -> the nearest e4m3 number, the one with an even code of two as near; 448 at most; NaN for what is not finite."""
    levels = code_values()[:127].to(y.device)
    at = torch.searchsorted(levels, y.abs().clamp(max=448.0).nan_to_num(0.0).contiguous()).clamp(max=126)
    below = (at - 1).clamp(min=0)
    a, lo, hi = y.abs().clamp(max=448.0), levels[below], levels[at]
    out = torch.where((a - lo < hi - a) | ((a - lo == hi - a) & (below % 2 == 0)), lo, hi)
    return torch.where(y.isfinite(), torch.where(torch.signbit(y), -out, out), math.nan)


def exponent_of(x):
    """(heads, tokens, 128) -> (heads): the least e from -100 to 119 with no finite magnitude above 448 * 2^e, by trying all."""
    a = x.double().abs()
    largest = torch.where(a.isfinite(), a, 0.0).flatten(1).amax(-1)
    e = torch.full_like(largest, 119.0)
    for n in range(118, -101, -1):
        e = torch.where(largest <= 448 * 2.0 ** n, float(n), e)
    return e


def block_of(pages, page, t, kv):
    """Block t of one page, K (kv 0) or V (1): its values as they stand (heads, 32, 128) float64, codes (uint8) and exponents (heads)."""
    at = torch.arange(BLOCK, device=pages.k.device) + t * BLOCK
    codes = pages.k.view(torch.uint8)[page, :, at] if kv == 0 else pages.v.view(torch.uint8)[page][:, at // 8, :, at % 8].transpose(0, 1)
    e = (pages.k_scale, pages.v_scale)[kv][page, :, t].double() - 127
    return code_values().to(codes.device)[codes.long()] * two_to(e)[:, None, None], codes, e


def tokens_of(pages, table_row, n):
    """The first n tokens of a sequence, (heads, n, 128) float64 K and V; zeros where the page is not in the pool."""
    heads, size = pages.k.shape[1:3]
    out = torch.zeros(2, heads, (n + BLOCK - 1) // BLOCK * BLOCK, 128, dtype=torch.float64, device=pages.k.device)
    for t in range(out.shape[2] // BLOCK):
        slot = t * BLOCK // size
        page = int(table_row[slot]) if slot < len(table_row) else -1
        if 0 <= page < pages.k.shape[0]:
            for kv in range(2):
                out[kv, :, t * BLOCK:(t + 1) * BLOCK] = block_of(pages, page, t % (size // BLOCK), kv)[0]
    return out[0, :, :n], out[1, :, :n]


def clone(pages):
    return KVPages(pages.k.clone(), pages.v.clone(), pages.k_scale.clone(), pages.v_scale.clone())


def check_append(before, after, table_row, past, k, v):
    """That `after` is `before` with k and v (heads, n, 128) as the tokens `past` .. of a sequence: its blocks, to the bit of value and scale, and the codes
    behind its last token as they were.  Returns the (page, block) that it looked at."""
    size, n, seen = before.k.shape[2], k.shape[1], set()
    for t in range(past // BLOCK, (past + n + BLOCK - 1) // BLOCK):
        slot = t * BLOCK // size
        page = int(table_row[slot]) if slot < len(table_row) else -1
        if not 0 <= page < before.k.shape[0]:
            continue
        seen.add((page, t % (size // BLOCK)))
        lo, hi = max(past - t * BLOCK, 0), min(past + n - t * BLOCK, BLOCK)     # places of the block that are written
        for kv, x in enumerate((k, v)):
            new = x[:, t * BLOCK + lo - past:t * BLOCK + hi - past].double()
            old, codes, e_old = block_of(before, page, t % (size // BLOCK), kv)
            e = exponent_of(new)
            if lo > 0:
                e = torch.maximum(e, e_old)
            got, codes_now, e_now = block_of(after, page, t % (size // BLOCK), kv)
            assert torch.equal(e_now, e), (page, t, kv)
            unit = two_to(e)[:, None, None]
            for want, have in ((rounded(new / unit) * unit, got[:, lo:hi]), (rounded(old[:, :lo] / unit) * unit, got[:, :lo])):
                assert torch.equal(want.isnan(), have.isnan()) and torch.equal(want.nan_to_num(0), have.nan_to_num(0)), (page, t, kv)
            assert torch.equal(codes_now[:, hi:], codes[:, hi:]), (page, t, kv)
    return seen


def check_untouched(before, after, touched):
    """That every block but those of `touched` is what it was, to the bit."""
    for page in range(before.k.shape[0]):
        for t in range(before.k.shape[2] // BLOCK):
            if (page, t) not in touched:
                for kv in range(2):
                    (_, a, e), (_, b, f) = block_of(before, page, t, kv), block_of(after, page, t, kv)
                    assert torch.equal(a, b) and torch.equal(e, f), (page, t, kv)


def held_after(pieces):
    """What a cache that is empty holds of tokens that come in pieces (heads, n, 128): (heads, all, 128) float64."""
    out, e_now = torch.zeros(pieces[0].shape[0], 0, 128, dtype=torch.float64, device=pieces[0].device), None
    for x in pieces:
        x = x.double()
        while x.shape[1]:
            at = out.shape[1] % BLOCK
            new, x = x[:, :BLOCK - at], x[:, BLOCK - at:]
            e = exponent_of(new)
            if at:
                e = torch.maximum(e, e_now)
            unit, before = two_to(e)[:, None, None], out.shape[1] - at
            out = torch.cat((out[:, :before], rounded(out[:, before:] / unit) * unit, rounded(new / unit) * unit), 1)
            e_now = e
    return out
