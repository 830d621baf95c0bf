"""A paged cache in plain float64, for the tests: what the pages hold, value by value, and the attention over it."""
import math

import torch

LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def two_to(e):
    """2^e, exactly (a device's pow is not exact in float64)."""
    return torch.tensor([2.0 ** n for n in range(-128, 129)], dtype=torch.float64, device=e.device)[e.long() + 128]


def held_in_4_bits(x):
    """(.., 128) bf16 -> float64 values that a 4-bit cache holds of it, by brute force over the exponents and levels."""
    g = x.double().unflatten(-1, (4, 32))
    a = g.abs()
    bad = ~g.isfinite().all(-1, keepdim=True)
    largest = a.amax(-1, keepdim=True).nan_to_num(0.0, 0.0, 0.0)
    e = torch.full_like(largest, 125.0)
    for n in range(124, -101, -1):
        e = torch.where(largest <= 7 * 2.0 ** n, float(n), e)
    y = torch.where(bad, 0.0, a) / two_to(e)
    out = torch.zeros_like(y)
    for lo, hi, even_is_hi in ((0, 1, False), (1, 2, True), (2, 3, False), (3, 4, True), (4, 5, False), (5, 6, True), (6, 7, False)):
        half = (LEVELS[lo] + LEVELS[hi]) / 2
        out = torch.where((y >= half) if even_is_hi else (y > half), LEVELS[hi], out)
    out = out * two_to(e) * torch.where(g < 0, -1.0, 1.0)
    return torch.where(bad, math.nan, out).flatten(-2)


def tokens_in_page(pages, page, at):
    """K and V of tokens `at` (a tensor) of one page, (heads, tokens, 128) float64 each, straight from the layout's description."""
    page = torch.full_like(at, page)
    if pages.k_scale is None:
        k, v = pages.k[page, :, at].double(), pages.v[page, :, at // 8, :, at % 8].double()
        return k.transpose(0, 1), v.transpose(0, 1)
    found = []
    for codes, scale in ((pages.k[page, :, at], pages.k_scale), (pages.v[page, :, at // 4, :, at % 4].flatten(2), pages.v_scale)):
        nibbles = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
        table = torch.tensor(LEVELS + [-v for v in LEVELS], dtype=torch.float64, device=codes.device)
        e = scale[page, :, at // 32, :, at % 32].double().repeat_interleave(32, -1)
        found.append(torch.where(e == 255, math.nan, table[nibbles] * two_to(e - 127)).transpose(0, 1))
    return found


def tokens_of(pages, table_row, n):
    """The first n tokens of a sequence, (heads, n, 128) float64 K and V; zeros where the page is not in the pool."""
    heads, size = pages.k.shape[1:3]
    k = torch.zeros(heads, n, 128, dtype=torch.float64, device=pages.k.device)
    v = torch.zeros_like(k)
    for slot in range((n + size - 1) // size):
        page = int(table_row[slot]) if slot < len(table_row) else -1
        if 0 <= page < pages.k.shape[0]:
            m = min(size, n - slot * size)
            here = slice(slot * size, slot * size + m)
            k[:, here], v[:, here] = tokens_in_page(pages, page, torch.arange(m, device=pages.k.device))
    return k, v


def rotated(x, cos, sin):
    """(B, H, S, 128) in float64, and the bound of one fp32 sum and one rounding to bf16 around it."""
    x, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]
    turned = torch.cat((-x[..., 64:], x[..., :64]), -1)
    y = x * c + turned * s
    return y, y.abs() * 2.0 ** -8 + ((x * c).abs() + (turned * s).abs()) * 2.0 ** -24 * 1.01 + 1e-38


def attention(q, k, v, past, new, scale, there=None):
    """One sequence: q (Hq, S, 128), k and v (Hkv, past + new, 128) float64 -> output (Hq, S, 128) and the error that the kernels' roundings
    can add up to: weights and output to bf16 (half a step is 2^-8), logits and sums in fp32 (2^-24 an addition)."""
    Hq, S, _ = q.shape
    out, tol = torch.zeros(Hq, S, 128, dtype=torch.float64, device=q.device), torch.zeros(Hq, S, 128, dtype=torch.float64, device=q.device)
    n = past + new
    if new <= 0 or n <= 0:
        return out, tol
    group = Hq // k.shape[0]
    hidden = torch.arange(n, device=q.device) > past + torch.arange(new, device=q.device)[:, None]
    if there is not None:
        hidden = hidden | ~there[:n]
    for h in range(Hq):
        qh, kh, vh = q[h, :new].double(), k[h // group, :n], v[h // group, :n]
        z = (qh @ kh.T) * scale
        z = z.masked_fill(hidden, -math.inf)
        w = torch.softmax(z, -1)
        w = torch.where(hidden.all(-1, keepdim=True), 0.0, w)
        out[h, :new] = w @ vh
        # a logit is off by its fp32 sum (132 roundings of at most the sum of magnitudes) and by the scale's and the subtraction's rounding
        off = (132 * 2.0 ** -24 * (qh.abs() @ kh.abs().T) * scale + 2.0 ** -22 * z.abs().nan_to_num(0, 0, 0)).masked_fill(hidden, 0).amax(-1, keepdim=True)
        mass = w @ vh.abs()
        # weights: 2^-8, twice the logits' error (above and below the line), 2^-20 for the exponentials, the sums over n keys
        tol[h, :new] = mass * (2.0 ** -8 + 2.1 * off + 2.0 ** -20 + 2 * (n + 64) * 2.0 ** -24) + out[h, :new].abs() * 2.0 ** -8 + 1e-30
    return out, tol * 1.02   # (second-order terms)
