"""The workloads that a paged key-value cache in 8 bits is timed on: writing new keys and values into it with the rotary embedding on the way
(``paged_append``), reading it back (``paged_read``) and the attention of new tokens over it (``paged_attn``).

A case is one attention layer.  ``op``:

``append_read``  rotary embedding of Q and K, K and V into the pages, which are then read back: what an attention over them will see
``read``         the pages of a filled cache as bf16 tensors, for a layer with an attention of its own
``attn``         attention of a batch's new tokens over the pages; the tokens are in the cache already

Pages of P tokens, head-major: K (page, head, token, 128), V (page, head, token / 8, 128, token % 8), both e4m3 codes.  32 tokens of a head
(positions 32 t .. 32 t + 31 of the sequence) share a power of two for K and one for V, held as its exponent + 127 in
(page, head, token / 32): the smallest that leaves none of their finite values above 448 of it, between 2^-100 and 2^119.  Tokens
that join such a block later may take its power up, never down: the codes that are there then follow, rounded to nearest even once more.
"""
import math
import random

import torch

own = False

D = 128
T = 32      # tokens of a block
FP8 = torch.float8_e4m3fn


def _case(**kw):
    c = dict(op="attn", B=1, Hq=32, Hkv=8, S=1, past_min=0, past_max=0, ragged=False, page=64)
    c.update(kw)
    return c


def listed():
    return [
        # a chat's next token enters the cache, in the middle of a block: latency is all there is
        _case(name="append_chat_token", op="append_read", past_min=777, past_max=777),
        # a decoding step of 32 sequences
        _case(name="append_batch32_token", op="append_read", B=32, Hq=28, Hkv=4, past_min=1, past_max=700, page=32),
        # a prompt of 8k tokens enters a fresh cache; its rotated keys also go on to the prefill attention
        _case(name="append_prompt_8k", op="append_read", S=8192, page=128),
        # four prompts padded to one length, some of them follow-ups
        _case(name="append_prompts_4k", op="append_read", B=4, Hq=28, Hkv=4, S=4001, past_min=0, past_max=600, ragged=True),
        # a layer with an attention of its own gets a chat's cache of 1003 tokens
        _case(name="read_chat", op="read", past_min=1003, past_max=1003),
        # the same behind a document, two sequences of different lengths
        _case(name="read_2x32k", op="read", B=2, past_min=20000, past_max=32768, page=256),
        # the next token of a chat of about a thousand tokens
        _case(name="attn_chat_token", past_min=1003, past_max=1003),
        # a decoding step of 64 sequences of very different lengths
        _case(name="attn_batch64_token", B=64, Hq=28, Hkv=4, past_min=17, past_max=8191),
        # the next token behind a prompt of 128k
        _case(name="attn_token_128k", past_min=131071, past_max=131071, page=128),
        # a decoding step of a full server: 128 sequences
        _case(name="attn_batch128_token", B=128, past_min=100, past_max=16383),
        # five drafted tokens of 16 sequences are checked at once
        _case(name="attn_batch16_draft5", B=16, Hq=28, Hkv=4, S=5, past_min=1000, past_max=32000),
        # a follow-up prompt behind a document of 32k
        _case(name="attn_followup_1000", S=1000, past_min=32768, past_max=32768, page=256),
    ]


def draw(rng):
    """One more case: any page size and head grouping in use, one new token to a few thousand, an empty cache to 128k tokens; never more
    work than the largest listed one of its op."""
    spread = lambda lo, hi: int(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999))))  # noqa: E731
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (28, 4), (8, 2), (4, 1), (16, 16)])
    page = rng.choice([32, 64, 64, 128, 256])
    kind = rng.random()
    if kind < 0.35:
        B = spread(1, 64)
        S = 1 if rng.random() < 0.4 else spread(2, max(2, 8192 // B))
        past = spread(1, 1024) - 1
        return _case(op="append_read", B=B, Hq=Hq, Hkv=Hkv, S=S, past_min=past // 3, past_max=past, ragged=rng.random() < 0.5, page=page)
    if kind < 0.5:
        B = spread(1, 64)
        past = spread(1, max(1, 32768 * 2 * 8 // (B * Hkv)))
        return _case(op="read", B=B, Hq=Hq, Hkv=Hkv, past_min=past // rng.choice([1, 3, 50]), past_max=past, page=page)
    B = spread(1, 128)
    S = rng.choice([1, 1, 1, rng.randint(2, 8), spread(9, 1000)])
    past = spread(1, 131072) - 1
    while B * past * Hkv > 131072 * 8 or Hq * B * S * past > 32 * 1000 * 32768:
        if B > 1:
            B //= 2
        elif S > 1:
            S //= 2
        else:
            past //= 2
    return _case(B=B, Hq=Hq, Hkv=Hkv, S=S, past_min=past // rng.choice([1, 3, 50]), past_max=past, ragged=rng.random() < 0.5, page=page)


def _lengths(case):
    """Tokens in the cache before the call, and new ones, of every sequence (a case that reads has no new ones)."""
    rng = random.Random(case["B"] * 1000003 + case["S"] * 1009 + case["past_max"])
    past = [rng.randint(case["past_min"], case["past_max"]) for _ in range(case["B"])]
    past[-1] = case["past_max"]
    new = [0 if case["op"] == "read" else case["S"]] * case["B"]
    if case["ragged"]:
        new = [rng.randint((case["S"] + 1) // 2, case["S"]) for _ in range(case["B"])]
        new[0] = case["S"]
    return past, new


def prepare(case, seed):
    B, Hq, Hkv, S, P = case["B"], case["Hq"], case["Hkv"], case["S"], case["page"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    past, new = _lengths(case)
    total = [a + b for a, b in zip(past, new)]
    pages_of = [-(-t // P) for t in total]
    pool = sum(pages_of) + 3
    order = torch.randperm(pool, generator=g, device="cuda")    # a sequence's pages lie anywhere in the pool
    table = torch.zeros(B, max(pages_of), dtype=torch.int32)
    order, at = order.cpu().int(), 0
    for b, n in enumerate(pages_of):
        table[b, :n] = order[at:at + n]
        at += n
    # some channels of the keys are larger than others, and tokens differ in size, as they do in trained models
    scale = torch.ones(D, device="cuda")
    scale[5::19] = 3.0
    size = lambda *shape: randn(*shape, 1).mul_(0.3).exp_()  # noqa: E731
    state = dict(table=table.cuda(), past=torch.tensor(past, dtype=torch.int32).cuda(), new=torch.tensor(new, dtype=torch.int32).cuda(),
                 total=torch.tensor(total, dtype=torch.int32).cuda(), longest=max(total), op=case["op"], prompt=S > 1 and case["past_max"] == 0)
    codes, state["k_scale"] = _quantise((randn(pool, Hkv, P, D) * size(pool, Hkv, P) * scale).to(torch.bfloat16))
    state["k_pages"] = codes
    codes, state["v_scale"] = _quantise((randn(pool, Hkv, P, D) * size(pool, Hkv, P)).to(torch.bfloat16))
    state["v_pages"] = codes.view(torch.uint8).unflatten(2, (P // 8, 8)).transpose(3, 4).contiguous().view(FP8)
    if case["op"] == "read":
        return state
    if case["op"] == "attn":
        state["q"] = randn(B, Hq, S, D).to(torch.bfloat16)
        return state
    # Q, K and V as the projections leave them: (batch, token, head, d) in memory
    for name, heads in (("q", Hq), ("k", Hkv), ("v", Hkv)):
        x = randn(B, S, heads, D) * size(B, S, heads)
        state[name] = (x * scale if name == "k" else x).to(torch.bfloat16).transpose(1, 2)
    at = (state["past"].double()[:, None] + torch.arange(S, device="cuda").double())[..., None]
    angle = at * 500000.0 ** (-torch.arange(0, D, 2, device="cuda").double() / D)
    angle = torch.cat((angle, angle), dim=-1)
    state["cos"], state["sin"] = angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)
    return state


def _two_to(e):
    """2^e in float32 for whole numbers -126 .. 127, from its bits (a device's exp2 and ldexp are off by a last bit, which decides ties)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _power(largest):
    """Exponent + 127 of the smallest power of two with nothing above 448 of it, for magnitudes that are bf16 values."""
    field = largest.to(torch.bfloat16).view(torch.int16).int()
    return (((field + 0x1F) >> 7) - 8).clamp(27, 246)       # up where the largest is above 1.75 * 2^n


def _quantise(x):
    """Codes (.., tokens, 128) and exponents + 127 (.., tokens / 32) of bf16 rows."""
    blocks = x.unflatten(-2, (-1, T))
    a = blocks.abs()
    e = _power(torch.where(a.isfinite(), a, 0).amax((-1, -2)))
    y = blocks.float() * _two_to(127 - e)[..., None, None]
    return _codes(y).flatten(-3, -2), e.to(torch.uint8)


def _codes(y):
    return torch.where(y.isfinite(), y.clamp(-448, 448), math.nan).to(FP8)


def _read(s):
    """K and V of every sequence's pages in order, (batch, head, token, 128) float32."""
    out = []
    for codes, scale in ((s["k_pages"].view(torch.uint8)[s["table"]].transpose(1, 2).flatten(2, 3), s["k_scale"]),
                         (s["v_pages"].view(torch.uint8)[s["table"]].transpose(1, 2).transpose(-1, -2).flatten(2, 4), s["v_scale"])):
        power = _two_to(scale[s["table"]].transpose(1, 2).flatten(2, 3).int() - 127)
        out.append((codes.view(FP8).float().unflatten(2, (-1, T)) * power[..., None, None]).flatten(2, 3))
    return out


def _rotate(x, cos, sin):
    x, cos, sin = x.float(), cos[:, None].float(), sin[:, None].float()
    return (x * cos + torch.cat((-x[..., D // 2:], x[..., :D // 2]), dim=-1) * sin).to(torch.bfloat16)


def _write(s, k, v):
    """K and V into the blocks that they touch: each block whole, with the tokens that it holds already."""
    P, S = s["k_pages"].shape[2], k.shape[2]
    first = s["past"].long() // T
    t = first[:, None] + torch.arange((S + 2 * T - 2) // T, device="cuda")
    b, t = (t * T < (s["past"] + s["new"])[:, None]).logical_and((s["new"] > 0)[:, None]).nonzero(as_tuple=True)
    t = first[b] + t
    page, at = s["table"][b, t * T // P].long(), t % (P // T)
    i = (t * T)[:, None] + torch.arange(T, device="cuda") - s["past"].long()[b][:, None]        # the call's row at each place of a block
    fresh, before = (i >= 0) & (i < s["new"][b][:, None]), i < 0
    rows = i.clamp(0, S - 1)
    for x, name in ((k, "k"), (v, "v")):
        new = torch.where(fresh[:, None, :, None], x[b[:, None], :, rows].transpose(1, 2), 0)            # (blocks, head, 32, 128)
        a = new.abs()
        e = _power(torch.where(a.isfinite(), a, 0).amax((-1, -2)))
        scale, pages = s[name + "_scale"], s[name + "_pages"].view(torch.uint8)
        old = scale[page, :, at].int()
        e = torch.where(before.any(-1)[:, None], torch.maximum(e, old), e)
        # (heads whole: a view of the blocks of a pool)
        tiles = pages.unflatten(2, (-1, T)) if name == "k" else pages.unflatten(2, (-1, T // 8))
        held = tiles[page, :, at]
        held = held if name == "k" else held.transpose(-1, -2).flatten(2, 3)
        moved = _codes(held.view(FP8).float() * _two_to((old - e).clamp(min=-126))[..., None, None]).view(torch.uint8)
        written = _codes(new.float() * _two_to(127 - e)[..., None, None]).view(torch.uint8)
        held = torch.where(fresh[:, None, :, None], written, torch.where(before[:, None, :, None], moved, held))
        tiles[page, :, at] = held if name == "k" else held.unflatten(2, (T // 8, 8)).transpose(-1, -2)
        scale[page, :, at] = e.to(torch.uint8)


def _plain(s):
    if s["op"] == "attn":
        q = s["q"].float()
        B, Hq, S, _ = q.shape
        k, v = _read(s)
        Hkv, L = k.shape[1:3]
        logits = (q.reshape(B, Hkv, Hq // Hkv * S, D) @ k.transpose(-1, -2)).view(B, Hkv, Hq // Hkv, S, L)
        i, j = torch.arange(S, device="cuda"), torch.arange(L, device="cuda")
        seen = (j <= s["past"][:, None, None] + i[:, None]) & (i < s["new"][:, None])[..., None]
        seen = seen[:, None, None]
        logits = logits.mul_(D ** -0.5).masked_fill_(~seen, -math.inf)
        e = logits.sub_(logits.amax(-1, keepdim=True)).exp_()
        out = (e.view(B, Hkv, -1, L) @ v).view(B, Hkv, -1, S, D) / e.sum(-1, keepdim=True)
        return out.masked_fill_(~(i < s["new"][:, None])[:, None, None, :, None], 0).view(B, Hq, S, D).to(torch.bfloat16)
    out = {}
    if s["op"] == "append_read":
        out["q"], k = _rotate(s["q"], s["cos"], s["sin"]), _rotate(s["k"], s["cos"], s["sin"])
        _write(s, k, s["v"])
        if s["prompt"]:
            out["k_rotated"] = k
    inside = torch.arange(s["longest"], device="cuda") < s["total"][:, None]
    out["k"], out["v"] = (torch.where(inside[:, None, :, None], x[:, :, :s["longest"]], 0).to(torch.bfloat16) for x in _read(s))
    return out


def _own(s):
    from pbs_attn_amd import ops
    from pbs_attn_amd.paged import KVPages
    pages = KVPages(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
    if s["op"] == "attn":
        return ops.paged_attn(s["q"], pages, s["table"], s["past"], s["new"], max_len=s["longest"])
    out = {}
    if s["op"] == "append_read":
        out["q"], k = ops.paged_append(pages, s["table"], s["past"], s["k"], s["v"], q=s["q"], cos=s["cos"], sin=s["sin"], new_lens=s["new"],
                                       want_k=s["prompt"])
        if s["prompt"]:
            out["k_rotated"] = k
    out["k"], out["v"] = ops.paged_read(pages, s["table"], s["total"], s["longest"])
    return out


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    """Each new row in, its rotated row out, its place in the pages; the cache of the sequences' own lengths once; two products for every
    pair of a query and a key that it sees."""
    past, new = _lengths(case)
    Hq, Hkv, held = case["Hq"], case["Hkv"], 2 * D + 2 / T     # bytes of a token's K and V in a page
    total = sum(past) + sum(new)
    if case["op"] == "attn":
        pairs = sum(n * p + n * (n + 1) / 2 for p, n in zip(past, new))
        return {"bytes": total * Hkv * held + 2.0 * sum(new) * Hq * 256, "flops": 4.0 * D * Hq * pairs}
    out = case["B"] * max(p + n for p, n in zip(past, new)) * Hkv * 512
    if case["op"] == "read":
        return {"bytes": total * Hkv * held + out, "flops": 2.0 * total * Hkv * D}
    rows = case["B"] * case["S"]
    b = rows * (2 * Hq * 256 + Hkv * 512 + 512) + sum(new) * Hkv * held + total * Hkv * held + out
    if case["S"] > 1 and case["past_max"] == 0:
        b += rows * Hkv * 256
    return {"bytes": float(b), "flops": 6.0 * rows * (Hq + Hkv) * D}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _exact_rotated(x, cos, sin):
    x, c, s = x.double(), cos.double().unsqueeze(1), sin.double().unsqueeze(1)
    lo, hi = x[..., :64], x[..., 64:]
    return torch.cat((lo * c[..., :64] - hi * s[..., :64], hi * c[..., 64:] + lo * s[..., 64:]), -1)


def _exact_times(x, n):
    """x 2^n in float64."""
    return x * ((n.long() + 1023) << 52).view(torch.float64)


def _exact_exponent(x):
    """Of (.., 32, 128) float64: the smallest n with max <= 448 * 2^n, (..)."""
    m, e = torch.frexp(x.abs().flatten(-2).amax(-1))             # max = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    return torch.where(m > 0.875, e - 8, e - 9).clamp(-100, 119)


def _exact_rounded(x, n):
    """x as an e4m3 number times 2^n: 4 bits, the last of them worth 2^-9 at least."""
    y = _exact_times(x, -n)
    step = torch.frexp(y)[1].clamp(min=-5) - 4
    return _exact_times(torch.round(_exact_times(y, -step)), step + n)


def _exact_cache(s, b, n):
    """K and V of sequence b's first n tokens, (head, n, 128) float64, and their blocks' exponents, (head, blocks)."""
    P = s["k_pages"].shape[2]
    at = torch.arange(n, device="cuda")
    page, at = s["table"][b].long()[at // P], at % P
    out = []
    table = torch.empty(256, dtype=torch.float64)
    for code in range(256):
        e, m = code >> 3 & 15, code & 7
        value = math.nan if code & 127 == 127 else math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)
        table[code] = -value if code & 128 else value
    table = table.cuda()
    k, v = s["k_pages"].view(torch.uint8), s["v_pages"].view(torch.uint8)
    for codes, scale in ((k[page, :, at], s["k_scale"]), (v[page, :, at // 8, :, at % 8], s["v_scale"])):
        e = scale[page, :, at // T].int() - 127
        out.append(_exact_times(table[codes.long()], e[..., None]).transpose(0, 1))
        out.append(e[::T].T)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    past, new = _lengths(case)
    B, Hq, Hkv, S = case["B"], case["Hq"], case["Hkv"], case["S"]
    if case["op"] == "attn":
        out = torch.zeros(B, Hq, S, D, device="cuda", dtype=torch.float64)
        for b in range(B):
            k, _, v, _ = _exact_cache(s, b, past[b] + new[b])
            hidden = torch.arange(past[b] + new[b], device="cuda") > torch.arange(past[b], past[b] + new[b], device="cuda")[:, None]
            for h in range(Hq):
                z = s["q"][b, h, :new[b]].double() @ k[h * Hkv // Hq].T / math.sqrt(D)
                z[hidden] = -math.inf
                out[b, h, :new[b]] = torch.softmax(z, -1) @ v[h * Hkv // Hq]
        return out
    out = dict(k=torch.zeros(B, Hkv, s["longest"], D, device="cuda", dtype=torch.float64))
    out["v"] = torch.zeros_like(out["k"])
    fresh = {}
    if case["op"] == "append_read":
        out["q"], fresh["k"] = _exact_rotated(s["q"], s["cos"], s["sin"]), _exact_rotated(s["k"], s["cos"], s["sin"])
        if s["prompt"]:
            out["k_rotated"] = fresh["k"]
        fresh = dict(k=fresh["k"].to(torch.bfloat16).double(), v=s["v"].double())
    for b in range(B):
        k, k_e, v, v_e = _exact_cache(s, b, past[b])
        for name, held, exponents in (("k", k, k_e), ("v", v, v_e)):
            out[name][b, :, :past[b]] = held
            p = past[b]
            while p < past[b] + new[b]:      # block by block
                begin, end = p // T * T, min(p // T * T + T, past[b] + new[b])
                x = fresh[name][b, :, p - past[b]:end - past[b]]
                n = _exact_exponent(x)
                if begin < p:
                    n = torch.maximum(n, exponents[:, -1])
                    out[name][b, :, begin:p] = _exact_rounded(held[:, begin:p], n[:, None, None])
                out[name][b, :, p:end] = _exact_rounded(x, n[:, None, None])
                p = end
    return out
