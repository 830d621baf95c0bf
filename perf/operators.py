"""The workloads that the paged key-value cache is timed on: writing new keys and values into it with the rotary embedding on
the way (``paged_append``), the attention of new tokens over it (``paged_attn``) and reading it back (``paged_read``).

A case is one attention layer.  ``op``:

``append``       rotary embedding of Q and K, K and V into the pages of a bf16 cache
``append_read``  the same into a 4-bit cache, which is then read back: what an attention over it will see
``attn``         attention of a batch's new tokens over the pages (bf16 or 4 bits); the tokens are in the cache already

Pages of P tokens, head-major: bf16 K as (page, head, token, 128), V as (page, head, token / 8, 128, token % 8).  In 4 bits a group
of 32 channels of a token and head shares a power of two, the smallest that leaves no value above 7 steps of one, held as its exponent +
127 in (page, head, token / 32, group, token % 32); values are e2m1 codes, two a byte: K as (page, head, token, 64), V as
(page, head, token / 4, 16 bytes' group, token % 4, 4).
"""
import math
import random

import torch

own = False

D = 128
CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _case(**kw):
    c = dict(op="attn", form="bf16", B=1, Hq=32, Hkv=8, S=1, past_min=0, past_max=0, ragged=False, page=64)
    c.update(kw)
    return c


def listed():
    return [
        # a chat's next token enters the cache: one token of one sequence, where the call's latency is all there is
        _case(name="append_chat_token", op="append", past_min=777, past_max=777),
        # a prompt of 8k tokens enters a fresh cache; its rotated keys also go on to the prefill attention
        _case(name="append_prompt_8k", op="append", S=8192, page=128),
        # a decoding step of 32 sequences with 4-bit pages
        _case(name="append4_batch32_token", op="append_read", form="fp4", B=32, Hq=28, Hkv=4, past_min=1, past_max=700, page=32),
        # four prompts padded to one length, two of them follow-ups, into 4-bit pages
        _case(name="append4_prompts_4k", op="append_read", form="fp4", B=4, Hq=28, Hkv=4, S=4001, past_min=0, past_max=600, ragged=True),
        # the next token of a chat of about a thousand tokens
        _case(name="attn_chat_token", past_min=1003, past_max=1003),
        # a decoding step of 64 sequences of very different lengths
        _case(name="attn_batch64_token", B=64, Hq=28, Hkv=4, past_min=17, past_max=8191),
        # the next token behind a prompt of 128k
        _case(name="attn_token_128k", past_min=131071, past_max=131071, page=128),
        # two follow-up prompts on filled caches
        _case(name="attn_followup_500", B=2, S=500, past_min=6000, past_max=16000, ragged=True),
        # the next token of a chat, 4-bit pages
        _case(name="attn4_chat_token", form="fp4", past_min=4100, past_max=4100),
        # a decoding step of a full server: 128 sequences with 4-bit pages
        _case(name="attn4_batch128_token", form="fp4", B=128, past_min=100, past_max=16383),
        # five drafted tokens of 16 sequences are checked at once
        _case(name="attn4_batch16_draft5", form="fp4", B=16, Hq=28, Hkv=4, S=5, past_min=1000, past_max=32000),
        # a follow-up prompt behind a document of 32k
        _case(name="attn4_followup_1000", form="fp4", S=1000, past_min=32768, past_max=32768, page=256),
    ]


def draw(rng):
    """One more case: either form, any page size and head grouping in use, one new token to a few thousand, an empty cache to 128k
    tokens; never more work than the largest listed case of its op."""
    spread = lambda lo, hi: int(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999))))  # noqa: E731
    form = rng.choice(["bf16", "fp4"])
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (28, 4), (8, 2), (4, 1), (16, 16)])
    page = rng.choice([32, 64, 64, 128, 256])
    if rng.random() < 0.35:
        B = spread(1, 64)
        S = 1 if rng.random() < 0.4 else spread(2, max(2, 8192 // B))
        past = spread(1, 1024) - 1
        return _case(op="append" if form == "bf16" else "append_read", form=form, B=B, Hq=Hq, Hkv=Hkv, S=S, past_min=past // 3,
                     past_max=past, ragged=rng.random() < 0.5, page=page)
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
    return _case(form=form, B=B, Hq=Hq, Hkv=Hkv, S=S, past_min=past // rng.choice([1, 3, 50]), past_max=past, ragged=rng.random() < 0.5, page=page)


def _lengths(case):
    """Tokens in the cache before the call, and new ones, of every sequence."""
    rng = random.Random(case["B"] * 1000003 + case["S"] * 1009 + case["past_max"])
    past = [rng.randint(case["past_min"], case["past_max"]) for _ in range(case["B"])]
    past[-1] = case["past_max"]
    new = [case["S"]] * case["B"]
    if case["ragged"]:
        new = [rng.randint((case["S"] + 1) // 2, case["S"]) for _ in range(case["B"])]
        new[0] = case["S"]
    return past, new


def prepare(case, seed):
    B, Hq, Hkv, S, P = case["B"], case["Hq"], case["Hkv"], case["S"], case["page"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
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
    # some channels of the keys are larger than others, as they are in trained models
    scale = torch.ones(D, device="cuda", dtype=torch.bfloat16)
    scale[5::19] = 3.0
    k_pool, v_pool = randn(pool, Hkv, P, D) * scale, randn(pool, Hkv, P, D)
    state = dict(table=table.cuda(), past=torch.tensor(past, dtype=torch.int32).cuda(), new=torch.tensor(new, dtype=torch.int32).cuda(),
                 total=torch.tensor(total, dtype=torch.int32).cuda(), longest=max(total), op=case["op"], k_scale=None, v_scale=None)
    if case["form"] == "bf16":
        state["k_pages"] = k_pool
        state["v_pages"] = v_pool.view(pool, Hkv, P // 8, 8, D).transpose(3, 4).contiguous()
    else:
        codes, exponents = _quantise(k_pool.float())
        state["k_pages"] = codes
        state["k_scale"] = exponents.view(pool, Hkv, P // 32, 32, 4).transpose(3, 4).contiguous()
        codes, exponents = _quantise(v_pool.float())
        state["v_pages"] = codes.view(pool, Hkv, P // 4, 4, 16, 4).transpose(3, 4).contiguous()
        state["v_scale"] = exponents.view(pool, Hkv, P // 32, 32, 4).transpose(3, 4).contiguous()
    if case["op"] == "attn":
        state["q"] = randn(B, Hq, S, D)
        return state
    # Q, K and V as the projections leave them: (batch, token, head, d) in memory
    for name, heads in (("q", Hq), ("k", Hkv), ("v", Hkv)):
        state[name] = randn(B, S, heads, D).transpose(1, 2)
    at = (state["past"].double()[:, None] + torch.arange(S, device="cuda").double())[..., None]
    angle = at * 500000.0 ** (-torch.arange(0, D, 2, device="cuda").double() / D)
    angle = torch.cat((angle, angle), dim=-1)
    state["cos"], state["sin"] = angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)
    return state


def _quantise(x):
    """Codes (.., 64) and exponents + 127 (.., 4) of float32 rows of 128 bf16 values."""
    groups = x.unflatten(-1, (4, 32))
    largest = groups.abs().amax(-1)
    field = (largest.to(torch.bfloat16).view(torch.int16).int() + 0x1F) >> 7    # up where the largest is above 1.75 * 2^n
    exponents = torch.where(largest.isfinite(), (field - 2).clamp(27, 252), 255)
    y = groups * torch.exp2(127.0 - exponents)[..., None]
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).to(torch.uint8)
    code = (code + 8 * torch.signbit(y)).to(torch.uint8).flatten(-2)
    return code[..., ::2] | (code[..., 1::2] << 4), exponents.to(torch.uint8)


def _values(codes, exponents):
    """Float32 rows of 128 from codes (.., 64) and exponents + 127 (.., 4)."""
    code = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    table = torch.tensor(CODES + tuple(-c for c in CODES), device=codes.device)
    scale = torch.where(exponents == 255, math.nan, torch.exp2(exponents.float() - 127.0))
    return (table[code.int()].unflatten(-1, (4, 32)) * scale[..., None]).flatten(-2)


def _read(s):
    """K and V of every sequence's pages in order, (batch, head, token, 128) float32."""
    k, v = s["k_pages"][s["table"]].transpose(1, 2), s["v_pages"][s["table"]].transpose(1, 2)
    if s["k_scale"] is None:
        return k.flatten(2, 3).float(), v.transpose(-1, -2).flatten(2, 4).float()
    ks, vs = (x[s["table"]].transpose(1, 2).transpose(-1, -2).flatten(2, 4) for x in (s["k_scale"], s["v_scale"]))
    return _values(k.flatten(2, 3), ks), _values(v.transpose(4, 5).flatten(5, 6).flatten(2, 4), vs)


def _rotate(x, cos, sin):
    x, cos, sin = x.float(), cos[:, None].float(), sin[:, None].float()
    return (x * cos + torch.cat((-x[..., D // 2:], x[..., :D // 2]), dim=-1) * sin).to(torch.bfloat16)


def _write(s, k, v):
    P = s["k_pages"].shape[2]
    i = torch.arange(k.shape[2], device="cuda")
    b, i = ((i[None] < s["new"][:, None]).nonzero(as_tuple=True))
    at = s["past"][b].long() + i
    page, at = s["table"][b, at // P].long(), at % P
    k, v = k[b, :, i], v[b, :, i]     # (tokens, head, 128)
    if s["k_scale"] is None:
        s["k_pages"][page, :, at] = k
        s["v_pages"][page, :, at // 8, :, at % 8] = v
        return
    codes, exponents = _quantise(k.float())
    s["k_pages"][page, :, at] = codes
    s["k_scale"][page, :, at // 32, :, at % 32] = exponents
    codes, exponents = _quantise(v.float())
    s["v_pages"][page, :, at // 4, :, at % 4] = codes.unflatten(-1, (16, 4))
    s["v_scale"][page, :, at // 32, :, at % 32] = exponents


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
    q, k = _rotate(s["q"], s["cos"], s["sin"]), _rotate(s["k"], s["cos"], s["sin"])
    _write(s, k, s["v"])
    if s["op"] == "append":
        return dict(q=q, k=k, k_pages=s["k_pages"], v_pages=s["v_pages"]) if q.shape[2] > 1 else dict(q=q, k_pages=s["k_pages"], v_pages=s["v_pages"])
    inside = torch.arange(s["longest"], device="cuda") < (s["past"] + s["new"])[:, None]
    k, v = (torch.where(inside[:, None, :, None], x[:, :, :s["longest"]], 0).to(torch.bfloat16) for x in _read(s))
    return dict(q=q, k=k, v=v)


def _own(s):
    from pbs_attn_amd import ops
    from pbs_attn_amd.paged import KVPages
    pages = KVPages(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
    if s["op"] == "attn":
        return ops.paged_attn(s["q"], pages, s["table"], s["past"], s["new"], max_len=s["longest"])
    prompt = s["op"] == "append" and s["q"].shape[2] > 1
    q, k = ops.paged_append(pages, s["table"], s["past"], s["k"], s["v"], q=s["q"], cos=s["cos"], sin=s["sin"], new_lens=s["new"], want_k=prompt)
    if s["op"] == "append":
        return dict(q=q, k=k, k_pages=pages.k, v_pages=pages.v) if prompt else dict(q=q, k_pages=pages.k, v_pages=pages.v)
    k, v = ops.paged_read(pages, s["table"], s["total"], s["longest"])
    return dict(q=q, k=k, v=v)


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    """Each new row in, its rotated row out, its place in the pages; the cache of the sequences' own lengths once; two products for every
    pair of a query and a key that it sees."""
    past, new = _lengths(case)
    Hq, Hkv, held = case["Hq"], case["Hkv"], 512 if case["form"] == "bf16" else 136     # bytes of a token's K and V in a page
    total = sum(past) + sum(new)
    if case["op"] == "attn":
        pairs = sum(n * p + n * (n + 1) / 2 for p, n in zip(past, new))
        return {"bytes": float(total * Hkv * held + 2 * sum(new) * Hq * 256), "flops": 4.0 * D * Hq * pairs}
    rows = case["B"] * case["S"]
    b = rows * (2 * Hq * 256 + Hkv * 512 + 512) + sum(new) * Hkv * held
    if case["op"] == "append_read":
        b += total * Hkv * held + case["B"] * max(p + n for p, n in zip(past, new)) * Hkv * 512
    elif case["S"] > 1:
        b += rows * Hkv * 256
    return {"bytes": float(b), "flops": 6.0 * rows * (Hq + Hkv) * D}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _exact_rotated(x, cos, sin):
    x, c, s = x.double(), cos.double().unsqueeze(1), sin.double().unsqueeze(1)
    lo, hi = x[..., :64], x[..., 64:]
    return torch.cat((lo * c[..., :64] - hi * s[..., :64], hi * c[..., 64:] + lo * s[..., 64:]), -1)


def _exact_held(x):
    """What 4 bits hold of rows of 128 (float64): the nearest of the levels, the even one of two as near."""
    g = x.reshape(*x.shape[:-1], 4, 32)
    largest = g.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(largest)                       # largest = m 2^e, m in [0.5, 1)
    e = torch.where(m > 0.875, e - 2, e - 3).clamp(-100, 125)
    y = torch.ldexp(g.abs(), -e)
    levels = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=x.device)                                     # even codes first: they win ties
    at = torch.tensor(CODES, device=x.device, dtype=torch.float64)[levels]
    best, far = torch.zeros_like(y), torch.full_like(y, math.inf)
    for level in at:
        d = (y - level).abs()
        best, far = torch.where(d < far, level, best), torch.minimum(d, far)
    return torch.ldexp(best, e).copysign(g).reshape(x.shape)


def _exact_cache(s, b, n):
    """K and V of sequence b's first n tokens, (head, n, 128) float64."""
    P = s["k_pages"].shape[2]
    at = torch.arange(n, device="cuda")
    page, at = s["table"][b].long()[at // P], at % P
    if s["k_scale"] is None:
        return s["k_pages"][page, :, at].double().transpose(0, 1), s["v_pages"][page, :, at // 8, :, at % 8].double().transpose(0, 1)
    out = []
    for codes, scale in ((s["k_pages"][page, :, at], s["k_scale"]), (s["v_pages"][page, :, at // 4, :, at % 4].flatten(2), s["v_scale"])):
        x = torch.empty(*codes.shape[:2], D, device="cuda", dtype=torch.float64)
        table = torch.tensor(CODES, device="cuda", dtype=torch.float64)
        for half in (0, 1):
            nibble = (codes >> (4 * half)).long() & 15
            x[..., half::2] = table[nibble & 7] * (1 - 2 * (nibble >> 3))
        e = scale[page, :, at // 32, :, at % 32].int() - 127
        out.append(torch.ldexp(x, e.repeat_interleave(32, dim=-1)).transpose(0, 1))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    past, new = _lengths(case)
    B, Hq, Hkv, S = case["B"], case["Hq"], case["Hkv"], case["S"]
    if case["op"] == "attn":
        out = torch.zeros(B, Hq, S, D, device="cuda", dtype=torch.float64)
        for b in range(B):
            k, v = _exact_cache(s, b, past[b] + new[b])
            hidden = torch.arange(past[b] + new[b], device="cuda") > torch.arange(past[b], past[b] + new[b], device="cuda")[:, None]
            for h in range(Hq):
                z = s["q"][b, h, :new[b]].double() @ k[h * Hkv // Hq].T / math.sqrt(D)
                z[hidden] = -math.inf
                out[b, h, :new[b]] = torch.softmax(z, -1) @ v[h * Hkv // Hq]
        return out
    q, k = _exact_rotated(s["q"], s["cos"], s["sin"]), _exact_rotated(s["k"], s["cos"], s["sin"])
    P = case["page"]
    if case["op"] == "append":
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        for b in range(B):
            at = torch.arange(past[b], past[b] + new[b], device="cuda")
            page, at = s["table"][b].long()[at // P], at % P
            k_pages[page, :, at] = k[b, :, :new[b]].transpose(0, 1)
            v_pages[page, :, at // 8, :, at % 8] = s["v"][b, :, :new[b]].double().transpose(0, 1)
        return dict(q=q, k=k, k_pages=k_pages, v_pages=v_pages) if S > 1 else dict(q=q, k_pages=k_pages, v_pages=v_pages)
    read_k = torch.zeros(B, Hkv, s["longest"], D, device="cuda", dtype=torch.float64)
    read_v = torch.zeros_like(read_k)
    for b in range(B):
        read_k[b, :, :past[b]], read_v[b, :, :past[b]] = _exact_cache(s, b, past[b])
        read_k[b, :, past[b]:past[b] + new[b]] = _exact_held(k[b, :, :new[b]].to(torch.bfloat16).double())
        read_v[b, :, past[b]:past[b] + new[b]] = _exact_held(s["v"][b, :, :new[b]].double())
    return dict(q=q, k=read_k, v=read_v)
