"""GPU: what every layer of a patched model does on an 8-bit cache: the attention that reaches its output projection is that over what its pages hold, and they
hold its keys and values; a layer that is not patched gets them back."""
import pytest
import torch

from pbs_attn_amd import ops
from tests.paged_fp8_plain import BLOCK, block_of, held_after, tokens_of
from tests.paged_plain import attention, rotated, two_to
from tests.test_hip_paged_model import _patched

pytestmark = pytest.mark.gpu


def _check_keys(cache, layer, b, want, tol, pieces):
    """Each of at most `pieces` roundings is off by 2^-4 of a value or, near zero, by half of 2^-9 units."""
    n = want.shape[1]
    for t in range((n + BLOCK - 1) // BLOCK):
        size, row = cache.layers[layer].pages.page_size, cache.page_table[b].tolist()
        got, _, e = block_of(cache.layers[layer].pages, row[t * BLOCK // size], t % (size // BLOCK), 0)
        x, m = want[:, t * BLOCK:t * BLOCK + BLOCK], min(BLOCK, n - t * BLOCK)
        bound = tol[:, t * BLOCK:t * BLOCK + BLOCK] + pieces * (x.abs() * 2.0 ** -4 + 2.0 ** -10 * two_to(e)[:, None, None]) * 1.1
        assert ((got[:, :m] - x).abs() <= bound).all(), (layer, b, t)


@pytest.mark.parametrize("name,skip", [("llama31_8b", None), ("qwen25_7b", None), ("llama31_8b", [1]), ("llama31_8b", [0])])
def test_every_layers_attention(dev, monkeypatch, name, skip):
    from pbs_attn.patch.huggingface import get_paged_cache
    from pbs_attn_amd.ttft import build_model
    model = build_model(name, layers=2, device=dev)
    B, cuts = 2, [0, 300, 301, 302, 330, 331]
    ids = torch.randint(0, 1000, (B, cuts[-1]), generator=torch.Generator().manual_seed(3)).to(dev)
    _patched(model, skip)
    cache = get_paged_cache(model, B, 340, page_size=32, form="fp8")
    heads, kv_heads = model.config.num_attention_heads, model.config.num_key_value_heads
    queries, read, out = [], [], [None, None]
    k_rows, v_rows = [[], []], [[], []]
    split = lambda x: x.unflatten(-1, (-1, 128)).transpose(1, 2)  # noqa: E731
    for i, layer in enumerate(model.model.layers):
        at = layer.self_attn
        at.o_proj.register_forward_pre_hook(lambda _, args, i=i: out.__setitem__(i, split(args[0])))
        at.k_proj.register_forward_hook(lambda _, __, y, i=i: k_rows[i].append(split(y)))
        at.v_proj.register_forward_hook(lambda _, __, y, i=i: v_rows[i].append(split(y)))
    paged_attn, paged_read = ops.paged_attn, ops.paged_read
    monkeypatch.setattr(ops, "paged_attn", lambda q, *args, **kw: (queries.append(q.clone()), paged_attn(q, *args, **kw))[1])
    monkeypatch.setattr(ops, "paged_read", lambda *args: (read.append(paged_read(*args)), read[-1])[1])
    patched = [i for i in range(2) if i not in (skip or [])]
    for lo, hi in zip(cuts, cuts[1:]):
        if skip and 1 < hi - lo and lo:          # (an unpatched module's mask for several tokens on a filled cache is the module's own)
            steps = [(i, i + 1) for i in range(lo, hi)]
        else:
            steps = [(lo, hi)]
        for lo, hi in steps:
            queries.clear(), read.clear()
            with torch.no_grad():
                model(ids[:, lo:hi], past_key_values=cache)
            assert len(queries) == (len(patched) if lo else 0) and len(read) == len(skip or [])
            cos, sin = model.model.rotary_emb(out[0], torch.arange(hi, device=dev)[None])
            for i in range(2):
                pieces = len(k_rows[i])
                k_want, k_tol = rotated(torch.cat(k_rows[i], 2), cos, sin)
                for b in range(B):
                    k, v = tokens_of(cache.layers[i].pages, cache.page_table[b].tolist(), hi)
                    assert torch.equal(v, held_after([x[b] for x in v_rows[i]])), (i, b, hi)
                    # (an unpatched layer's keys are rotated in bf16, two roundings more)
                    _check_keys(cache, i, b, k_want[b], k_tol[b] + (0 if i in patched else 2.0 ** -6 * k_want[b].abs().amax()), pieces)
                    if i not in patched:
                        assert torch.equal(read[0][0][b].double(), k) and torch.equal(read[0][1][b].double(), v)
                    elif lo:
                        q = queries[patched.index(i)][b]
                        assert q.shape == (heads, hi - lo, 128) and k.shape[0] == kv_heads
                        want, tol = attention(q, k, v, lo, hi - lo, 128 ** -0.5)
                        assert ((out[i][b].double() - want).abs() <= tol).all(), (i, b, hi)
