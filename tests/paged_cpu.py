"""The paged cache's operators in plain torch on the CPU, for the tests of what surrounds them, and a small model."""
import torch

from tests.paged_plain import attention, rotated, tokens_of


def append(pages, page_table, past_lens, k, v, q=None, cos=None, sin=None, new_lens=None, want_k=False):
    assert pages.form == "bf16" and new_lens is None
    if cos is not None:
        k = rotated(k, cos, sin)[0].to(torch.bfloat16)
        q = None if q is None else rotated(q, cos, sin)[0].to(torch.bfloat16)
    size = pages.page_size
    for b in range(k.shape[0]):
        for i in range(k.shape[2]):
            t = int(past_lens[b]) + i
            page, t = int(page_table[b, t // size]), t % size
            pages.k[page, :, t], pages.v[page, :, t // 8, :, t % 8] = k[b, :, i], v[b, :, i]
    return q, k if want_k else None


def attn(q, pages, page_table, past_lens, new_lens=None, softmax_scale=None, max_len=None):
    S = q.shape[2]
    out = []
    for b in range(q.shape[0]):
        past = int(past_lens[b])
        out.append(attention(q[b], *tokens_of(pages, page_table[b].tolist(), past + S), past, S, 128 ** -0.5)[0])
    return torch.stack(out).to(torch.bfloat16)


def read(pages, page_table, lens, max_len):
    found = [tokens_of(pages, page_table[b].tolist(), int(lens[b])) for b in range(len(lens))]
    return tuple(torch.stack([f[i] for f in found]).to(torch.bfloat16) for i in range(2))


def prefill(q, k, v):
    S = q.shape[2]
    return torch.stack([attention(q[b], k[b].double(), v[b].double(), 0, S, 128 ** -0.5)[0] for b in range(q.shape[0])]).to(torch.bfloat16)


prefill.native_gqa = True


def use(monkeypatch):
    from pbs_attn_amd import ops
    for name, fn in (("paged_append", append), ("paged_attn", attn), ("paged_read", read)):
        monkeypatch.setattr(ops, name, fn)


def model(skip=None, layers=2, patched=True, **kw):
    from transformers import LlamaConfig, LlamaForCausalLM

    from pbs_attn_amd.patch.huggingface import apply_patch_with_prefill
    torch.manual_seed(0)
    m = LlamaForCausalLM(LlamaConfig(**{**dict(hidden_size=256, intermediate_size=256, num_attention_heads=2, num_key_value_heads=1, head_dim=128,
                                               num_hidden_layers=layers, vocab_size=101, attn_implementation="sdpa"), **kw})).to(torch.bfloat16).eval()
    return apply_patch_with_prefill(m, prefill, skip) if patched else m
