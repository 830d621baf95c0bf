"""A paged key-value cache for patched Hugging Face models: ``model(ids, past_key_values=PagedKVCache(...))``, ``model.generate(...)``.

A patched layer (``apply_patch_with_prefill``) that is handed this cache writes its keys and values into the pages with the rotary embedding
on the way.  The first prompt's attention is the prefill function's; single tokens and later prompts attend to the pages
(``ops.paged_attn``), where the reference sends single tokens to the module's original forward and lets a later prompt attend to itself
alone (pbs_attn/patch/huggingface.py:169-241).  Layers that are not patched (``skip_layers``) read their keys and values back (``update``).

All sequences of a batch have one length, as the module's inputs have: there is no padding.  A mask that hides anything a causal one does not is
refused (``check_mask``), and so are models with sliding windows.  The lengths are the host's: a program that captures its decoding step into a graph calls
``ops.paged_append`` and ``ops.paged_attn`` with lengths of its own on the GPU."""
from __future__ import annotations

import torch
from transformers.cache_utils import Cache, CacheLayerMixin

from pbs_attn_amd import ops
from pbs_attn_amd.paged import HEAD_DIM, PAGE_SIZES, alloc_pages


def check_mask(mask, past, new):
    """Raises ValueError unless a module's attention mask says what the attention on a paged cache does: the first of ``new`` queries sees
    ``past + 1`` keys, each one after it one more.  None says so, and a mask of (batch, keys) of ones, and one of (batch, heads, queries, keys)
    that is causal, of truth values or added to the logits; columns behind the last key are not looked at.  Reads the mask on the host."""
    if mask is None:
        return
    n = past + new
    fits = False
    if isinstance(mask, torch.Tensor) and mask.dim() in (2, 4) and mask.shape[-1] >= n:
        if mask.dim() == 2:
            fits = mask[:, :n].all()
        elif mask.shape[2] == new:
            fits = torch.ones((), dtype=torch.bool, device=mask.device)
            keys = torch.arange(n, device=mask.device)
            for i in range(0, new, 1024):       # (a prompt's mask is large)
                rows = mask[:, :, i:i + 1024, :n]
                seen = keys <= torch.arange(past + i, past + i + rows.shape[2], device=mask.device)[:, None]
                same = rows == seen if rows.dtype == torch.bool else (rows == 0) == seen
                fits &= same.all()
    if not fits:
        raise ValueError("a paged cache attends causally to all that is cached: no padding, windows or other masks")


class _Sequences:
    """What the layers of a cache share: their number, the tokens that each has room for, their pages and lengths.  (It knows neither the
    cache nor its layers: in a cycle the pages would stay until the collector's next pass.)"""

    def __init__(self, count, room, page_size, device):
        slots = (room + page_size - 1) // page_size
        self.count, self.room = count, room
        self.page_table = torch.arange(count * slots, dtype=torch.int32, device=device).view(count, slots)
        self.kept = {}

    def lengths(self, n):
        """``n`` for every sequence, on the GPU; the last two are kept, as all layers of a step ask for the same.  A tensor is used on the
        stream that filled it only: there its memory may be given away while the last call that reads it is still to come."""
        stream = 0
        if self.page_table.is_cuda:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a paged cache's lengths are the host's and cannot be captured: capture ops.paged_append and ops.paged_attn")
            stream = torch._C._cuda_getCurrentRawStream(self.page_table.device.index)
        key = (n, stream)
        if key not in self.kept:
            if len(self.kept) >= 2:
                del self.kept[next(iter(self.kept))]
            self.kept[key] = torch.full((self.count,), n, dtype=torch.int32, device=self.page_table.device)
        return self.kept[key]


class _PagedLayer(CacheLayerMixin):
    def __init__(self, sequences, pages):
        super().__init__()
        self.sequences, self.pages, self.length = sequences, pages, 0
        self.is_initialized = True

    def lazy_initialization(self, key_states, value_states):
        pass

    def append(self, k, v, **rotation):
        """New tokens k, v (batch, heads, S, 128) behind those that are there; the arguments and results of ``ops.paged_append``."""
        s = self.sequences
        if k.shape[0] != s.count:
            raise ValueError(f"a cache of {s.count} sequences, {k.shape[0]} given")
        if self.length + k.shape[2] > s.room:
            raise ValueError(f"{self.length} + {k.shape[2]} tokens, and the cache holds {s.room}")
        rotated = ops.paged_append(self.pages, s.page_table, s.lengths(self.length), k, v, **rotation)
        self.length += k.shape[2]
        return rotated

    def attention(self, q):
        """Of the last tokens, appended before: q (batch, heads, S, 128)."""
        past = self.length - q.shape[2]
        return ops.paged_attn(q, self.pages, self.sequences.page_table, self.sequences.lengths(past), max_len=self.length)

    def update(self, key_states, value_states, *args, **kwargs):
        """For modules with an attention of their own: stores the (rotated) keys and the values, and returns all of them."""
        self.append(key_states, value_states)
        return ops.paged_read(self.pages, self.sequences.page_table, self.sequences.lengths(self.length), self.length)

    def get_mask_sizes(self, query_length, *args):
        return self.length + query_length, 0

    def get_seq_length(self, *args):
        return self.length

    def get_max_length(self):
        return self.sequences.room

    get_max_cache_shape = get_max_length

    def reset(self):
        self.length = 0

    def crop(self, tokens_to_remove):
        """Takes that many tokens (negative: -3 for the last three) off the end; a positive number is how many stay, as the library's own
        caches still have it."""
        n = tokens_to_remove
        self.length = max(self.length + n, 0) if n <= 0 else min(self.length, n)

    def reorder_cache(self, beam_idx):
        raise NotImplementedError("a paged cache does not reorder, repeat or drop its sequences")

    batch_select_indices = batch_repeat_interleave = reorder_cache


class PagedKVCache(Cache):
    """Room for ``batch_size`` sequences of up to ``max_len`` tokens of a model with ``config``, in pages of ``page_size`` tokens, bf16,
    8 bits (``form="fp8"``: half of the memory and of a decoding step's traffic) or 4 bits (``form="fp4"``: about a quarter); the first prompt's own
    attention still sees bf16.  In 8 bits a block of 32 tokens keeps the scale that its largest value asked for, also of tokens that ``crop`` took off
    again (looked-up or drafted ones that were rejected): those that stay, and those after them, are then held as coarsely as that value made them.
    ``num_kv_heads``: of this process, where it is not the configuration's (tensor parallel)."""

    is_paged = True

    def __init__(self, config, batch_size, max_len, page_size=64, form="bf16", device="cuda", num_kv_heads=None):
        head_dim = getattr(config, "head_dim", None) or config.hidden_size // config.num_attention_heads
        if head_dim != HEAD_DIM:
            raise ValueError(f"a paged cache holds heads of {HEAD_DIM}, not {head_dim}")
        if batch_size <= 0 or max_len <= 0:
            raise ValueError("a cache holds at least one sequence of at least one token")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"pages of {PAGE_SIZES} tokens, got {page_size}")
        kinds = getattr(config, "layer_types", None)
        if any(kind != "full_attention" for kind in kinds) if kinds else getattr(config, "use_sliding_window", False):
            raise ValueError("a layer on a paged cache attends to all that is cached, and this model has layers with sliding windows")
        heads = num_kv_heads or config.num_key_value_heads
        self._shared = shared = _Sequences(batch_size, max_len, page_size, device)
        super().__init__(layers=[_PagedLayer(shared, alloc_pages(shared.page_table.numel(), heads, page_size, form, device))
                                 for _ in range(config.num_hidden_layers)])

    sequences = property(lambda self: self._shared.count)
    room = property(lambda self: self._shared.room)
    page_table = property(lambda self: self._shared.page_table)
    _lengths = property(lambda self: self._shared.kept)

    def lengths(self, n):
        """``n`` for every sequence, on the GPU."""
        return self._shared.lengths(n)
