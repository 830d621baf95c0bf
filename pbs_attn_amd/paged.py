"""A paged key-value cache: the pages of a layer (``KVPages``, ``alloc_pages``), which ``ops.paged_append`` writes, ``ops.paged_attn``
attends to and ``ops.paged_read`` reads back, in bf16, 8 or 4 bits."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib

PAGE_SIZES = (32, 64, 128, 256)
HEAD_DIM = 128
FORMATS = ("bf16", "fp4", "fp8")
FP8 = torch.float8_e4m3fn


@dataclass
class KVPages:
    """One layer's pages of P tokens, head-major.

    bf16: ``k`` (pages, heads, P, 128), ``v`` (pages, heads, P / 8, 128, 8) with the eight tokens of a channel side by side.

    8 bits (``k`` and ``v`` float8_e4m3fn): their layouts as in bf16, and a power of two for 32 tokens of a head, as its exponent + 127:
    ``k_scale``, ``v_scale`` (pages, heads, P / 32) uint8.  Tokens that are appended to a block of 32 may take its power up, and those that it
    holds are then rounded anew: no call reads the block meanwhile, for a sequence that shares its page either.

    4 bits (``k_scale`` and ``v_scale`` given): uint8, two e2m1 codes a byte, the even channel in the low half: ``k`` (pages, heads, P, 64),
    ``v`` (pages, heads, P / 4, 16, 4, 4) = (token / 4, channel / 8, token % 4, byte), and a power of two for 32 channels of a token, as its
    exponent + 127: ``k_scale``, ``v_scale`` (pages, heads, P / 32, 4, 32) = (token / 32, channel / 32, token % 32)."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    def __post_init__(self):
        if self.k.is_cuda and (_lib._paged_host or _lib.paged_host()).pages_ok(self.k, self.v, self.k_scale, self.v_scale):
            return
        self.check()

    def check(self):
        """Raises ValueError where the tensors are not the pages of a layer."""
        k, v, ks, vs = self.k, self.v, self.k_scale, self.v_scale
        if k.dim() != 4 or k.shape[2] not in PAGE_SIZES:
            raise ValueError(f"pages are (pages, heads, tokens, channels) with {PAGE_SIZES} tokens, got {tuple(k.shape)}")
        n, h, p, last = k.shape
        if ks is None and vs is None:
            ok = k.dtype == v.dtype == torch.bfloat16 and last == HEAD_DIM and v.shape == (n, h, p // 8, HEAD_DIM, 8)
            tensors = (k, v)
        elif k.dtype == FP8:
            ok = (ks is not None and vs is not None and v.dtype == FP8 and ks.dtype == vs.dtype == torch.uint8 and last == HEAD_DIM
                  and v.shape == (n, h, p // 8, HEAD_DIM, 8) and ks.shape == vs.shape == (n, h, p // 32))
            tensors = (k, v, ks, vs)
        else:
            ok = (ks is not None and vs is not None and k.dtype == v.dtype == ks.dtype == vs.dtype == torch.uint8 and last == HEAD_DIM // 2
                  and v.shape == (n, h, p // 4, 16, 4, 4) and ks.shape == vs.shape == (n, h, p // 32, 4, 32))
            tensors = (k, v, ks, vs)
        if not ok or n == 0 or h == 0:
            raise ValueError("pages are either bf16 K (pages, heads, P, 128) and V (pages, heads, P / 8, 128, 8), or uint8 K (.., P, 64) and "
                             "V (.., P / 4, 16, 4, 4) with two scales (.., P / 32, 4, 32), or float8_e4m3fn in the shapes of bf16 with two uint8 "
                             "scales (.., P / 32)")
        for t in tensors:
            if not t.is_contiguous() or t.device != k.device or t.data_ptr() % 16:
                raise ValueError("the pages of a layer are contiguous, 16-byte aligned tensors on one device")

    @property
    def form(self) -> str:
        return "bf16" if self.k_scale is None else "fp8" if self.k.dtype == FP8 else "fp4"

    @property
    def bits(self) -> int:
        return {"bf16": 16, "fp8": 8, "fp4": 4}[self.form]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]


def alloc_pages(num_pages, num_kv_heads, page_size=64, form="bf16", device="cuda") -> KVPages:
    """Pages whose tokens are not written yet."""
    if form not in FORMATS:
        raise ValueError(f"Invalid form: {form}")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"pages of {PAGE_SIZES} tokens, got {page_size}")
    if num_pages <= 0 or num_kv_heads <= 0:
        raise ValueError("a pool has at least one page and one head")
    n, h, p = num_pages, num_kv_heads, page_size

    def empty(*shape, dtype=torch.uint8):
        return torch.empty(shape, dtype=dtype, device=device)
    if form == "bf16":
        return KVPages(empty(n, h, p, HEAD_DIM, dtype=torch.bfloat16), empty(n, h, p // 8, HEAD_DIM, 8, dtype=torch.bfloat16))
    if form == "fp8":
        return KVPages(empty(n, h, p, HEAD_DIM, dtype=FP8), empty(n, h, p // 8, HEAD_DIM, 8, dtype=FP8), empty(n, h, p // 32), empty(n, h, p // 32))
    return KVPages(empty(n, h, p, HEAD_DIM // 2), empty(n, h, p // 4, 16, 4, 4), empty(n, h, p // 32, 4, 32), empty(n, h, p // 32, 4, 32))
