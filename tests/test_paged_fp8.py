"""CPU: what the entry points of a paged cache refuse in 8 bits, before anything reaches a GPU."""
import pytest
import torch

from pbs_attn_amd import _lib, ops
from pbs_attn_amd.paged import KVPages, alloc_pages
from tests.test_paged import FAKE, _append, _attn, _config, _read

SCALES = dict(ks=FAKE, vs=FAKE)


@pytest.mark.parametrize("call", [_append, _attn, _read])
def test_pools_that_no_call_takes(call):
    lib = _lib.load()
    for change, word in [(dict(), b"8 with its scales"), (dict(ks=FAKE), b"8 with its scales"), (dict(vs=FAKE), b"8 with its scales"),
                         (dict(ks=FAKE, vs=FAKE + 8), b"aligned"), (dict(SCALES, kp=FAKE + 8), b"aligned"), (dict(SCALES, vp=None), b"null"),
                         (dict(SCALES, size=16), b"pages of"), (dict(SCALES, D=64), b"head_dim"), (dict(SCALES, table=None), b"null")]:
        assert call(lib, **{**dict(bits=8), **change}) == -1 and word in lib.pbs_last_error(), (change, lib.pbs_last_error())
    for bits in (0, 1, 7, 9, 32, -8):
        assert call(lib, bits=bits, **SCALES) == -1 and b"bits" in lib.pbs_last_error()


def test_arguments_that_the_library_refuses():
    lib = _lib.load()
    assert _attn(lib, bits=8, max_len=5000, n=1000, **SCALES) == -1 and b"workspace" in lib.pbs_last_error()
    assert _attn(lib, bits=8, scale=float("nan"), **SCALES) == -1 and b"softmax_scale" in lib.pbs_last_error()
    assert _append(lib, bits=8, S=0, **SCALES) == -1 and b"shape" in lib.pbs_last_error()
    assert _read(lib, bits=8, L=0, **SCALES) == -1 and b"shape" in lib.pbs_last_error()


def test_a_workspace_does_not_grow_with_lengths_that_no_sequence_has():
    size = _lib.load().pbs_paged_attn_workspace_bytes
    most = size(2, 8, 2, 1, 128, 8, 1 << 30)
    assert 0 < most < 1 << 24 and size(2, 8, 2, 1, 128, 8, (1 << 31) - 1) == most
    assert size(2, 8, 2, 1, 128, 8, 0) == size(2, 8, 2, 1, 128, 8, -1) == 0


def test_pages_of_a_layer_in_8_bits():
    for size in (32, 64, 128, 256):
        p = alloc_pages(3, 2, size, "fp8", device="cpu")
        assert p.form == "fp8" and p.bits == 8 and p.page_size == size and p.k.shape == (3, 2, size, 128) and p.v.shape == (3, 2, size // 8, 128, 8)
        assert p.k.dtype == p.v.dtype == torch.float8_e4m3fn and p.k_scale.shape == p.v_scale.shape == (3, 2, size // 32)
    assert alloc_pages(3, 2, 64, "bf16", "cpu").bits == 16 and alloc_pages(3, 2, 64, "fp4", "cpu").bits == 4
    p, b, f = (alloc_pages(3, 2, 64, form, "cpu") for form in ("fp8", "bf16", "fp4"))
    ks, vs = p.k_scale, p.v_scale
    for bad in [(p.k, p.v), (p.k, p.v, ks), (p.k, p.v, None, vs), (p.k, b.v, ks, vs), (b.k, p.v, ks, vs), (p.k.view(torch.uint8), p.v.view(torch.uint8), ks, vs),
                (p.k.view(torch.float8_e5m2), p.v.view(torch.float8_e5m2), ks, vs), (p.k, p.v, f.k_scale, f.v_scale), (p.k, p.v, ks[:2], vs), (p.k, p.v, ks, vs[..., :1]),
                (p.k, p.v, ks.float(), vs.float()), (p.k[..., :64], p.v, ks, vs), (p.k, p.k, ks, vs), (p.k[:, :1], p.v, ks, vs), (p.k[0], p.v, ks, vs),
                (p.k, p.v, ks.transpose(0, 1).contiguous().transpose(0, 1), vs), (f.k, f.v, ks, vs)]:
        with pytest.raises(ValueError):
            KVPages(*bad)


def test_there_is_no_cpu_path():
    p = alloc_pages(3, 2, 64, "fp8", "cpu")
    x = torch.zeros(1, 2, 4, 128, dtype=torch.bfloat16)
    table, n = torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.paged_append(p, table, n, x, x), lambda: ops.paged_attn(x, p, table, n), lambda: ops.paged_read(p, table, n, 5)):
        with pytest.raises(_lib.PbsHipError, match="GPU"):
            call()


def test_paged_cache_of_a_model_in_8_bits():
    from pbs_attn_amd.patch.paged_cache import PagedKVCache
    cache = PagedKVCache(_config(), 2, 100, page_size=32, form="fp8", device="cpu")
    assert cache.layers[1].pages.form == "fp8" and cache.layers[1].pages.k.shape == (8, 2, 32, 128)
    with pytest.raises(ValueError):
        PagedKVCache(_config(), 2, 100, form="fp8_e5m2", device="cpu")
