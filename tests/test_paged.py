"""CPU: what the paged cache's entry points refuse, before anything reaches a GPU."""
import pytest
import torch

from pbs_attn_amd import _lib, ops
from pbs_attn_amd.paged import KVPages, alloc_pages

FAKE = 1 << 20


def _append(lib, **kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, cos=FAKE, sin=FAKE, q_out=FAKE, k_out=None, kp=FAKE, vp=FAKE, ks=None, vs=None, table=FAKE, past=FAKE, new=None,
             B=1, Hq=4, Hkv=2, S=1, D=128, pages=8, max_pages=4, size=64, bits=16, strides=[512, 128, 128] * 3, c=[128, 128], t=4)
    a.update(kw)
    return lib.pbs_paged_append(a["q"], a["k"], a["v"], a["cos"], a["sin"], a["q_out"], a["k_out"], a["kp"], a["vp"], a["ks"], a["vs"], a["table"],
                                a["past"], a["new"], a["B"], a["Hq"], a["Hkv"], a["S"], a["D"], a["pages"], a["max_pages"], a["size"], a["bits"],
                                *a["strides"], *a["c"], a["t"], None)


def _attn(lib, **kw):
    a = dict(q=FAKE, kp=FAKE, vp=FAKE, ks=None, vs=None, table=FAKE, past=FAKE, new=None, out=FAKE, B=1, Hq=4, Hkv=2, S=1, D=128, pages=8, max_pages=4,
             size=64, bits=16, max_len=256, strides=[512, 128, 128] * 2, t=4, scale=0.1, ws=FAKE, n=1 << 40)
    a.update(kw)
    return lib.pbs_paged_attn_fwd(a["q"], a["kp"], a["vp"], a["ks"], a["vs"], a["table"], a["past"], a["new"], a["out"], a["B"], a["Hq"], a["Hkv"], a["S"],
                                  a["D"], a["pages"], a["max_pages"], a["size"], a["bits"], a["max_len"], *a["strides"], a["t"], a["scale"], a["ws"],
                                  a["n"], None)


def _read(lib, **kw):
    a = dict(kp=FAKE, vp=FAKE, ks=None, vs=None, table=FAKE, lens=FAKE, k=FAKE, v=FAKE, B=1, Hkv=2, L=10, D=128, pages=8, max_pages=4, size=64, bits=16, t=4)
    a.update(kw)
    return lib.pbs_paged_read(a["kp"], a["vp"], a["ks"], a["vs"], a["table"], a["lens"], a["k"], a["v"], a["B"], a["Hkv"], a["L"], a["D"], a["pages"],
                              a["max_pages"], a["size"], a["bits"], a["t"], None)


POOL = [(dict(kp=None), b"null"), (dict(vp=None), b"null"), (dict(table=None), b"null"), (dict(D=64), b"head_dim"), (dict(bits=8), b"16 or 4 bits"),
        (dict(bits=4), b"scales"), (dict(bits=4, ks=FAKE), b"scales"), (dict(size=16), b"pages of"), (dict(size=96), b"pages of"),
        (dict(size=512), b"pages of"), (dict(B=0), b"shape"), (dict(Hkv=0), b"shape"), (dict(B=65536), b"shape"), (dict(pages=0), b"pages"),
        (dict(max_pages=0), b"pages"), (dict(max_pages=(1 << 24) + 1), b"2^30"), (dict(kp=FAKE + 8), b"aligned"), (dict(bits=4, ks=FAKE, vs=FAKE + 4), b"aligned")]


@pytest.mark.parametrize("call", [_append, _attn, _read])
def test_pools_that_no_call_takes(call):
    lib = _lib.load()
    for change, word in POOL:
        assert call(lib, **change) == -1 and word in lib.pbs_last_error(), (change, lib.pbs_last_error())


def test_arguments_that_the_library_refuses():
    lib = _lib.load()
    for change, word in [(dict(k=None), b"null"), (dict(v=None), b"null"), (dict(past=None), b"null"), (dict(q=None), b"q goes with q_out"),
                         (dict(q_out=None), b"q goes with q_out"), (dict(cos=None), b"cos goes with sin"), (dict(sin=None), b"cos goes with sin"),
                         (dict(S=0), b"shape"), (dict(S=(1 << 26) + 1), b"shape"), (dict(Hq=0), b"shape"), (dict(Hq=-1), b"shape"),
                         (dict(strides=[512, 128, 132] + [512, 128, 128] * 2), b"strides"), (dict(c=[0, 4]), b"strides"), (dict(k=FAKE + 2), b"aligned"),
                         (dict(k_out=FAKE + 8), b"aligned"), (dict(Hq=65535, Hkv=65535), b"too many heads")]:
        assert _append(lib, **change) == -1 and word in lib.pbs_last_error(), (change, lib.pbs_last_error())
    for change, word in [(dict(q=None), b"null"), (dict(out=None), b"null"), (dict(past=None), b"null"), (dict(S=0), b"shape"), (dict(Hq=5), b"shape"),
                         (dict(Hq=0), b"shape"), (dict(S=1 << 26, Hq=4, Hkv=1), b"too many query rows"), (dict(B=65535, Hq=65, Hkv=65), b"too many query rows"),
                         (dict(max_len=0), b"max_len"), (dict(max_len=5000, n=1000), b"workspace"), (dict(max_len=5000, ws=FAKE + 128), b"workspace"),
                         (dict(scale=0.0), b"softmax_scale"),
                         (dict(scale=-1.0), b"softmax_scale"), (dict(scale=float("nan")), b"softmax_scale"), (dict(scale=float("inf")), b"softmax_scale"),
                         (dict(strides=[512, 128, 128, 512, 128, 129]), b"strides"), (dict(q=FAKE + 8), b"aligned")]:
        assert _attn(lib, **change) == -1 and word in lib.pbs_last_error(), (change, lib.pbs_last_error())
    for change, word in [(dict(lens=None), b"null"), (dict(k=None), b"null"), (dict(v=None), b"null"), (dict(L=0), b"shape"), (dict(L=(1 << 28) + 1), b"shape"), (dict(v=FAKE + 8), b"aligned")]:
        assert _read(lib, **change) == -1 and word in lib.pbs_last_error(), (change, lib.pbs_last_error())


def test_a_workspace_does_not_grow_with_lengths_that_no_sequence_has():
    size = _lib.load().pbs_paged_attn_workspace_bytes
    for bits in (16, 4):
        most = size(2, 8, 2, 1, 128, bits, 1 << 30)
        assert 0 < most < 1 << 24 and size(2, 8, 2, 1, 128, bits, (1 << 31) - 1) == most
        assert size(2, 8, 2, 1, 128, bits, 0) == size(2, 8, 2, 1, 128, bits, -1) == 0


def test_pages_of_a_layer_have_one_of_two_forms():
    for form in ("bf16", "fp4"):
        for size in (32, 64, 128, 256):
            p = alloc_pages(3, 2, size, form, device="cpu")
            assert p.form == form and p.page_size == size and p.k.shape[:3] == (3, 2, size)
    b, f = alloc_pages(3, 2, 64, "bf16", "cpu"), alloc_pages(3, 2, 64, "fp4", "cpu")
    for bad in [(b.k.half(), b.v.half()), (b.k, b.k), (b.k, b.v, f.k_scale, f.v_scale), (f.k, f.v), (f.k, f.v, f.k_scale), (f.k, f.v, f.k_scale, f.v_scale[:2]),
                (b.k[0], b.v), (b.k[:, :, :48], b.v), (b.k[:0], b.v[:0]), (b.k[..., :64], b.v), (b.k[:, :1], b.v[:, :1]), (b.k.transpose(0, 1), b.v.transpose(0, 1))]:
        with pytest.raises(ValueError):
            KVPages(*bad)
    for bad in [dict(form="int4"), dict(page_size=16), dict(num_pages=0), dict(num_kv_heads=0)]:
        with pytest.raises(ValueError):
            alloc_pages(**{**dict(num_pages=2, num_kv_heads=2, device="cpu"), **bad})


def test_there_is_no_cpu_path():
    p = alloc_pages(3, 2, 64, "bf16", "cpu")
    x = torch.zeros(1, 2, 4, 128, dtype=torch.bfloat16)
    table, n = torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.paged_append(p, table, n, x, x), lambda: ops.paged_attn(x, p, table, n), lambda: ops.paged_read(p, table, n, 5)):
        with pytest.raises(_lib.PbsHipError, match="GPU"):
            call()
    with pytest.raises(AssertionError):
        ops.paged_append(p, table, n, x, x[:, :, :3])
    with pytest.raises(AssertionError):
        ops.paged_attn(x[..., :64], p, table, n)
    with pytest.raises(ValueError, match="cos goes with sin"):
        ops.paged_append(p, table, n, x, x, cos=x[0])


def _config(**kw):
    from transformers import LlamaConfig
    return LlamaConfig(**{**dict(hidden_size=512, num_attention_heads=4, num_key_value_heads=2, head_dim=128, num_hidden_layers=3), **kw})


def test_paged_cache_of_a_model():
    from pbs_attn_amd.patch.paged_cache import PagedKVCache
    cache = PagedKVCache(_config(), 2, 100, page_size=32, device="cpu")
    assert cache.page_table.shape == (2, 4) and len(cache.layers) == 3 and cache.layers[1].pages.k.shape == (8, 2, 32, 128)
    assert cache.get_seq_length() == 0 and cache.layers[2].get_mask_sizes(5) == (5, 0) and cache.layers[0].get_max_length() == 100
    assert cache.lengths(3) is cache.lengths(3) and cache.lengths(3).tolist() == [3, 3]
    cache.lengths(4), cache.lengths(5)
    assert len(cache._lengths) == 2 and cache.lengths(3).tolist() == [3, 3]
    assert PagedKVCache(_config(), 1, 100, form="fp4", device="cpu", num_kv_heads=1).layers[0].pages.k.shape == (2, 1, 64, 64)
    with pytest.raises(ValueError, match="2 sequences"):
        cache.layers[0].append(torch.zeros(1, 2, 1, 128), torch.zeros(1, 2, 1, 128))
    with pytest.raises(ValueError, match="the cache holds 100"):
        cache.layers[0].append(torch.zeros(2, 2, 101, 128), torch.zeros(2, 2, 101, 128))
    x = torch.zeros(2, 2, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(_lib.PbsHipError, match="GPU"):
        cache.update(x, x, 0)
    assert cache.get_seq_length() == 0     # nothing was stored
    with pytest.raises(NotImplementedError):
        cache.reorder_cache(torch.zeros(2, dtype=torch.long))
    for bad in [dict(config=_config(head_dim=64)), dict(batch_size=0), dict(max_len=0), dict(page_size=48), dict(form="int4")]:
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(config=_config(), batch_size=1, max_len=8, device="cpu"), **bad})


@pytest.mark.parametrize("kind", ["missing", "of another kind"])
def test_without_the_native_module_python_takes_every_call(kind, monkeypatch, tmp_path):
    path = tmp_path / "module.so"
    if kind != "missing":
        path.write_bytes(b"no module")
    monkeypatch.setattr(_lib, "PAGED_HOST_PATH", str(path))
    monkeypatch.setattr(_lib, "_paged_host", None)
    with pytest.warns(UserWarning, match="through Python"):
        host = _lib.paged_host()
    assert host.append() is None and host.attn() is None and host.read() is None and host.pages_ok() is None and _lib.paged_host() is host


def test_the_native_module_takes_plain_calls_only():
    import os
    if not os.path.exists(_lib.PAGED_HOST_PATH):
        from pbs_attn_amd.build import build_paged_host_module
        build_paged_host_module()
    host = _lib.paged_host()
    assert host is not _lib._no_paged_host
    p = alloc_pages(3, 2, 64, "bf16", "cpu")
    x, table, n = torch.zeros(1, 2, 4, 128, dtype=torch.bfloat16), torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    assert host.pages_ok(p.k, p.v, None, None) is False            # (not on the GPU)
    assert host.append(p, table, n, x, x, None, None, None, None, False) is None
    assert host.attn(x, p, table, n, None, None, None) is None and host.read(p, table, n, 5) is None
    assert host.append(*[None] * 10) is None and host.attn(*"abcdefg") is None and host.read(1, 2.0, "3", 4) is None
    for call in (host.append, host.attn, host.read, host.pages_ok):
        with pytest.raises(TypeError):
            call(p)
