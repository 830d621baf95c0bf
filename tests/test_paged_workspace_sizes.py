"""CPU: the workspace of an attention over a paged cache: one that was made for the largest call of a model serves every smaller one."""
import random
import re

import pytest
import torch

from pbs_attn_amd import _lib
from tests.test_paged import FAKE, _attn

LENGTHS = sorted({1, 31, 32, 33, *range(64, 6200, 64), *range(65, 6200, 448), 639, 640, 641, 999, 1000, 1001, 1099, 1100, 1101, 1279, 1280, 1281, 1599, 1600, 1601,
                  1999, 2000, 2001, 2699, 2700, 2701, *range(6200, 140000, 1531), 30000, 32768, 131072, 1 << 20, 1 << 30, (1 << 31) - 1})
BATCHES = [*range(1, 70), 96, 127, 128, 129, 160, 192, 255, 256, 257, 300, 511, 512, 513, 1000, 1025, 4096, 65535]
NEW = [*range(1, 70), 96, 128, 129, 200, 256, 257, 500, 1000, 1024, 4001, 8192, 65536]
HEADS = [(1, 1), (32, 8), (28, 4), (8, 2), (4, 1), (16, 16), (5, 1), (32, 1), (64, 64), (128, 8)]


def _falls(sizes):
    return [(a, b) for a, b in zip(sizes, sizes[1:]) if a[1] > b[1]]


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("Hq,Hkv", HEADS)
def test_the_size_never_falls(bits, Hq, Hkv):
    size = lambda B, S, n: _lib.load().pbs_paged_attn_workspace_bytes(B, Hq, Hkv, S, 128, bits, n)  # noqa: E731
    for S in (1, 2, 3, 5, 9, 16, 40, 500, 8192):
        for B in (1, 2, 8, 17, 64, 150, 1000):
            assert not _falls([(n, size(B, S, n)) for n in LENGTHS]), (S, B)
        for n in (640, 1000, 1101, 1300, 1700, 2500, 2800, 5000, 40000, 131072):
            assert not _falls([(B, size(B, S, n)) for B in BATCHES]), (S, n)
    for B in (1, 3, 16, 100):
        for n in (640, 1101, 1500, 2100, 5000, 131072):
            assert not _falls([(S, size(B, S, n)) for S in NEW]), (B, n)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_a_call_is_not_refused_a_larger_ones_workspace(bits):
    lib, rng = _lib.load(), random.Random(bits)
    for _ in range(400):
        Hq, Hkv = rng.choice(HEADS)
        B, S, n = rng.choice(BATCHES[:-2]), rng.choice(NEW), rng.choice(LENGTHS)
        room = lib.pbs_paged_attn_workspace_bytes(B, Hq, Hkv, S, 128, bits, n)
        b, s, m = rng.randint(1, B), rng.randint(1, S), rng.randint(1, n)
        need = lib.pbs_paged_attn_workspace_bytes(b, Hq, Hkv, s, 128, bits, m)
        assert need <= room, (B, S, n, b, s, m)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_the_size_holds_what_a_call_asks_for(bits):
    """Calls that are cut in any case: with no workspace at all they are refused, and the message says how much this very call needs."""
    if torch.cuda.is_available():
        pytest.skip("addresses of no memory")
    lib, rng, seen = _lib.load(), random.Random(bits + 1), set()
    scales = {} if bits == 16 else dict(ks=FAKE, vs=FAKE)
    for _ in range(1500):
        Hq, Hkv = rng.choice(HEADS)
        B, S, n = rng.choice(BATCHES), rng.choice(NEW), rng.choice([x for x in LENGTHS if 3300 < x < 1 << 28])
        if B * Hkv * ((S * (Hq // Hkv) + 15) // 16) >= 2048:
            continue
        assert _attn(lib, B=B, Hq=Hq, Hkv=Hkv, S=S, bits=bits, max_len=n, max_pages=1 << 20, size=256, n=0, **scales) == -1
        need = int(re.search(rb"workspace of (\d+) bytes", lib.pbs_last_error())[1])
        assert 0 < need <= lib.pbs_paged_attn_workspace_bytes(B, Hq, Hkv, S, 128, bits, n), (B, Hq, Hkv, S, n)
        seen.add(need)
    assert len(seen) > 10


def test_sizes_stay_small():
    """Two slots of 130 floats a row for each of 512 workers: 8.5 MB for 16 rows, 68 for 128, whatever the lengths."""
    size = _lib.load().pbs_paged_attn_workspace_bytes
    for bits in (16, 8, 4):
        assert size(65535, 32, 8, 1, 128, bits, (1 << 31) - 1) < 9 << 20
        assert size(65535, 32, 8, 8192, 128, bits, (1 << 31) - 1) < 69 << 20
        assert size(64, 32, 8, 8192, 128, bits, 600) == 0                    # (never cut)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_what_a_call_needs_is_named_and_less_is_refused(bits):
    lib = _lib.load()
    scales = {} if bits == 16 else dict(ks=FAKE, vs=FAKE)
    n = lib.pbs_paged_attn_workspace_bytes(1, 4, 2, 1, 128, bits, 4096)
    big = dict(bits=bits, max_pages=64, max_len=4096, t=64, **scales)
    assert n > 0 and _attn(lib, n=1000, **big) == -1 and b"workspace" in lib.pbs_last_error()
    assert _attn(lib, ws=None, n=n, **big) == -1 and b"workspace" in lib.pbs_last_error()
