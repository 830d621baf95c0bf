"""CPU: what a pool without scales is told."""
import pytest

from pbs_attn_amd import _lib
from tests.test_paged import FAKE, _append, _attn, _read


@pytest.mark.parametrize("call", [_append, _attn, _read])
def test_a_pool_of_8_bits_without_scales_is_told_so(call):
    lib = _lib.load()
    for scales in (dict(), dict(ks=FAKE), dict(vs=FAKE)):
        assert call(lib, bits=8, **scales) == -1 and lib.pbs_last_error().endswith(b"got 8 without them")
        assert call(lib, bits=4, **scales) == -1 and lib.pbs_last_error().endswith(b"a cache of 4 bits needs its scales")
        assert call(lib, bits=5, **scales) == -1 and lib.pbs_last_error().endswith(b"got 5")
