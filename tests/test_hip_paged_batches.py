"""GPU: batches of more sequences than a wave or a workgroup has lanes, one long sequence among short ones: the shares that workgroups take of them."""
import pytest
import torch

from tests.test_hip_paged import Filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["bf16", "fp4"])
@pytest.mark.parametrize("B,Hq,Hkv,S", [(65, 4, 2, 1), (130, 4, 1, 3), (130, 4, 2, 40), (256, 2, 1, 1), (257, 7, 1, 5), (600, 2, 1, 1), (600, 4, 1, 9)])
def test_many_sequences_one_of_them_long(dev, form, B, Hq, Hkv, S):
    g = torch.Generator().manual_seed(B)
    past = torch.randint(0, 100, (B,), generator=g).tolist()
    new = torch.randint(0, S + 1, (B,), generator=g).tolist()
    past[-1 - B // 9], new[-1 - B // 9] = 1400, S
    past[0], new[0], past[B // 2], new[B // 2], new[-1] = 0, 0, 0, S, 0
    f = Filled(form, Hq, Hkv, S, past, new, page=64, seed=B)
    out = f.attn()              # (the table has room for more tokens than a single workgroup takes)
    f.check(out)
    for b, n in enumerate(new):
        if n < S:
            assert not out[b, :, n:].any()
    assert f.attn().equal(out)
