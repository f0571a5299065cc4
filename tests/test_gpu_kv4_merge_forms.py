"""GPU tests that rows' records are merged to the same bits by 16 lanes a row (2048 rows and more) and by a workgroup a row."""
import pytest
import torch

from moe_fused_inference_amd import kv4
from tests.kv4_mask_helpers import Call

pytestmark = pytest.mark.gpu


# Sizes whose shares are as many as the sequences' lengths make, whatever the heads (four units each at least, and those of the
# line's places): twice the kv heads are the same shares, and rows enough for the other merge.
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("B,M,Hkv,G,D,S", [(1, 64, 4, 8, 128, 1024), (1, 64, 4, 8, 64, 1024), (4, 32, 2, 8, 128, 640), (4, 32, 2, 8, 64, 640)])
def test_both_merges_give_the_same_bits(B, M, Hkv, G, D, S, tree):
    half = Hkv // 2
    for dpos in ([S - M] * B, [S - M - 150 * b for b in range(B)], [-M] * (B - 1) + [S - M - 1]):
        c = Call(B, M, Hkv, G, D, 0, S, dpos, tree=tree)
        assert 2048 <= B * M * Hkv * G < 4096
        for dt in (torch.float32, torch.bfloat16):
            o = c.run(dt).view(B, M, 2, half * G, D)
            for h in range(2):
                cache = kv4.KV4(*(x[:, h * half:(h + 1) * half].contiguous() for x in c.cache))
                q = c.q.view(B, M, 2, half * G, D)[:, :, h].contiguous()
                assert torch.equal(o[:, :, h], c.run(dt, cache=cache, q=q))
