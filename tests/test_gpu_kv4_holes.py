"""GPU test of values that are not finite beside a hole of the page table (kv4.py)."""
import numpy as np
import pytest
import torch

from moe_fused_inference_amd import kv4
from tests.gpu_helpers import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,G,hole", [(3, 4, 1), (3, 4, 2), (5, 8, 1), (40, 2, 4)])
def test_an_infinite_value_beside_a_hole(M, G, hole, D):
    """Pages of 16, so that a hole takes half of 32 positions: the other half's infinite value, which every token
    sees, is in every token's sum."""
    S = 16 * 8
    cache = kv4.empty_cache(8, 16, 1, D)
    for c, x in zip(cache, (0x22, 127, 0x11, 127)):
        c.fill_(x)
    pages = torch.arange(8, dtype=torch.int32, device=DEV)[None].contiguous()
    pages[0, hole] = -1
    at = hole ^ 1                                    # the page beside the hole
    cache.vq[at, 0, 5, 3], cache.vs[at, 0, 5, 0] = 0x70, 254      # 6 * 2^127 in column 7
    q = torch.from_numpy(np.random.default_rng(M).standard_normal((1, M, G, D))).bfloat16().to(DEV)
    for dt in (torch.float32, torch.bfloat16):
        o = kv4.attn_decode4(q, cache, torch.tensor([S - M], dtype=torch.int32, device=DEV), pages, dt)
        col = torch.zeros(D, dtype=torch.bool, device=DEV)
        col[7] = True
        assert not torch.isfinite(o[..., col]).any() and torch.isfinite(o[..., 32:]).all()
