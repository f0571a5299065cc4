"""GPU tests of values that are not finite in trees without a window (kv4.attn_decode4): what a draft's infinity reaches."""
import pytest
import torch

from moe_fused_inference_amd import kv4
from tests.kv4_mask_helpers import Call

pytestmark = pytest.mark.gpu


# up to 16 rows of a kv head and more; a share of one sequence, of a batch's line, and a workgroup a sequence; positions in one
# unit of 32 with the context's last, in the next, and past 32 drafts
@pytest.mark.parametrize("q", ["bf16", "fp16"])
@pytest.mark.parametrize("B,M,Hkv,G,D,page,S,base", [
    (1, 5, 2, 3, 64, 0, 4096, 2001), (1, 4, 1, 4, 128, 32, 4096, 2020), (5, 4, 1, 4, 128, 0, 2048, 1003), (5, 5, 2, 3, 64, 16, 2048, 1003),
    (1, 6, 1, 2, 128, 0, 32, 9), (40, 3, 1, 4, 64, 0, 64, 37),
    (1, 30, 2, 2, 128, 0, 4096, 2005), (1, 40, 1, 3, 64, 32, 4096, 2005), (3, 26, 1, 4, 128, 0, 2048, 1021), (3, 33, 2, 2, 64, 16, 2048, 1021),
    (1, 20, 1, 1, 128, 0, 32, 11), (4, 30, 4, 2, 64, 0, 64, 33)])
def test_an_infinity_reaches_the_drafts_that_see_it(B, M, Hkv, G, D, page, S, base, q):
    """Those alone: the others' bits stay, those of a sibling in the same unit among them."""
    b = B // 2
    dpos = [base - 7 * abs(i - b) for i in range(B)]
    c = Call(B, M, Hkv, G, D, page, S, dpos, q, tree=True, seed=M)
    seen = [int(c.see[b, :, at].sum()) for at in range(base, base + M)]
    assert any(0 < n < M for n in seen)
    for at in (base - 1, base, base + 1, base + M // 2, base + M - 1):
        col, tile = at % D, (b, at) if not page else (int(c.pages[b, at // page]), at % page)
        for dt in (torch.float32, torch.bfloat16):
            o = c.run(dt)
            bad = kv4.KV4(*(x.clone() for x in c.cache))
            bad.vs[tile[0], :, tile[1], col // 32] = 254
            bad.vq[tile[0], :, tile[1], col // 32 * 16:col // 32 * 16 + 16] = 0        # (zeros of a large scale are zeros)
            clean = c.run(dt, cache=kv4.KV4(*(x.clone() for x in bad)))
            for code, byte in ((254, 0x77), (255, 0x11)):                              # an infinity, NaN
                bad.vs[tile[0], :, tile[1], col // 32] = code
                bad.vq[tile[0], :, tile[1], col // 32 * 16:col // 32 * 16 + 16] = 0
                bad.vq[tile[0], :, tile[1], col // 2] = byte & 0x0F << 4 * (col & 1)
                got = c.run(dt, cache=bad)
                hit = torch.zeros_like(o, dtype=torch.bool)
                if code == 254:
                    hit[b, :, :, col] = c.see[b, :, at, None]
                else:                                                                  # 0 times NaN is NaN: the block's 32 columns
                    hit[b, :, :, col // 32 * 32:col // 32 * 32 + 32] = c.see[b, :, at, None, None]
                assert not torch.isfinite(got[hit]).any()
                assert torch.equal(got[~hit], clean[~hit])
            unseen = torch.ones((B, M), dtype=torch.bool, device=o.device)
            unseen[b] = ~c.see[b, :, at]
            assert torch.isfinite(clean).all() and torch.equal(o[unseen], clean[unseen])
