"""GPU tests of attention over the MXFP4 cache with windows at the sizes where its plan changes (csrc/attn_kv4.hip): a
workgroup of four or sixteen waves for a sequence, or shares and a merge, up to 16 rows of a kv head and more."""
import pytest
import torch

from tests.kv4_mask_helpers import Call, check

pytestmark = pytest.mark.gpu

# the last room for which a sequence has one workgroup, 34 or 16 (15 or 24 with more rows) positions for each, is inside
# each of these lists of windows
FEW = [(1, 2, 4, 64, [40, 300, 400]), (6, 2, 4, 128, [300, 350, 400, 450]), (3, 5, 3, 64, [300, 450, 520]), (16, 4, 8, 128, [384, 1500, 2100, 2300]),
       (65, 4, 4, 64, [300, 3900, 4200])]
MANY = [(1, 2, 8, 128, [200, 300]), (4, 4, 5, 64, [200, 440, 560, 700]), (12, 8, 4, 128, [900, 1300, 1500]), (50, 8, 4, 64, [3000])]


def _lens(B, M, S):
    return [S - M] + [int((S - M) * ((i * 0.618 + 0.3) % 1)) - S * (i % 7 == 3) for i in range(1, B)]


def _run(B, M, Hkv, G, D, S, window, sinks, tree, out):
    call = Call(B, M, Hkv, G, D, 64, S, _lens(B, M, S), window=window, sinks=sinks, tree=tree, seed=window)
    got = call.run(out)
    check(got, call.q, call.cache, call.see, call.pages)
    assert torch.equal(got, call.run(out, cache=call.fill_unseen()))        # NaN in all that no token sees


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("B,Hkv,G,D,window", [(*c[:4], w) for c in FEW for w in c[4]])
def test_up_to_16_rows(B, Hkv, G, D, window, tree):
    _run(B, 16 // G if B < 10 else 1, Hkv, G, D, 4480, window, window % 37, tree, torch.float32)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("B,Hkv,G,D,window", [(*c[:4], w) for c in MANY for w in c[4]])
def test_more_rows(B, Hkv, G, D, window, tree):
    _run(B, 1 + 16 // G * (3 if B < 10 else 1), Hkv, G, D, 4480, window, window % 37, tree, torch.bfloat16 if D == 128 else torch.float32)
