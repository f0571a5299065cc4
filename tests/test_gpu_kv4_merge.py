"""GPU tests of how rows' records are merged (csrc/attn_kv4.hip): many rows, sequences across few and many shares of a batch."""
import numpy as np
import pytest
import torch

from tests.kv4_mask_helpers import Call, check

pytestmark = pytest.mark.gpu


def _lens(kind, B, M, S):
    full = S - M
    if kind == "one":                  # the second alone is full: four units a share, from the middle of one on
        return [1 - M] + [full] + [-M] * (B - 2)
    if kind == "all":
        return [full] * B
    return [int(full * ((i * 0.618 + 0.3) % 1)) - (M + 1) * (i % 5 == 2) for i in range(B)]


# rows of all tokens and heads 2048 and more; a full sequence of 4096 positions is 128 units
@pytest.mark.parametrize("kind", ["one", "all", "spread"])
@pytest.mark.parametrize("B,M,Hkv,G,D,S,window,tree,out", [
    (64, 1, 4, 8, 128, 4096, None, False, "fp32"), (64, 1, 4, 8, 64, 4080, None, False, "bf16"), (64, 1, 4, 8, 128, 3904, None, False, "fp16"),
    (65, 2, 2, 8, 128, 4096, None, True, "fp32"), (128, 1, 1, 16, 64, 6000, 4000, False, "fp32"), (16, 16, 1, 8, 128, 4096, None, True, "bf16"),
    (8, 33, 2, 4, 64, 2000, None, True, "fp32"), (1, 64, 4, 8, 128, 4096, None, False, "bf16"), (3, 90, 2, 4, 128, 4096, 3000, True, "bf16"),
    (2, 300, 1, 4, 64, 4096, 2000, False, "fp32")])
def test_many_rows(B, M, Hkv, G, D, S, window, tree, out, kind):
    if kind == "one" and B == 1:
        kind = "all"
    S = S // 16 * 16
    call = Call(B, M, Hkv, G, D, 0, S, _lens(kind, B, M, S), window=window, sinks=5 if window else 0, tree=tree, seed=7)
    dtype = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}[out]
    check(call.run(dtype), call.q, call.cache, call.see)
    oq, os_ = call.run_mx()
    want = call.run(torch.bfloat16).float().view(-1, Hkv * G * D)
    if M * G <= 16:                    # (more rows to bf16 have p in two parts, and to MXFP4 in three)
        from oracle import mxfp4 as fmt
        q, s = fmt.quantize_rows(want.cpu().numpy())
        assert np.array_equal(oq.cpu().numpy(), q) and np.array_equal(os_.cpu().numpy(), s)
