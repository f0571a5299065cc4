"""GPU tests of attention over the MXFP4 KV cache where a wave has several units of 32 positions: what it carries from
one to the next.  Each case says how many it means to have, and is held to that by the library's own shares."""
import numpy as np
import pytest
import torch

from moe_fused_inference_amd import kv4
from tests.gpu_helpers import DEV
from tests.kv4_helpers import check64, random_cache, streams_k, units_a_wave

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# B, M, Hkv, G, S of a few units a wave: up to 16 rows, and more, by shares and whole sequences
FEW_UNITS = {
    "rows16-share": (1, 2, 64, 4, 8192, "share", 4), "rows16-line": (2, 4, 64, 3, 8192, "line", 9),
    "rows16-sequence": (64, 1, 16, 8, 2048, "sequence", 16), "rows16-sixteen-waves": (16, 3, 8, 5, 2048, "sequence", 4),
    "rows32-share": (1, 32, 32, 2, 4096, "share", 4), "rows32-line": (2, 9, 32, 8, 4096, "line", 14),
    "rows32-sequence": (8, 70, 8, 2, 2048, "sequence", 16)}


def _i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def _few(name, D, seed=0):
    B, M, Hkv, G, S, mode, units = FEW_UNITS[name]
    dpos = [S - M - 3 * i for i in range(B)]
    assert units_a_wave(B, M, Hkv * G, Hkv, D, S, dpos) == (mode, units)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    q = torch.randn((B, M, Hkv * G, D), generator=g, device=DEV)
    return random_cache(B, Hkv, S, D, seed), dpos, q


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("name", FEW_UNITS)
def test_a_rows_bits_are_its_own(name, D):
    """Rows beside one whose scores jump from unit to unit, one past 2^18, and ones of NaN keep their bits."""
    cache, dpos, q = _few(name, D)
    B, M, Hq = q.shape[:3]
    for dt, out in ((torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16)):
        alone = kv4.attn_decode4(q.to(dt), cache, _i32(dpos), dtype=out)
        G = FEW_UNITS[name][3]
        rows = torch.zeros((B, M, Hq), dtype=torch.bool, device=DEV)
        rows[:, ::7, ::G] = True                    # one head of every group, of every seventh token
        for strange in (30.0, 3e4, float("nan")):   # scores of some hundred, of 2^18 and more
            x = q.clone()
            x[rows] *= strange
            if strange == strange:
                x = x.clamp(-6e4, 6e4)
            o = kv4.attn_decode4(x.to(dt), cache, _i32(dpos), dtype=out)
            assert torch.equal(o[~rows], alone[~rows])
            assert torch.isnan(o[rows]).all() if strange != strange else torch.isfinite(o[rows]).all()
