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


def _value(cache, b, g, pos, block, code, columns, nibble):
    """Value row (b, g, pos): nothing but `nibble` in columns `columns` of a block, under scale code `code`."""
    row = torch.zeros(32, dtype=torch.uint8)
    row[list(columns)] = nibble
    cache[2][b, g, pos, 16 * block:16 * block + 16] = (row[0::2] | row[1::2] << 4).to(DEV)
    cache[3][b, g, pos, block] = code


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("name", [n for n, c in FEW_UNITS.items() if c[1] > 1])
def test_values_that_only_later_tokens_see(name, D):
    """Infinities and NaN among the keys and values of a call's later tokens leave the earlier tokens' bits alone; of a
    value they reach their columns, and no others."""
    cache, dpos, q = _few(name, D)
    q = q.bfloat16()
    B, M, Hkv = q.shape[0], q.shape[1], FEW_UNITS[name][2]
    clean = [c.clone() for c in cache]
    bad = {}                                          # (sequence, kv head, token) -> columns that are not finite
    # scale code and nibble: infinite of either sign, NaN
    for i, (code, nibble) in enumerate(((253, 7), (253, 14), (254, 4), (254, 15), (255, 1), (255, 0))):
        b, g, j, block = i % B, (5 * i) % Hkv, max(1, M - 1 - 7 * (i % 4)), i % (D // 32)
        if i == 4:
            j = -2                                    # all tokens see it, in the unit of the first of them
        columns = (i, 31 - 3 * i)
        _value(cache, b, g, dpos[b] + j, block, code, columns, nibble)
        _value(clean, b, g, dpos[b] + j, block, 127, columns, 0)
        bad[b, g, j, i] = [32 * block + c for c in (range(32) if code == 255 else columns)]
    G = FEW_UNITS[name][3]
    for out in (torch.float32, torch.bfloat16):
        o, want = (kv4.attn_decode4(q, c, _i32(dpos), dtype=out) for c in (cache, clean))
        hit = torch.zeros_like(o, dtype=torch.bool)
        for (b, g, j, _), columns in bad.items():
            for c in columns:
                hit[b, max(j, 0):, g * G:(g + 1) * G, c] = True
        assert torch.equal(o[~hit], want[~hit]) and torch.isfinite(want).all()
        assert not torch.isfinite(o[hit]).any()
    # keys: a token before them sees nothing of them
    for i, code in enumerate((253, 254, 255)):
        b, g, j = i % B, (3 * i + 1) % Hkv, max(1, M - 1 - 5 * i)
        keys = [c.clone() for c in clean]
        keys[0][b, g, dpos[b] + j] = 0x7E
        keys[1][b, g, dpos[b] + j] = code
        o = kv4.attn_decode4(q, keys, _i32(dpos))
        want = kv4.attn_decode4(q, clean, _i32(dpos))
        same = torch.ones_like(o, dtype=torch.bool)
        same[b, j:, g * G:(g + 1) * G] = False
        assert torch.equal(o[same], want[same])


def test_large_values_that_are_finite_stay():
    """1, 2 and 3 times 2^126, 1.5 times 2^127, seen by some tokens: they are values, not infinities."""
    B, M, Hkv, G, S, _, _ = FEW_UNITS["rows16-share"]
    for M, Hkv, S in ((M, Hkv, S), (32, 32, 4096)):
        cache = random_cache(1, Hkv, S, 64, 3)
        dpos = [S - M - 1]
        g = torch.Generator(device=DEV)
        g.manual_seed(M)
        q = torch.randn((1, M, Hkv * 2, 64), generator=g, device=DEV).bfloat16()
        j = M - 1
        for g, (code, nibble) in enumerate(((253, 2), (253, 4), (253, 13), (254, 3), (254, 9))):
            _value(cache, 0, g, dpos[0] + j, 1, code, (3, 4), nibble)
            cache[0][0, g, dpos[0] + j] = 0          # a score of 0: a small part of the row's sum
        small = [c.clone() for c in cache]
        for g in range(5):
            small[3][0, g, dpos[0] + j, 1] -= 120    # the same times 2^-120
        o, s = kv4.attn_decode4(q, cache, _i32(dpos)), kv4.attn_decode4(q, small, _i32(dpos))
        assert torch.isfinite(o).all() and torch.equal(o[:, :j], s[:, :j])
        for g in range(5):
            big = o[0, j, 2 * g:2 * g + 2, 35:37].abs()
            assert (big > 2.0 ** 60).any()
