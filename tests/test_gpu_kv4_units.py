"""GPU tests of attention over the MXFP4 KV cache where a wave has several units of 32 positions: what it carries from
one to the next.  Each case says how many it means to have, and is held to that by the library's own shares."""
import numpy as np
import pytest
import torch

from moe_fused_inference_amd import kv4
from tests.gpu_helpers import DEV
from tests.kv4_helpers import P_BITS, check64, decode64, p_rows, random_cache, streams_k, units_a_wave

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


# ------------------------------------------------------------------ many units
@pytest.mark.parametrize("D,dt,out", [(64, "fp16", "fp32"), (128, "bf16", "bf16"), (128, "bf16", "fp32"), (64, "bf16", "fp16")])
@pytest.mark.parametrize("name", FEW_UNITS)
def test_several_units(name, D, dt, out):
    cache, dpos, q = _few(name, D, seed=1)
    q = (1.5 * q).to(DT[dt])
    o = kv4.attn_decode4(q, cache, _i32(dpos), dtype=DT[out])
    check64(o, q, cache, dpos, two_parts=name.startswith("rows32") and out != "fp32")


def _paged(name, B, M, Hkv, G, S, D, dpos, pool, mode, units, dt, out):
    """Sequences whose tables name a small pool's pages again and again."""
    page = 128
    assert units_a_wave(B, M, Hkv * G, Hkv, D, S, dpos) == (mode, units), name
    g = torch.Generator(device=DEV)
    g.manual_seed(units + M)
    pages = torch.randint(0, pool, (B, S // page), generator=g, device=DEV, dtype=torch.int32)
    cache = random_cache(pool, Hkv, page, D, units)
    q = (1.5 * torch.randn((B, M, Hkv * G, D), generator=g, device=DEV)).to(DT[dt])
    o = kv4.attn_decode4(q, cache, _i32(dpos), pages, DT[out])
    check64(o, q, cache, dpos, pages, two_parts=M * G > 16 and out != "fp32")


FORMS = [(128, "bf16", "fp32"), (64, "fp16", "bf16"), (128, "fp16", "bf16"), (64, "bf16", "fp32")]


@pytest.mark.parametrize("units", [4, 5, 64, 65, 66])
@pytest.mark.parametrize("D,dt,out", FORMS)
def test_many_units_more_rows_a_sequence(D, dt, out, units):
    """A piece of a prompt, a workgroup for every 32 rows of it."""
    _paged("rows sequence", 1, 128, 8, 16, 8704, D, [128 * units - 128 - units], 20, "sequence", units, dt, out)


@pytest.mark.parametrize("units", [4, 5, 64, 65, 66])
@pytest.mark.parametrize("D,dt,out", FORMS)
def test_many_units_more_rows_a_share(D, dt, out, units):
    _paged("rows share", 1, 64, 8, 16, 17408, D, [256 * units - 64 - units], 20, "share", units, dt, out)


@pytest.mark.parametrize("D,dt,out", FORMS)
def test_many_units_more_rows_in_the_line(D, dt, out):
    _paged("rows line", 2, 64, 8, 16, 17408, D, [16600, 16601], 20, "line", 131, dt, out)


@pytest.mark.parametrize("pool", [8, 128])
@pytest.mark.parametrize("D,dt,out", FORMS)
def test_many_units_a_share(D, dt, out, pool):
    assert streams_k(1, 34816, pool, 128, 256, D) == (pool == 128)
    for units in (64, 65, 66) if (pool, dt, out) == (8, "bf16", "fp32") else (66,):
        _paged("share", 1, 2, 256, 2, 34816, D, [512 * units - 2 - units], pool, "share", units, dt, out)


@pytest.mark.parametrize("pool", [8, 256])
@pytest.mark.parametrize("D,dt,out", FORMS)
def test_many_units_a_sequence(D, dt, out, pool):
    """Most of the batch's slots are empty, or as good as."""
    assert streams_k(64, 8704, pool, 128, 64, D) == (pool == 256)
    dpos = [-3] * 64
    dpos[5], dpos[17], dpos[40], dpos[41], dpos[63] = 8448 - 3, 8192 + 31, 4 * 32 - 3, 0, 8320 - 2
    _paged("sequence", 64, 3, 64, 5, 8704, D, dpos, pool, "sequence", 66, dt, out)


@pytest.mark.parametrize("pool", [8, 128])
@pytest.mark.parametrize("D,dt,out", FORMS)
def test_many_units_in_the_line(D, dt, out, pool):
    assert streams_k(2, 17408, pool, 128, 256, D) == (pool == 128)
    _paged("line", 2, 1, 256, 3, 17408, D, [16895, 16700], pool, "line", 67, dt, out)


# ------------------------------------------------------------------ scores that move a row's reference
# levels of a wave's units in turn, as shares of the top one
SHAPES = {"rising": [0, 1, 2, 3], "falling": [3, 2, 1, 0], "peak": [0, 3, 1, 0], "valley": [2, 0, 0, 3], "late": [0, 0, 0, 3],
          "zigzag": [1, 3, 0, 2], "level": [3, 3, 3, 3]}
# log2 of a step between levels.  A reference moves where a lane's eight terms (16 of them with more rows) sum past 2^11:
# at a step of about 8 (7), and far above
STEPS = (0.5, 5.0, 6.9, 7.1, 7.9, 8.1, 9.0, 11.1, 13.0, 30.0)


def _staircase(name, D, shape, steps, seed):
    """Keys whose score is step * (level of the unit + 0 .. 6 eighths): sums that fp32 holds.  Values of a level have one
    sign, so that what is left of lower levels shows (tests/test_kv4_mistakes.py)."""
    B, M, Hkv, G, S, mode, units = FEW_UNITS[name]
    cache, dpos, _ = _few(name, D, seed)
    waves = 16 if "sixteen" in name else 4
    j = torch.arange(S // 32, device=DEV) // waves % units                       # the wave's units in turn
    level = torch.tensor(SHAPES[shape], device=DEV)[j * 4 // units]
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    cache[0].zero_()
    cache[1].fill_(127)
    level = level.repeat_interleave(32)
    fine = torch.randint(0, 8, (B, Hkv, S), generator=g, device=DEV, dtype=torch.uint8)
    one = 2 * torch.stack((level & 1, level >> 1)).to(torch.uint8)               # E2M1 1 in dimensions 0 and 1: a bit of the level each
    cache[0][..., 0] = one[0] | one[1] << 4
    cache[0][..., 1] = fine                                                      # dimension 2
    cache[2].copy_(cache[2] & 0x77 | (0x88 * (level & 1)).to(torch.uint8)[:, None])          # a value's sign is its level's
    cache[3].copy_(torch.randint(124, 131, cache[3].shape, generator=g, device=DEV, dtype=torch.uint8))
    step = torch.tensor([steps[(7 * i) % len(steps)] for i in range(B * M * Hkv * G)], device=DEV).view(B, M, Hkv * G)
    q = torch.zeros((B, M, Hkv * G, D), device=DEV)
    s = (step * np.log(2) * D ** 0.5).bfloat16().float()
    q[..., 0], q[..., 1], q[..., 2] = s, 2 * s, s / 8
    return cache, dpos, q.bfloat16()


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("name", ["rows16-share", "rows16-sequence", "rows16-sixteen-waves", "rows32-share", "rows32-sequence"])
def test_references_that_move(name, D, shape):
    cache, dpos, q = _staircase(name, D, shape, STEPS, 5)
    o = kv4.attn_decode4(q, cache, _i32(dpos))
    check64(o, q, cache, dpos, exact_scores=True)
    # one row's reference past 2^18 among the others': theirs as before, and its own the mean over the largest score's
    # values, whose sum (multiples of 2^-4 below 2^20) fp32 holds
    far = torch.zeros(q.shape[:3], dtype=torch.bool, device=DEV)
    far[:, ::3, ::FEW_UNITS[name][3]] = True
    x = q.clone()
    s = torch.tensor(2.0 ** 18 * np.log(2) * D ** 0.5, device=DEV).bfloat16()
    x[far] = 0
    for d, f in ((0, 1), (1, 2), (2, 1 / 8)):
        x[..., d][far] = s * f
    of = kv4.attn_decode4(x, cache, _i32(dpos))
    assert torch.equal(of[~far], o[~far])
    b, m, h = far.nonzero().T
    for i in range(0, len(b), max(1, len(b) // 64)):
        bi, mi, hi = int(b[i]), int(m[i]), int(h[i])
        g, n = hi // FEW_UNITS[name][3], dpos[bi] + mi + 1
        keys, values = (decode64(cache[c][bi, g, :n], cache[c + 1][bi, g, :n]) for c in (0, 2))
        score = keys @ x[bi, mi, hi].double()
        top = score == score.max()
        want = values[top].mean(0)
        assert ((of[bi, mi, hi].double() - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,Hkv,G", [(1, 8, 16), (4, 16, 4), (16, 32, 1), (17, 16, 1), (32, 8, 1), (64, 4, 4)])
def test_probabilities_keep_their_bits(M, Hkv, G, D):
    """24 of them where fp32 goes out, for any number of rows; 16 at least of bf16(o) and fp16(o)."""
    n = Hkv * G * M
    x = p_rows(n, D).to(DEV).view(1, M, Hkv * G)
    q = torch.zeros((1, M, Hkv * G, D), dtype=torch.bfloat16, device=DEV)
    q[..., 0] = x
    p = torch.exp2(-x.double() * np.log2(np.e) / np.sqrt(D))
    want = (p / (p + torch.arange(1, M + 1, device=DEV)[:, None]))[..., None]
    for S in (128, 8192):
        cache = kv4.empty_cache(1, S, Hkv, D)
        for c in (cache.ks, cache.vs):
            c.fill_(127)
        cache.kq[0, :, 1, 0] = 0x0A                   # -1 in dimension 0
        cache.vq[0, :, 1] = 0x22                      # 1
        for dt in (torch.float32, torch.bfloat16, torch.float16):
            o = kv4.attn_decode4(q, cache, _i32([1]), dtype=dt)
            lim = P_BITS * want
            if dt != torch.float32:
                lim = lim + 2.0 ** -17 * want
                lim = lim + torch.finfo(dt).eps / 2 * (want + lim) + (2.0 ** -25 if dt == torch.float16 else 0.0)
            assert ((o.double() - want).abs() <= lim).all()
