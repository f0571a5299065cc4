"""What the tests of attention over the MXFP4 cache share: how many units a wave gets, and the 64-bit result on the GPU.

A unit is 32 positions.  The library tells its shares by the workspace that it asks for: B places of 16 bytes and a
record of D + 4 floats for every row (M * Hq) and each of shares + B - 1 segments, or nothing where a workgroup has a
whole sequence.
"""
import math

import torch

from moe_fused_inference_amd import _lib
from oracle import kv4 as ref
from tests.gpu_helpers import DEV

MAGS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
PAD, FEW, LEAST = 8, 32, 4      # units before a sequence in the line; shares a sequence past which they double; units of a share


def units_a_wave(B, M, Hq, Hkv, D, max_pos, dpos):
    """(mode, the most units that a wave gets of one sequence): "sequence", "share" or "line"."""
    n = [(min(max(d + M, 0), max_pos) + 31) // 32 for d in dpos]
    ws = _lib.load().mxfp4_attn_kv4_workspace_size(B, M, Hq, Hkv, D, max_pos)
    if ws == 0:
        sixteen = M * (Hq // Hkv) <= 16 and max_pos > 128 and max_pos <= 2048 and 128 <= B * Hkv <= 256
        return "sequence", -(-max(n) // (16 if sixteen else 4))
    records = (ws - 16 * B) // (M * Hq * (D + 4) * 4)
    assert ws == 16 * B + records * M * Hq * (D + 4) * 4
    shares = records - B + 1
    total = sum(n) if B == 1 else sum(x + PAD for x in n if x)
    per = max(-(-(-(-total // shares)) // 4) * 4, 2 * LEAST if total > FEW * LEAST * B else LEAST)
    if B == 1 and shares * LEAST * 32 >= max_pos:
        per = LEAST
    return "share" if B == 1 else "line", -(-min(per, max(n)) // 4)


def streams_k(B, max_pos, n_pages, page, Hkv, D):
    """K goes by streaming loads: the room is more than 128 MB (up to 16 query rows)."""
    return min(B * max_pos, n_pages * page) * Hkv * (D + D // 16) > 128 << 20


def random_cache(n_pages, Hkv, page, D, seed, lo=121, hi=130):
    """Every nibble, scale codes lo .. hi - 1."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def t(w, a, b):
        return torch.randint(a, b, (n_pages, Hkv, page, w), generator=g, device=DEV, dtype=torch.uint8)

    return [t(D // 2, 0, 256), t(D // 32, lo, hi), t(D // 2, 0, 256), t(D // 32, lo, hi)]


def decode64(q, s):
    """Nibbles (..., D/2) and codes (..., D/32) as float64 (..., D)."""
    mags = torch.tensor(MAGS + tuple(-m for m in MAGS), dtype=torch.float64, device=q.device)
    v = mags[torch.stack((q & 15, q >> 4), -1).long()].reshape(*s.shape, 32)
    return torch.ldexp(v, (s.int() - 127)[..., None]).flatten(-2)


def attention64(q, cache, dpos, pages=None, exact_scores=False):
    """(o, bound) of q (B, M, Hq, D), float64 on q's device: softmax(q K^T / sqrt(D)) V, and how far fp32 may be
    from it (ref.rounding; exact_scores: the products' sums are exact in fp32)."""
    B, M, Hq, D = q.shape
    Hkv, page = cache[0].shape[1], cache[0].shape[2]
    G, top = Hq // Hkv, page * (1 if pages is None else pages.shape[1])
    o, bound = (torch.zeros((B, M, Hq, D), dtype=torch.float64, device=q.device) for _ in range(2))
    for b in range(B):
        n = min(int(dpos[b]) + M, top)
        if n <= 0:
            continue
        there = torch.ones(n, dtype=torch.bool, device=q.device)
        if pages is None:
            rows = [c[b, :, :n] for c in cache]
        else:
            ids = pages[b, :-(-n // page)].long()
            ok = (ids >= 0) & (ids < cache[0].shape[0])
            there = ok.repeat_interleave(page)[:n]
            rows = [c[torch.where(ok, ids, 0)].transpose(0, 1).flatten(1, 2)[:, :n] for c in cache]
        pos = int(dpos[b]) + torch.arange(M, device=q.device)
        see = there & (torch.arange(n, device=q.device) <= pos[:, None]) & ((pos >= 0) & (pos < top))[:, None]   # (M, n)
        see = see.repeat_interleave(G, 0)
        any_ = see.any(-1, keepdim=True)
        step = max(1, (1 << 26) // max(M * G * n, n * D))        # kv heads at a time
        for g in range(0, Hkv, step):
            h = slice(g, min(g + step, Hkv))
            k, v = decode64(rows[0][h], rows[1][h]), decode64(rows[2][h], rows[3][h])
            k, v = torch.where(there[:, None], k, 0.0), torch.where(there[:, None], v, 0.0)
            x = q[b].unflatten(1, (Hkv, G))[:, h].transpose(0, 1).flatten(1, 2).double()         # (heads, M * G, D)
            s = torch.matmul(x, k.transpose(1, 2).contiguous()) / math.sqrt(D)
            size = s.abs().masked_fill(~see, 0).amax(-1, keepdim=True)
            big = torch.matmul(x.abs(), k.abs().transpose(1, 2).contiguous()) / math.sqrt(D)
            big = big.masked_fill(~see, 0).amax(-1, keepdim=True)
            s = s.masked_fill(~see, -math.inf)
            p = torch.exp(s - torch.where(any_, s.amax(-1, keepdim=True), 0.0))
            den = torch.where(any_, p.sum(-1, keepdim=True), 1.0)
            want = torch.matmul(p, v) / den
            rel = ref.rounding(D, n, 0.0 if exact_scores else big, size, 2 if q.dtype == torch.float16 else 1)
            lim = rel * torch.matmul(p, v.abs()) / den + 2 * 2.0 ** -24 * want.abs() + 4 * n * 2.0 ** -126 * v.abs().max()
            lim = torch.where(any_, lim, 0.0)
            for t, to in ((want, o), (lim, bound)):
                to[b].unflatten(1, (Hkv, G))[:, h] = t.unflatten(1, (M, G)).transpose(0, 1)
    return o, bound


def check64(got, q, cache, dpos, pages=None, exact_scores=False, two_parts=False):
    """got within the bound, and half a step of its type; two_parts: the probabilities are off by 2^-17 of themselves."""
    want, bound = attention64(q, cache, dpos, pages, exact_scores)
    if two_parts:
        assert got.dtype != torch.float32
    lim = bound + (2.0 ** -17 * _sizes(q, cache, dpos, pages) if two_parts else 0)
    if got.dtype != torch.float32:
        lim = lim + torch.finfo(got.dtype).eps / 2 * (want.abs() + lim) + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    off = (got.double() - want).abs()
    bad = ~(off <= lim)
    assert not bad.any(), (int(bad.sum()), float((off / lim.clamp_min(1e-300)).max()), bad.nonzero()[:4].tolist())


def _sizes(q, cache, dpos, pages):
    """sum p |v| / sum p."""
    plus = [cache[0], cache[1], cache[2] & 0x77, cache[3]]
    return attention64(q, plus, dpos, pages)[0]


# ------------------------------------------------------------------ the bits of a probability
P_BITS = 24 * 2.0 ** -24     # see p_rows


def p_rows(n, D):
    """n bf16 values x in (0, 4 sqrt(D) log 2): with a key of -x / q at one position and zeros at the others of a row, that
    position's probability is p = 2^-t over 1 + others, t = x log2(e) / sqrt(D) < 4, and a value of 1 there alone makes the
    output p / (p + others).

    How far fp32 may be from it, relatively, u = 2^-24: t's constant and its fma 2.8 u each (u t log 2), exp2 4 u; p's three
    parts are its 24 bits, their sum one rounding at most; the denominator ten (three in a lane, two over lanes, four waves,
    one merge), its reciprocal and the product two: under 24 u.  A p of two bf16 parts is off by up to 64 u more.
    """
    x = torch.linspace(0.02, 1.0, n, dtype=torch.float64) * 4 * math.sqrt(D) * math.log(2) * 0.99
    return x.to(torch.bfloat16)
