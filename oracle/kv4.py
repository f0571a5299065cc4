"""The MXFP4 KV cache in numpy, float64 -- test infrastructure only.

Restates the layout and rules of the kv4 entry points of include/mxfp4_hip.h on
host arrays: kq, vq (n_pages, Hkv, page, D/2), ks, vs (n_pages, Hkv, page, D/32),
pages (B, max_pages) or None.  A head row is a row of oracle.mxfp4.
"""
import numpy as np

from . import mxfp4 as fmt


def place(cache, pages, b, pos):
    """(page, row) of position pos of sequence b, or None outside the cache and on no page."""
    n_pages, _, page, _ = cache[0].shape
    top = page if pages is None else pages.shape[1] * page
    if pos < 0 or pos >= top:
        return None
    if pages is None:
        return b, pos
    pid = int(pages[b, pos // page])
    return (pid, pos % page) if 0 <= pid < n_pages else None


def write(k, v, cache, dpos, pages=None):
    """k, v (B, M, Hkv, D) float32 -> the cache, in place."""
    B, M, Hkv, D = k.shape
    for x, q, s in ((k, cache[0], cache[1]), (v, cache[2], cache[3])):
        wp, ws = fmt.quantize_rows(x.reshape(-1, D))
        wp, ws = wp.reshape(B, M, Hkv, -1), ws.reshape(B, M, Hkv, -1)
        for b in range(B):
            for m in range(M):
                at = place(cache, pages, b, int(dpos[b]) + m)
                if at is not None:
                    q[at[0], :, at[1]] = wp[b, m]
                    s[at[0], :, at[1]] = ws[b, m]


def read(cache, n, start, pages=None):
    """Positions start[b] .. start[b] + n - 1 as float32 (B, n, Hkv, D), and which of them there are (B, n)."""
    Hkv, D = cache[0].shape[1], cache[0].shape[3] * 2
    B = len(start)
    k, v = np.zeros((B, n, Hkv, D), np.float32), np.zeros((B, n, Hkv, D), np.float32)
    there = np.zeros((B, n), bool)
    for b in range(B):
        at = [place(cache, pages, b, int(start[b]) + i) for i in range(n)]
        idx = [i for i, a in enumerate(at) if a is not None]
        if not idx:
            continue
        p, r = np.array([at[i][0] for i in idx]), np.array([at[i][1] for i in idx])
        for out, q, s in ((k, cache[0], cache[1]), (v, cache[2], cache[3])):
            rows = fmt.dequant_rows(q[p, :, r].reshape(-1, D // 2), s[p, :, r].reshape(-1, D // 32))
            out[b, idx] = rows.reshape(len(idx), Hkv, D)
        there[b, idx] = True
    return k, v, there


def attention(q, cache, dpos, pages=None):
    """q (B, M, Hq, D) float -> (o, bound), float64 (B, M, Hq, D).

    bound: how far fp32 sums of the same operands may be from o, element by
    element.  A score is D products summed in fp32 (error <= (D + 2) u sum|q k|,
    u = 2^-24) and its exponent, in units of log 2, is a product, a difference
    and a hardware exp2 of error <= 2 ulp (4 u); so every weight is off by a
    factor 1 +- e, e <= log 2 * (scale * (D + 2) u max sum|q k| + 2 u max|x|) + 4 u.
    Numerator and denominator sum n such terms (at most n/128 + 32 rounded
    additions in a row, every V and part of p exact), and both merge twice.  An
    output sum p v / sum p is then off by at most (2 e + 2 (n/128 + 40) u)
    sum p |v| / sum p, and a rounding of its own.  A term, or a part of one, below
    2^-126 of a row whose largest is at least 1 (and at most 2^8) is flushed: up to
    four such parts a position, each at most 2^-126 max|v|, over a sum of at least 1.
    """
    u = 2.0 ** -24
    B, M, Hq, D = q.shape
    Hkv = cache[0].shape[1]
    G = Hq // Hkv
    o, bound = np.zeros((B, M, Hq, D)), np.zeros((B, M, Hq, D))
    top = cache[0].shape[2] * (1 if pages is None else pages.shape[1])
    for b in range(B):
        n = min(int(dpos[b]) + M, top)
        if n <= 0:
            continue
        one = (cache, pages[b:b + 1]) if pages is not None else ([x[b:b + 1] for x in cache], None)
        k, v, there = read(one[0], n, [0], one[1])
        k, v, there = k[0].astype(np.float64), v[0].astype(np.float64), there[0]
        k[~there] = 0
        v[~there] = 0
        for m in range(M):
            pos = int(dpos[b]) + m
            if pos < 0 or pos >= top:
                continue
            see = there & (np.arange(n) <= pos)
            if not see.any():
                continue
            for h in range(Hq):
                kk, vv = k[see, h // G], v[see, h // G]
                x = q[b, m, h].astype(np.float64)
                s = kk @ x / np.sqrt(D)
                p = np.exp(s - s.max())
                den = p.sum()
                o[b, m, h] = p @ vv / den
                big = (np.abs(kk) @ np.abs(x)).max() / np.sqrt(D)
                e = np.log(2) * (1.4427 * (D + 2) * u * big + 2 * u * 1.4427 * np.abs(s).max()) + 4 * u
                bound[b, m, h] = ((2 * e + 2 * (len(s) / 128 + 40) * u) * (p @ np.abs(vv)) / den + u * np.abs(o[b, m, h])
                                  + 4 * len(s) * 2.0 ** -126 * np.abs(vv).max())
    return o, bound
