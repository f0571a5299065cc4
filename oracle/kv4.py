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


def rounding(D, n, big, size, q_parts=1):
    """How far fp32 sums of the same operands may be from o = sum p v / sum p, as a multiple of sum p |v| / sum p.

    Every fp32 addition and product rounds once, by at most u = 2^-24 of its result, in whatever order the matrix
    unit and the lanes add; hardware exp2 is off by at most 2 ulp (4 u).  big: the largest sum |q k| / sqrt(D) of
    a row (0 where the sums are exact), size: its largest |score|, X = log2(e) size.
    - A score is q_parts D exact products: off by q_parts D u big.  In units of log 2 its exponent is a product by a
      rounded constant (u X), rounded itself where the row's reference is far (u X), and a difference from the
      reference (2 u X); then exp2.
    - Sums meet by factors exp2(reference - reference): the difference rounds by u of it, exp2 and the product by
      5 u.  A wave's reference moves up by 8 at least each time after the first, so 1 + X / 4 times and 2 X in all; the
      waves' sums meet in LDS, the records in a wave of the merge (64 batches of eight at most) and its waves once
      more: each level 2 X in all.
    So a weight is off by a factor 1 +- e, e = log 2 u (log2(e) q_parts D big + 12 X) + (4 + 5 (1 + X / 4 + 2 + 64)) u.
    - A numerator adds three parts of each of a wave's n / 4 positions, a denominator the terms of n / 16 in a lane
      and the lanes; then the waves, and 1024 records at most by eights in waves: 3 n / 4 + 300 and n / 16 + 300
      additions in a row.
    """
    u, x = 2.0 ** -24, np.log2(np.e) * size
    e = np.log(2) * u * (np.log2(np.e) * q_parts * D * big + 12 * x) + (4 + 5 * (67 + x / 4)) * u
    return 2 * e + (13 * n / 16 + 600) * u


def attention(q, cache, dpos, pages=None):
    """q (B, M, Hq, D) float -> (o, bound), float64 (B, M, Hq, D).

    bound: a tolerance on fp32 sums of the same operands, element by element: scores (D + 2) u sum|q k| each, u = 2^-24,
    exponents 2 u max|x| and exp2's 4 u, sums n / 128 + 40 additions in a row.  It is not a proof (rounding is one).  A
    score of fp16 has 2 D products; a wave with a whole sequence adds three parts of its terms, 3 n / 128 matrix steps for
    up to 16 rows and 6 n / 128 for more, each a sum of products itself.  Errors of either sign make up for that: on
    random operands the kernels stay below a hundredth of it.  A term, or a part of one, below 2^-126 of a row whose
    denominator is at least 1 is flushed: up to four such parts a position, each at most 2^-126 max|v|.
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
