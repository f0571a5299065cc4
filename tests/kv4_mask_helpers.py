"""Attention over the MXFP4 cache by a mask of what each token sees, in 64 bits on the GPU, and the bound on fp32 (oracle/kv4.py)."""
import math

import numpy as np
import torch

from moe_fused_inference_amd import kv4
from oracle import kv4 as ref
from oracle import kv4_masks
from tests.gpu_helpers import DEV
from tests.kv4_helpers import decode64

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, dtype=np.int64).astype(np.int32))).to(DEV)


def table(rng, B, max_pages, n_pages):
    return rng.permutation(n_pages)[:B * max_pages].reshape(B, max_pages).astype(np.int32)


def random_parents(rng, B, M, empty=True):
    """Trees of M drafts; with `empty` some drafts are none, and so their children."""
    p = np.array([[-1 if m == 0 else rng.integers(-1 if rng.random() < 0.05 else 0, m) for m in range(M)] for _ in range(B)], np.int32).reshape(B, M)
    if empty and M > 2:
        for b in range(B):
            for m in rng.integers(1, M, 1 + M // 20):
                p[b, m] = (-2, M, m, 2 ** 31 - 1, -2 ** 31)[rng.integers(5)]
    return p


def rows_of(cache, pages, b, S):
    """Sequence b's rows as float64 (Hkv, S, D) of k and v, zeros where there is no page, and which are there."""
    page = cache[0].shape[2]
    if pages is None:
        return *(decode64(cache[i][b, :, :S], cache[i + 1][b, :, :S]) for i in (0, 2)), torch.ones(S, dtype=torch.bool, device=DEV)
    ids = pages[b].long()
    ok = (ids >= 0) & (ids < cache[0].shape[0])
    there = ok.repeat_interleave(page)[:S]
    out = []
    for i in (0, 2):
        q, s = (cache[j][torch.where(ok, ids, 0)].transpose(0, 1).flatten(1, 2)[:, :S] for j in (i, i + 1))
        out.append(torch.where(there[:, None], decode64(q, s), 0.0))
    return *out, there


def attention64(q, cache, see, pages=None):
    """(o, bound) of q (B, M, Hq, D) by see bool (B, M, S), float64: softmax over what is seen and on a page, and how far fp32
    may be from it."""
    B, M, Hq, D = q.shape
    Hkv, S = cache[0].shape[1], see.shape[2]
    G = Hq // Hkv
    o, bound = (torch.zeros((B, M, Hq, D), dtype=torch.float64, device=DEV) for _ in range(2))
    for b in range(B):
        k, v, there = rows_of(cache, pages, b, S)
        sb = see[b] & there
        if not sb.any():
            continue
        at = sb.any(0).nonzero()[:, 0]             # only what some token sees
        k, v, sb = k[:, at], v[:, at], sb[:, at].repeat_interleave(G, 0)
        n, any_ = at.numel(), sb.any(-1, keepdim=True)
        for g in range(Hkv):
            x = q[b].unflatten(1, (Hkv, G))[:, g].flatten(0, 1).double()           # (M * G, D)
            s = (x @ k[g].T.contiguous()) / math.sqrt(D)
            size = s.abs().masked_fill(~sb, 0).amax(-1, keepdim=True)
            big = ((x.abs() @ k[g].abs().T.contiguous()) / math.sqrt(D)).masked_fill(~sb, 0).amax(-1, keepdim=True)
            s = s.masked_fill(~sb, -math.inf)
            p = torch.exp(s - torch.where(any_, s.amax(-1, keepdim=True), 0.0))
            den = torch.where(any_, p.sum(-1, keepdim=True), 1.0)
            want = p @ v[g] / den
            rel = ref.rounding(D, n, big, size, 2 if q.dtype == torch.float16 else 1)
            lim = rel * (p @ v[g].abs()) / den + 2 * 2.0 ** -24 * want.abs() + 4 * n * 2.0 ** -126 * v[g].abs().max()
            for t, to in ((want, o), (torch.where(any_, lim, 0.0), bound)):
                to[b].unflatten(1, (Hkv, G))[:, g] = t.unflatten(0, (M, G))
    return o, bound


def check(got, q, cache, see, pages=None):
    """got within the bound, and half a step of its type; more than 16 rows to 16 bits have probabilities off by 2^-17."""
    want, bound = attention64(q, cache, see, pages)
    lim = bound
    if got.dtype != torch.float32:
        plus = [cache[0], cache[1], cache[2] & 0x77, cache[3]]
        if q.shape[1] * q.shape[2] // cache[0].shape[1] > 16:
            lim = lim + 2.0 ** -17 * attention64(q, plus, see, pages)[0]
        lim = lim + torch.finfo(got.dtype).eps / 2 * (want.abs() + lim) + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    off = (got.double() - want).abs()
    bad = ~(off <= lim)
    assert not bad.any(), (int(bad.sum()), float((off / lim.clamp_min(1e-300)).max()), bad.nonzero()[:4].tolist())


class Call:
    """A random call: its cache, table, positions, q, masks, and what it sees."""

    def __init__(self, B, M, Hkv, G, D, page, S, dpos, qt="bf16", window=None, sinks=0, tree=False, seed=0, words=None, holes=0):
        rng = np.random.default_rng([B, M, Hkv, G, D, S, seed])
        n_pages, P = (B * (S // page) + 1, page) if page else (B, S)
        self.cache = kv4.KV4(*(torch.from_numpy(rng.integers(lo, hi, (n_pages, Hkv, P, w), dtype=np.uint8)).to(DEV)
                               for w, lo, hi in ((D // 2, 0, 256), (D // 32, 121, 130)) * 2))
        tab = table(rng, B, S // page, n_pages) if page else None
        for _ in range(holes):
            tab[rng.integers(B), rng.integers(S // page)] = -1
        self.pages = None if tab is None else i32(tab)
        self.dpos = i32(dpos)
        self.q = torch.from_numpy(rng.standard_normal((B, M, Hkv * G, D))).to(DT[qt]).to(DEV)
        if tree:
            words = kv4_masks.tree_masks(random_parents(rng, B, M))[0]
        self.tree = None if words is None else i32(words)
        self.window, self.sinks = window, sinks
        self.see = torch.from_numpy(kv4_masks.sees(dpos, M, S, window, sinks, words)).to(DEV)

    def run(self, dtype=torch.float32, cache=None, pages=None, q=None):
        return kv4.attn_decode4(self.q if q is None else q, cache or self.cache, self.dpos, self.pages if pages is None else pages, dtype,
                                window=self.window, sinks=self.sinks, tree=self.tree)

    def run_mx(self):
        return kv4.attn_decode4_mx(self.q, self.cache, self.dpos, self.pages, window=self.window, sinks=self.sinks, tree=self.tree)

    def fill_unseen(self, value=255):
        """A copy of the cache whose rows that no token sees hold `value` (255: -6 * NaN)."""
        page = self.cache[0].shape[2]
        new = [c.clone() for c in self.cache]
        used = torch.zeros(new[0].shape[0], page, dtype=torch.bool, device=DEV)
        for b in range(self.see.shape[0]):
            at = self.see[b].any(0).nonzero()[:, 0]
            if self.pages is None:
                used[b, at] = True
            else:
                ids = self.pages[b].long()[at // page]
                ok = (ids >= 0) & (ids < used.shape[0])
                used[ids[ok], (at % page)[ok]] = True
        for c in new:
            c.transpose(1, 2)[~used] = value
        return kv4.KV4(*new)
