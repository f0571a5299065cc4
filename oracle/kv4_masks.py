"""What a token sees of the MXFP4 KV cache under a window with sinks and in a tree of drafts, and the tree's masks
from its parents, in numpy from the words of include/mxfp4_hip.h -- test infrastructure only."""
import numpy as np


def sees(dpos, M, S, window=None, sinks=0, tree=None):
    """bool (B, M, S): token m of sequence b sees position p.  tree: int (B, M, words), or None."""
    B = len(dpos)
    out = np.zeros((B, M, S), bool)
    p = np.arange(S, dtype=np.int64)
    for b in range(B):
        base = int(dpos[b])
        for m in range(M):
            slot = base + m
            if slot < 0 or slot >= S:
                continue
            if tree is None:
                row, at = p <= slot, slot
            else:
                row, drafts = p < base, 0
                for i in range(M):
                    if (int(tree[b, m, i // 32]) >> (i % 32)) & 1:
                        drafts += 1
                        if 0 <= base + i < S:
                            row[base + i] = True
                at = base + drafts - 1
            if window is not None:
                begins = p > at - window
                if tree is not None:
                    begins |= p >= base          # a window hides no draft
                row &= begins | (p < sinks)
            out[b, m] = row
    return out


def line(parents, m):
    """Draft m and its ancestors, or nothing where it, or one of them, is no draft."""
    found = []
    while True:
        p = int(parents[m])
        if not -1 <= p < m:
            return []
        found.append(m)
        if p == -1:
            return found
        m = p


def tree_masks(parents):
    """parents int (B, M) -> (words int32 (B, M, ceil(M/32)), depth int32 (B, M))."""
    B, M = parents.shape
    words = np.zeros((B, M, (M + 31) // 32), np.uint32)
    depth = np.full((B, M), -1, np.int32)
    for b in range(B):
        for m in range(M):
            found = line(parents[b], m)
            for i in found:
                words[b, m, i // 32] |= np.uint32(1 << (i % 32))
            depth[b, m] = len(found) - 1
    return words.view(np.int32), depth
