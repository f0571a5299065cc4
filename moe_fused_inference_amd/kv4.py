"""The KV cache in MXFP4: allocation, write, read-back and decode attention.

A head row of D (64 or 128) keys or values is D/2 bytes of E2M1 nibbles and
D/32 E8M0 codes, the library's MXFP4 row, so a position of one head takes 68
bytes at D = 128 where the FP8 cache of ``attn_decode`` takes 128.  A cache is
the four uint8 tensors of :class:`KV4`, head-major within a page:

    kq, vq   (n_pages, Hkv, page, D/2)      ks, vs   (n_pages, Hkv, page, D/32)

Without a page table sequence b is page b and holds ``page`` positions; with
one (``pages``, int32 (B, max_pages) on the device, a power-of-two page) the
sequences share a pool, and entries outside [0, n_pages) are no page.  Token m
of sequence b sits at ``dpos[b] + m`` (int32 (B,) on the device, so a captured
graph follows it); a batch slot with dpos[b] <= -M is empty.

Every call checks its arguments (RuntimeError), allocates outputs and workspace
with torch's caching allocator and queues its work on torch's current stream of
the cache's device.
"""
from typing import NamedTuple

import torch

from . import fp4_ext


class KV4(NamedTuple):
    """A cache: any sequence of these four tensors does."""
    kq: torch.Tensor
    ks: torch.Tensor
    vq: torch.Tensor
    vs: torch.Tensor


def empty_cache(n_pages, page, Hkv, D=128, device="cuda"):
    """An unwritten cache of n_pages pages (sequences, without a page table) of
    `page` positions, a multiple of 16."""
    if D not in (64, 128) or page <= 0 or page % 16 or n_pages <= 0 or Hkv <= 0:
        raise RuntimeError(f"a cache needs D 64 or 128 and a page that is a multiple of 16, got D={D} page={page} "
                           f"n_pages={n_pages} Hkv={Hkv}")

    def t(w):
        return torch.zeros((n_pages, Hkv, page, w), dtype=torch.uint8, device=device)

    return KV4(t(D // 2), t(D // 32), t(D // 2), t(D // 32))


def _ext():
    return fp4_ext.load_compiled().kv4


def kv4_write(k, v, cache, dpos, pages=None):
    """k, v (B, M, Hkv, D) bf16, fp16 or fp32 -> the cache's rows dpos[b] + m, in
    place, bit-exact to the library's quantizer (``prequant``).  Tokens outside
    the cache or on no page write nothing.  Views whose tokens lie at one stride
    (slices of a projection) are read as they are."""
    kq, ks, vq, vs = cache
    _ext().write(k, v, kq, ks, vq, vs, dpos, pages)


def kv4_read(cache, n, start=None, pages=None, dtype=torch.bfloat16):
    """Positions start[b] .. start[b] + n - 1 (start None: 0 on) of every sequence
    -> (k, v), each (B, n, Hkv, D) of dtype bf16, fp16 or fp32; zeros outside the
    cache and on no page."""
    kq, ks, vq, vs = cache
    k, v = _ext().read(kq, ks, vq, vs, n, start, pages, dtype)
    return k, v


def attn_decode4(q, cache, dpos, pages=None, dtype=torch.float32, window=None, sinks=0, tree=None):
    """softmax(q K^T / sqrt(D)) V of q (B, M, Hq, D) bf16 or fp16, token m of
    sequence b over positions 0 .. dpos[b] + m -> (B, M, Hq, D) of dtype fp32,
    bf16 or fp16.  Zeros for tokens outside the cache and for ones that see no
    position.

    window: of those positions a token sees the last `window`, its own among them,
    and the first `sinks`.  Pages whose positions no token sees may be gone.
    tree: the M tokens are drafts that form a tree, and one sees positions
    0 .. dpos[b] - 1 and of the drafts those in its mask (``tree_masks``, int32
    (B, M, ceil(M / 32))); its window, M at least, counts from its place in its line."""
    kq, ks, vq, vs = cache
    return _ext().attn(q, kq, ks, vq, vs, dpos, pages, dtype, window, sinks, tree)


def attn_decode4_mx(q, cache, dpos, pages=None, window=None, sinks=0, tree=None):
    """attn_decode4 as the MXFP4 rows of its bf16 rounding, the activations of an
    o_proj ``lin_pq``: (oq uint8 (B*M, Hq*D/2), os uint8 (B*M, Hq*D/32))."""
    kq, ks, vq, vs = cache
    oq, os_ = _ext().attn_mx(q, kq, ks, vq, vs, dpos, pages, window, sinks, tree)
    return oq, os_
