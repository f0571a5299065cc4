"""The KV cache in MXFP4: allocation, write, read-back and decode attention; windows, trees of drafts, page tables.

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

A server's step over a pool, nothing of which needs the host: ``kv4_tables`` makes
room for each sequence's new tokens and says where they go, ``kv4_write_slots``
writes them, ``attn_decode4`` attends (``window=``, ``sinks=``; ``tree=`` from
``tree_masks`` where the tokens are drafts); ``kv4_keep`` moves an accepted path's
rows together, and ``kv4_tables`` with the lengths that stay takes the rest back.

Every call checks its arguments (RuntimeError), allocates outputs and workspace
with torch's caching allocator and queues its work on torch's current stream of
the cache's device.
"""
from typing import NamedTuple, Optional

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


class PageTables(NamedTuple):
    """A batch's page table over a pool, and what is left of the pool (:func:`page_tables`).  ``pages`` is what the
    calls here take as theirs; the others are ``kv4_tables``' own.  ``state``: free pages, and how many the sequences
    need and have not since the last call."""
    pages: torch.Tensor      # int32 (B, max_pages)
    span: torch.Tensor       # int32 (B, 2)
    free: torch.Tensor       # int32 (n_pages)
    state: torch.Tensor      # int32 (2)
    page: int
    window: Optional[int] = None
    sinks: int = 0


class Slots(NamedTuple):
    """Where a call's new tokens go, sequence after sequence: the pool's rows for ``kv4_write_slots`` (-1: none),
    each token's sequence and position (-1 past the last), and how many there are before each sequence's and in all."""
    slots: torch.Tensor      # int64 (T)
    seq: torch.Tensor        # int32 (T)
    pos: torch.Tensor        # int32 (T)
    starts: torch.Tensor     # int32 (B + 1)


def page_tables(B, max_pages, n_pages, page, window=None, sinks=0, device="cuda"):
    """The table of B sequences without pages, of max_pages each at most, over a pool of n_pages pages of `page`
    positions (a power of two from 16 on), all free.  window, sinks: those of its attention, if it has them;
    pages that no window reaches any more are then given back."""
    if B <= 0 or max_pages <= 0 or n_pages <= 0 or page < 16 or page & (page - 1):
        raise RuntimeError(f"a table needs sequences, pages, and a page of a power of two from 16 on, got B={B} max_pages={max_pages} "
                           f"n_pages={n_pages} page={page}")
    if (window is not None and window <= 0) or sinks < 0 or (sinks and window is None):
        raise RuntimeError(f"a window is positive, and sinks need one, got window={window} sinks={sinks}")

    def t(x):
        return x.to(device=device, dtype=torch.int32).contiguous()

    return PageTables(t(torch.full((B, max_pages), -1)), t(torch.zeros(B, 2)), t(torch.arange(n_pages - 1, -1, -1)),
                      t(torch.tensor([n_pages, 0])), page, window, sinks)


def _ext():
    return fp4_ext.load_compiled().kv4


def kv4_write(k, v, cache, dpos, pages=None):
    """k, v (B, M, Hkv, D) bf16, fp16 or fp32 -> the cache's rows dpos[b] + m, in
    place, bit-exact to the library's quantizer (``prequant``).  Tokens outside
    the cache or on no page write nothing.  Views whose tokens lie at one stride
    (slices of a projection) are read as they are."""
    kq, ks, vq, vs = cache
    _ext().write(k, v, kq, ks, vq, vs, dpos, pages)


def kv4_tables(tables, lens, new=None, T=0):
    """The page table follows the lengths (int32 (B,) on the device), in place: every sequence has the pages of its
    first lens[b] positions after the call (those that its window still reaches), taken from the pool; what it had
    beyond goes back, all of it where lens[b] <= 0, the end of a sequence.  Where the pool lacks pages, the first
    sequences get them, ``state[1]`` says how many lack, and the same call asks for them again.  A call and one with
    the lengths before it (drafts that are rejected) leave everything as it was.

    new (int32 (B,)): the last new[b] positions are new tokens; -> their Slots, T places.

    ``state[1]`` also counts the pages of lengths past max_pages * page, which no later call can give: tokens there get
    the slot -1.

    With a window, pages behind it that went back are not given again: a sequence that steps back to them has none
    there, its new tokens' slots are -1, and ``state[1]`` counts them.  One that begins in the place of another, all
    lens[b] positions of it new, has its pages from the first on, with or without a call of length 0 between."""
    got = _ext().tables(tables.pages, tables.span, tables.free, tables.state, tables.page, tables.window, tables.sinks, lens, new, T)
    return Slots(*got) if got else None


def kv4_write_slots(k, v, cache, slots):
    """kv4_write of tokens one after another: k, v (T, Hkv, D) -> the pool's rows slots (int64 (T,), those of
    ``kv4_tables``, each of them once); tokens whose slot is none write nothing."""
    kq, ks, vq, vs = cache
    _ext().write_slots(k, v, kq, ks, vq, vs, slots)


def tree_masks(parents):
    """parents (int32 (B, M)) of trees of drafts, each an earlier draft or -1 for none (anything else: no draft, nor
    are its children) -> (tree, depth): what ``attn_decode4`` takes, itself and its ancestors as bits, and the number
    of ancestors (-1: no draft), so that draft m's position, for its rotation, is dpos[b] + depth[b, m]."""
    tree, depth = _ext().tree_masks(parents)
    return tree, depth


def kv4_keep(caches, dpos, path, pages=None):
    """What stays of a verified tree moves together: the rows at positions dpos[b] + path[b, k] go to dpos[b] + k, in
    a cache or each of a list of them (a model's layers, one launch for 64).  path (int32 (B, A)): drafts in the
    order of their line, so path[b, k] >= k (others stay where they are), -1 from its end on.  Each cache is named once."""
    if len(caches) and isinstance(caches[0], torch.Tensor):
        caches = [caches]
    _ext().keep(caches, dpos, path, pages)


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
