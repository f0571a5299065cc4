"""GPU tests of page tables behind a window (kv4.kv4_tables) against oracle/kv4_tables.py: sequences that begin in the place of
others, and ones that step back to pages that are gone."""
import numpy as np
import pytest
import torch

from moe_fused_inference_amd import kv4
from oracle import kv4_masks
from oracle.kv4_tables import Tables
from tests.gpu_helpers import DEV, np_
from tests.kv4_mask_helpers import check, i32

pytestmark = pytest.mark.gpu


def _both(*a):
    return kv4.page_tables(*a), Tables(*a)


def _step(t, want, lens, new=None, T=0):
    got, said = kv4.kv4_tables(t, i32(lens), None if new is None else i32(new), T), want.update(lens, new, T)
    n = len(want.free)
    assert np.array_equal(np_(t.pages), want.pages) and np.array_equal(np_(t.span), want.span)
    assert t.state.tolist() == [n, want.lacked] and t.free[:n].tolist() == want.free
    for x, y in zip(got or (), said or ()):
        assert np.array_equal(np_(x), y)
    return got


# (one workgroup, and past its 32768 entries)
@pytest.mark.parametrize("B,max_pages", [(3, 40), (300, 120)])
@pytest.mark.parametrize("sinks", [0, 17])
def test_a_sequence_that_begins_in_the_place_of_another(B, max_pages, sinks):
    """Every new token has a place, and nothing lacks; no page is lost."""
    t, want = _both(B, max_pages, B * 45, 16, 100, sinks)
    old, new = 600 - np.arange(B) % 7, 20 + np.arange(B) % 50
    _step(t, want, old, old, int(old.sum()))
    _step(t, want, old)
    for _ in range(2):
        got = _step(t, want, new, new, int(new.sum()))
        assert (got.slots >= 0).all() and t.state[1] == 0 and got.slots.unique().numel() == got.slots.numel()
    _step(t, want, np.zeros(B))
    assert sorted(t.free.tolist()) == list(range(B * 45))


def test_its_tokens_are_seen():
    """What the next sequence writes by its slots is what its attention reads."""
    B, Hkv, D, page, window, sinks = 2, 2, 64, 16, 40, 5
    t = kv4.page_tables(B, 32, 64, page, window, sinks)
    cache, alone = kv4.empty_cache(64, page, Hkv, D), kv4.empty_cache(B, 64, Hkv, D)
    for lens, new in ((500, 500), (501, 1), (33, 33)):
        s = kv4.kv4_tables(t, i32([lens] * B), i32([new] * B), B * new)
        k, v = (torch.randn((B * new, Hkv, D), device=DEV).bfloat16() for _ in range(2))
        kv4.kv4_write_slots(k, v, cache, s.slots)
    kv4.kv4_write(k.view(B, 33, Hkv, D), v.view(B, 33, Hkv, D), alone, i32([0] * B))
    q = torch.randn((B, 33, 4 * Hkv, D), device=DEV).bfloat16()
    o, w = (kv4.attn_decode4(q, c, i32([0] * B), p, window=window, sinks=sinks) for c, p in ((cache, t.pages), (alone, None)))
    see = torch.from_numpy(kv4_masks.sees([0] * B, 33, 64, window, sinks)).to(DEV)
    for x in (o, w):
        check(x, q, alone, see)
        assert x.abs().sum(-1).min() > 0


@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 0), (100, 33), (300, 16)])
@pytest.mark.parametrize("B,max_pages,n_pages,page", [(1, 9, 9, 16), (7, 20, 90, 16), (70, 30, 900, 32), (1100, 33, 9000, 16), (300, 120, 5000, 16)])
def test_lives_with_steps_back(B, max_pages, n_pages, page, window, sinks):
    """Lengths that go anywhere, with and without new tokens, and pools that do not hold them all."""
    rng = np.random.default_rng([B, window])
    t, want = _both(B, max_pages, n_pages, page, window, sinks)
    room, lens, lacked, gone = max_pages * page, np.zeros(B, np.int64), 0, 0
    for i in range(12):
        kind = rng.random(B)
        to = np.where(kind < 0.3, rng.integers(0, room + 1, B), np.minimum(lens + rng.integers(0, 60, B), room))
        new = np.where(kind < 0.2, to, np.minimum(rng.integers(0, 60, B), to))
        had = want.span[:, 0] > 0
        got = _step(t, want, to, new, int(new.sum()) + 5) if i % 4 != 3 else _step(t, want, to)
        lens, lacked = to, lacked + want.lacked
        if got:
            gone += int((had[np_(got.seq[:int(got.starts[-1])])] & (np_(got.slots[:int(got.starts[-1])]) < 0)).sum())
    assert B < 70 or (lacked > 0 and gone > 0)
    _step(t, want, np.zeros(B))
    assert sorted(t.free.tolist()) == list(range(n_pages))


@pytest.mark.parametrize("B,max_pages", [(5, 40), (300, 120)])
def test_replays(B, max_pages):
    """A captured call over sequences that end, begin and step back is the call."""
    rng = np.random.default_rng(B)
    t, want = _both(B, max_pages, B * 30, 16, 60, 5)
    lens, new = i32(np.zeros(B)), i32(np.zeros(B))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        kv4.kv4_tables(t, lens, new, 700)
        with torch.cuda.graph(graph, stream=side):
            got = kv4.kv4_tables(t, lens, new, 700)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(8):
        to = rng.integers(0, max_pages * 16, B)
        n = np.where(rng.random(B) < 0.4, to, rng.integers(0, 30, B).clip(0, to))
        lens.copy_(i32(to))
        new.copy_(i32(n))
        graph.replay()
        said = want.update(to, n, 700)
        assert np.array_equal(np_(t.pages), want.pages) and np.array_equal(np_(t.span), want.span) and t.state.tolist() == [len(want.free), want.lacked]
        assert all(np.array_equal(np_(x), y) for x, y in zip(got, said))
