"""GPU tests of the page tables and slots (kv4.kv4_tables, kv4.kv4_write_slots) against oracle/kv4_tables.py: every value equal."""
import numpy as np
import pytest
import torch

from moe_fused_inference_amd import kv4
from oracle import kv4 as ref
from oracle.kv4_tables import Tables
from tests.gpu_helpers import DEV, np_
from tests.kv4_mask_helpers import i32

pytestmark = pytest.mark.gpu


def _same(t, want, got=None, said=None):
    n = len(want.free)
    assert np.array_equal(np_(t.pages), want.pages) and np.array_equal(np_(t.span), want.span)
    assert t.state.tolist() == [n, want.lacked] and t.free[:n].tolist() == want.free
    if got is not None:
        for x, y, dt in zip(got, said, (torch.int64, torch.int32, torch.int32, torch.int32)):
            assert x.dtype == dt and np.array_equal(np_(x), y)


def _both(B, max_pages, n_pages, page, window=None, sinks=0):
    return kv4.page_tables(B, max_pages, n_pages, page, window, sinks), Tables(B, max_pages, n_pages, page, window, sinks)


# the second group goes past what one workgroup does alone (32768 entries, 8192 tokens), the third past one round of sums
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 0), (100, 33), (1, 1), (5000, 16)])
@pytest.mark.parametrize("B,max_pages,n_pages,page,step", [(1, 4, 4, 16, 9), (7, 9, 50, 16, 30), (48, 20, 700, 64, 40), (1, 3, 2, 32, 20),
                                                           (130, 300, 9000, 16, 150), (600, 60, 12000, 32, 60), (1, 40000, 30000, 16, 9000),
                                                           (1100, 5, 4000, 16, 8), (1100, 33, 9000, 16, 60)])
def test_a_life(B, max_pages, n_pages, page, step, window, sinks):
    """Prompts, steps, rejected drafts, ends and new sequences, with pools that do not hold them all."""
    rng = np.random.default_rng([B, max_pages, sinks])
    t, want = _both(B, max_pages, n_pages, page, window, sinks)
    room = max_pages * page
    lens = np.zeros(B, np.int64)
    for i in range(14):
        fresh = lens == 0
        new = np.where(fresh, rng.integers(1, room + 1, B) // (1 if i % 3 else 4), rng.integers(0, step, B))
        new = np.where(fresh & (rng.random(B) < 0.3), 0, new)
        lens = np.where(rng.random(B) < 0.15, 0, lens + new)
        new = np.where(lens == 0, 0, new)
        T = int(new.sum()) + (0, 3, -2, 700)[i % 4]
        T = max(T, 0)
        _same(t, want, kv4.kv4_tables(t, i32(lens), new=i32(new), T=T), want.update(lens, new, T))
        if i % 2:
            lens = lens - np.minimum(rng.integers(0, 9, B), np.maximum(new - 1, 0))       # some of them are rejected
            assert kv4.kv4_tables(t, i32(lens)) is None
            want.update(lens)
            _same(t, want)
        lens = np.minimum(lens, room + 5)
    kv4.kv4_tables(t, i32(np.zeros(B)))
    want.update(np.zeros(B))
    _same(t, want)
    assert want.span.max() == 0 and sorted(t.free.tolist()) == list(range(n_pages))


def test_returned_pages_are_handed_on():
    """More sequences end than begin in one call, and fewer, in one workgroup and in many."""
    for B, max_pages in ((64, 30), (300, 200)):
        rng = np.random.default_rng(B)
        t, want = _both(B, max_pages, B * max_pages // 2 + 7, 16)
        for ends in (0.5, 0.9, 0.1):
            lens = np.where(rng.random(B) < ends, 0, rng.integers(0, max_pages * 16 + 1, B))
            new = np.minimum(lens, rng.integers(0, 200, B))
            _same(t, want, kv4.kv4_tables(t, i32(lens), i32(new), 9000), want.update(lens, new, 9000))


def test_strange_lengths():
    t, want = _both(9, 6, 40, 16)
    lens = np.array([-1, -2 ** 31, 2 ** 31 - 1, 96, 97, 1, 16, 17, 0])
    new = np.array([5, 3, 4, -7, 2, 3, -2 ** 31, 0, 2])
    got, said = kv4.kv4_tables(t, i32(lens), i32(new), 30), want.update(lens, new, 30)
    ok = said[1] != 1                    # (a position below -2^31 has no int32)
    assert np.array_equal(np_(got.slots), said[0]) and np.array_equal(np_(got.seq), said[1]) and np.array_equal(np_(got.pos)[ok], said[2][ok])
    _same(t, want)
    # more new tokens than there are places, by far
    got = kv4.kv4_tables(t, i32([3] * 9), i32([2 ** 31 - 1, 0, 2 ** 31 - 1] + [1] * 6), 50)
    assert got.starts.tolist() == [0] + [2 ** 30] * 9 and (got.seq == 0).all() and (got.slots == -1).all()
    assert got.pos.tolist() == [3 - (2 ** 31 - 1) + j for j in range(50)]


def test_state_that_is_wrong_is_kept_within_its_tensors():
    """Ranges, counts and ids that no call leaves: nothing is read or written past the tensors, and the rest stays."""
    rng = np.random.default_rng(3)
    for B, max_pages in ((40, 20), (300, 200)):
        n = B * max_pages // 3
        whole = [torch.full((m + 64,), 77, dtype=torch.int32, device=DEV) for m in (B * max_pages, 2 * B, n, 2)]
        pages, span, free, state = (w[32:-32] for w in whole)
        for x in (pages, span, free):
            x.copy_(i32(rng.integers(-2 ** 31, 2 ** 31, x.numel())))
        state.copy_(i32([rng.choice([2 ** 31 - 1, -5, n // 2]), 0]))
        t = kv4.PageTables(pages.view(B, max_pages), span.view(B, 2), free, state, 16)
        for _ in range(4):
            kv4.kv4_tables(t, i32(rng.integers(0, max_pages * 16, B)), i32(rng.integers(0, 9, B)), 500)
            assert 0 <= int(state[0]) <= n and int(span.min()) >= 0 and int(span.max()) <= max_pages
        assert all((w[:32] == 77).all() and (w[-32:] == 77).all() for w in whole)


@pytest.mark.parametrize("B,max_pages,T", [(48, 40, 500), (300, 200, 9000)])
def test_replays(B, max_pages, T):
    """Captured once, replayed over a batch's life with eager work between."""
    rng = np.random.default_rng(B)
    t, want = _both(B, max_pages, B * max_pages // 2, 16, window=300, sinks=5)
    lens, new = i32(np.zeros(B)), i32(np.zeros(B))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        kv4.kv4_tables(t, lens, new, T)
        with torch.cuda.graph(graph, stream=side):
            got = kv4.kv4_tables(t, lens, new, T)
    torch.cuda.current_stream().wait_stream(side)
    x = np.zeros(B, np.int64)
    for i in range(8):
        n = rng.integers(0, 60, B)
        x = np.where(rng.random(B) < 0.1, 0, np.minimum(x + n, max_pages * 16))
        n = np.where(x == 0, 0, n)
        lens.copy_(i32(x))
        new.copy_(i32(n))
        graph.replay()
        _same(t, want, got, want.update(x, n, T))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("Hkv,D,page", [(4, 128, 64), (5, 64, 16), (1, 64, 48), (3, 128, 16)])
def test_write_slots(Hkv, D, page, dtype):
    """Rows at slots in any order, some of them none: the bytes of kv4_write; views of a projection among them."""
    rng = np.random.default_rng(page)
    n_pages, T = 9, 140
    slots = rng.permutation(n_pages * page)[:T].astype(np.int64)
    slots[rng.integers(0, T, 9)] = [-1, n_pages * page, 2 ** 40, -2 ** 60, 2 ** 63 - 1, 2 ** 32, -1, -1, -1]
    proj = torch.randn((T, 3 * Hkv + 1, D), device=DEV).to(dtype)
    for k, v in ((proj[:, :Hkv], proj[:, Hkv:2 * Hkv]), (proj[:, 1:Hkv + 1].contiguous(), proj[:, 2 * Hkv:3 * Hkv].contiguous())):
        got, want = kv4.empty_cache(n_pages, page, Hkv, D), kv4.empty_cache(n_pages, page, Hkv, D)
        kv4.kv4_write_slots(k, v, got, torch.from_numpy(slots).to(DEV))
        host = [np_(c).copy() for c in want]
        ok = [t for t in range(T) if 0 <= slots[t] < n_pages * page]
        pages = np.array([[slots[t] // page] for t in ok])
        ref.write(np_(k[ok].float())[:, None], np_(v[ok].float())[:, None], host, slots[ok] % page, pages)
        assert all(np.array_equal(np_(a), b) for a, b in zip(got, host)) and any(c.any() for c in host)


def test_write_slots_far_in_a_pool():
    """Places past 2^31."""
    page, n_pages, D = 16, (1 << 27) + 2, 64
    cache = kv4.empty_cache(n_pages, page, 1, D)          # 73 GB
    slots = torch.tensor([n_pages * page - 1, 1 << 31, (1 << 31) - 1, 5], device=DEV)
    k = torch.randn((4, 1, D), device=DEV)
    kv4.kv4_write_slots(k, -k, cache, slots)
    ids = (slots // page).to(torch.int32)[:, None].contiguous()
    rk, rv = kv4.kv4_read(cache, 1, start=(slots % page).to(torch.int32).contiguous(), pages=ids, dtype=torch.float32)
    small = kv4.empty_cache(4, page, 1, D)
    kv4.kv4_write(k[:, None], -k[:, None], small, i32([0] * 4))
    assert torch.equal(rk, kv4.kv4_read(small, 1, dtype=torch.float32)[0]) and torch.equal(rv, -rk) and rk.any()
    del cache
    torch.cuda.empty_cache()


def test_the_tables_serve_the_cache():
    """A batch's life on the device: ragged prompts and steps, written by slots and attended to through the table with a
    window whose pages behind it go back; against a cache that keeps every position."""
    rng = np.random.default_rng(9)
    B, Hkv, G, D, page, S, window, sinks = 5, 2, 4, 64, 16, 512, 60, 10
    t = kv4.page_tables(B, S // page, 40, page, window, sinks)
    cache, whole = kv4.empty_cache(40, page, Hkv, D), kv4.empty_cache(B, S, Hkv, D)
    lens = np.zeros(B, np.int64)
    for i in range(30):
        new = np.where(lens == 0, rng.integers(1, 90, B), rng.integers(1, 7, B))
        if i == 12:
            lens[3], new[3] = 0, 0                     # it ends
        lens = lens + new
        M, T = int(new.max()), int(new.sum()) + 2
        s = kv4.kv4_tables(t, i32(lens), i32(new), T)
        assert int(t.state[1]) == 0
        k, v = (torch.randn((T, Hkv, D), device=DEV).bfloat16() for _ in range(2))
        kv4.kv4_write_slots(k, v, cache, s.slots)
        for b in range(B):
            a, e = s.starts[b].item(), s.starts[b + 1].item()
            if e > a:
                alone = kv4.KV4(*(c[b:b + 1] for c in whole))
                kv4.kv4_write(k[None, a:e], v[None, a:e], alone, i32([lens[b] - new[b]]))
        q = torch.randn((B, M, Hkv * G, D), device=DEV).bfloat16()
        dpos = i32(lens - M)                           # the last M positions of each, the new ones among them
        o, w = (kv4.attn_decode4(q, c, dpos, p, window=window, sinks=sinks) for c, p in ((cache, t.pages), (whole, None)))
        for b in range(B):
            n = int(new[b])
            if n:
                assert torch.isfinite(o[b, M - n:]).all() and (o[b, M - n:] - w[b, M - n:]).abs().max() <= 1e-5 * w[b].abs().max()


def test_shapes_without_work_and_refusals():
    t = kv4.page_tables(2, 3, 8, 16)
    lens, new = i32([20, 3]), i32([20, 3])
    got = kv4.kv4_tables(t, lens, new, 0)
    assert got.slots.shape == (0,) and got.starts.tolist() == [0, 20, 23]
    none = kv4.PageTables(torch.empty((0, 3), dtype=torch.int32, device=DEV), torch.empty((0, 2), dtype=torch.int32, device=DEV), t.free, t.state, 16)
    e = torch.empty(0, dtype=torch.int32, device=DEV)
    assert kv4.kv4_tables(none, e) is None and kv4.kv4_tables(none, e, e, 3).slots.tolist() == [-1] * 3
    before = [x.clone() for x in t[:4]]
    for bad in (dict(lens=lens[:1]), dict(lens=lens.long()), dict(lens=lens.cpu()), dict(new=new[:1]), dict(new=new.long()), dict(T=-1),
                dict(new=None, T=3), dict(t=t._replace(pages=t.pages.long())), dict(t=t._replace(pages=t.pages[0])), dict(t=t._replace(span=t.span[:1])),
                dict(t=t._replace(free=t.free.long())), dict(t=t._replace(state=t.state[:1])), dict(t=t._replace(page=24)), dict(t=t._replace(page=8)),
                dict(t=t._replace(page=0)), dict(t=t._replace(window=0)), dict(t=t._replace(sinks=4)), dict(t=t._replace(window=5, sinks=-1)),
                dict(t=t._replace(free=t.free[:0])), dict(t=t._replace(pages=t.pages[:, :0])), dict(t=t._replace(pages=t.pages.t())),
                dict(t=t._replace(page=1 << 30)), dict(t=t._replace(span=t.span.cpu()))):
        a = dict(t=t, lens=lens, new=new, T=4)
        a.update(bad)
        with pytest.raises(RuntimeError):
            kv4.kv4_tables(a["t"], a["lens"], a["new"], a["T"])
    assert all(torch.equal(x, y) for x, y in zip(t, before))
    cache, k = kv4.empty_cache(2, 16, 2, 64), torch.zeros((3, 2, 64), device=DEV)
    s = torch.zeros(3, dtype=torch.int64, device=DEV)
    kv4.kv4_write_slots(k[:0], k[:0], cache, s[:0])
    for k_, v_, s_ in ((k, k, s[:2]), (k, k, s.int()), (k, k, s.cpu()), (k, k.half(), s), (k[None], k[None], s), (k[:, :1], k[:, :1], s),
                       (k[..., :32], k[..., :32], s), (k.double(), k.double(), s), (k.cpu(), k, s)):
        with pytest.raises(RuntimeError):
            kv4.kv4_write_slots(k_, v_, cache, s_)
