"""GPU tests of a draft tree's masks and of the accepted path's move (kv4.tree_masks, kv4.kv4_keep): every bit equal."""
import numpy as np
import pytest
import torch

from moe_fused_inference_amd import kv4
from oracle import kv4 as ref
from oracle import kv4_masks
from tests.gpu_helpers import DEV, np_
from tests.kv4_mask_helpers import check, i32, random_parents, table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,M", [(1, 1), (1, 2), (3, 26), (1, 31), (2, 32), (2, 33), (5, 64), (2, 65), (3, 100), (2, 257), (64, 500), (1, 1030), (1, 4096)])
def test_masks(B, M):
    rng = np.random.default_rng(M)
    m = np.arange(M, dtype=np.int32)
    kinds = [random_parents(rng, B, M), random_parents(rng, B, M, empty=False), np.tile(m - 1, (B, 1)), np.full((B, M), -1, np.int32),
             np.tile(np.where(m % 2, 0, np.maximum(m - 2, -1)), (B, 1)).astype(np.int32)]
    kinds.append(np.where(np.arange(M) < M // 2, kinds[1], -2).astype(np.int32))
    for p in kinds[:2] + [kinds[-1]] if M > 500 or B > 10 else kinds:
        words, depth = kv4_masks.tree_masks(p)
        got, d = kv4.tree_masks(i32(p))
        assert got.dtype == d.dtype == torch.int32 and np.array_equal(np_(got), words) and np.array_equal(np_(d), depth)


def test_masks_of_long_lines():
    """One line of 4096 drafts, and one broken in the middle."""
    M = 4096
    p = np.tile(np.arange(-1, M - 1, dtype=np.int32), (2, 1))
    p[1, 2000] = M
    got, d = kv4.tree_masks(i32(p))
    bits = (got[..., None] >> torch.arange(32, device=DEV) & 1).flatten(2).bool()
    low = torch.tril(torch.ones(M, M, dtype=torch.bool, device=DEV))
    assert torch.equal(bits[0], low) and d[0].tolist() == list(range(M))
    assert torch.equal(bits[1, :2000], low[:2000]) and not bits[1, 2000:].any() and d[1].tolist() == list(range(2000)) + [-1] * 2096


def test_masks_replay_and_refuse():
    rng = np.random.default_rng(1)
    p = i32(random_parents(rng, 3, 70))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        kv4.tree_masks(p)
        with torch.cuda.graph(graph, stream=side):
            got = kv4.tree_masks(p)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(4):
        x = random_parents(rng, 3, 70)
        p.copy_(i32(x))
        graph.replay()
        assert all(np.array_equal(np_(a), b) for a, b in zip(got, kv4_masks.tree_masks(x)))
    assert kv4.tree_masks(p[:0])[0].shape == (0, 70, 3) and kv4.tree_masks(p[:, :0].contiguous())[0].shape == (3, 0, 0)
    for bad in (p.long(), p.cpu(), p[0], p.t(), torch.zeros((1, 4097), dtype=torch.int32, device=DEV), torch.zeros((65536, 1), dtype=torch.int32, device=DEV)):
        with pytest.raises(RuntimeError):
            kv4.tree_masks(bad)


def _keep(cache, dpos, path, pages):
    """The definition: all rows are read before any is written."""
    moves = []
    for b in range(path.shape[0]):
        for k, p in enumerate(path[b]):
            if p < 0:
                break
            if p > k:
                src, dst = (ref.place(cache, pages, b, int(dpos[b]) + int(i)) for i in (p, k))
                if src is not None and dst is not None:
                    moves.append((dst, [c[src[0], :, src[1]].copy() for c in cache]))
    for dst, rows in moves:
        for c, r in zip(cache, rows):
            c[dst[0], :, dst[1]] = r


def _caches(rng, L, n, Hkv, page, D):
    return [[rng.integers(0, 256, (n, Hkv, page, w), dtype=np.uint8) for w in (D // 2, D // 32) * 2] for _ in range(L)]


@pytest.mark.parametrize("B,A,L,Hkv,D,page,S,dpos", [
    (1, 1, 1, 4, 128, 0, 64, [5]), (1, 5, 3, 4, 128, 0, 64, [0]), (3, 9, 2, 5, 64, 16, 96, [3, 80, 17]), (2, 30, 1, 1, 128, 32, 128, [60, 90]),
    (2, 100, 1, 2, 64, 0, 400, [3, 150]), (2, 300, 1, 1, 128, 64, 1024, [0, 500]), (4, 8, 66, 1, 64, 16, 64, [0, 30, 60, 40]),
    (4, 8, 1, 2, 128, 16, 64, [-3, 2 ** 31 - 1, -2 ** 31, 63])])
def test_keep(B, A, L, Hkv, D, page, S, dpos):
    rng = np.random.default_rng(A + D)
    n, P = (B * (S // page) + 2, page) if page else (B, S)
    tab = table(rng, B, S // page, n) if page else None
    if page and S // page > 2:
        tab[rng.integers(B), rng.integers(S // page)] = -1
    for kind in range(4):
        if kind == 0:       # lines of a tree
            path = np.sort(np.stack([rng.permutation(3 * A)[:A] for _ in range(B)]), -1)
        elif kind == 1:     # the next one each: every row is read and written
            path = np.tile(np.arange(1, A + 1), (B, 1))
        elif kind == 2:     # any order, some below their place
            path = rng.integers(0, 2 * A, (B, A))
        else:               # the same draft again and again, far ones, ends
            path = np.full((B, A), A + 1)
            path[:, A // 2:] = 2 ** 31 - 1
        if kind != 1:
            path = np.where(np.arange(A) < rng.integers(0, A + 1, (B, 1)), path, rng.choice([-1, -2 ** 31], (B, A)))
        host = _caches(rng, L, n, Hkv, P, D)
        dev = [kv4.KV4(*(torch.from_numpy(c).to(DEV) for c in cache)) for cache in host]
        kv4.kv4_keep(dev if L > 1 else dev[0], i32(dpos), i32(path), None if tab is None else i32(tab))
        for cache, got in zip(host, dev):
            _keep(cache, dpos, path, tab)
            assert all(np.array_equal(np_(a), b) for a, b in zip(got, cache))


def test_keep_in_a_cache_past_four_gigabytes():
    B, Hkv, D, S = 9, 8, 128, 1 << 20
    cache = kv4.empty_cache(B, S, Hkv, D)
    k, v = (torch.randn((B, 20, Hkv, D), device=DEV).bfloat16() for _ in range(2))
    dp = i32([S - 20] * B)
    kv4.kv4_write(k, v, cache, dp)
    before = kv4.kv4_read(cache, 20, dp)
    path = i32([[0, 3, 4, 11, 19, -1, 2]] * B)
    kv4.kv4_keep(cache, dp, path)
    for x, y in zip(kv4.kv4_read(cache, 20, dp), before):
        assert torch.equal(x[:, :5], y[:, [0, 3, 4, 11, 19]]) and torch.equal(x[:, 5:], y[:, 5:])
    assert not cache.kq[:, :, :S - 20].any()
    del cache
    torch.cuda.empty_cache()


def test_keep_refuses():
    cache, dp, path = kv4.empty_cache(2, 32, 2, 64), i32([3, 4]), i32([[0, 2], [0, 1]])
    before = [c.clone() for c in cache]
    kv4.kv4_keep(cache, dp, path[:, :0].contiguous())
    other = kv4.empty_cache(2, 48, 2, 64)
    for c, d, p, t in ((cache, dp[:1], path, None), (cache, dp.long(), path, None), (cache, dp, path.long(), None), (cache, dp, path[:1], None),
                       (cache, dp, path[0], None), (cache, dp, path.cpu(), None), (cache, dp, path.t(), None), ([cache, other], dp, path, None),
                       ([cache[:3]], dp, path, None), (cache, dp, path, i32([[0]])), ([cache, cache._replace(vs=cache.vs.cpu())], dp, path, None),
                       ([cache, cache._replace(kq=cache.kq.float())], dp, path, None), ([cache, cache._replace(ks=cache.kq)], dp, path, None)):
        with pytest.raises(RuntimeError):
            kv4.kv4_keep(c, d, p, t)
    with pytest.raises((RuntimeError, IndexError)):
        kv4.kv4_keep([], dp, path)
    assert all(torch.equal(x, y) for x, y in zip(cache, before))


def test_steps_of_drafted_trees():
    """Two layers' caches over a pool, steps of a tree each: pages, slots, masks, attention, the accepted path's move, pages
    given back; in a captured graph beside eager steps, against a cache that only ever gets the accepted tokens."""
    rng = np.random.default_rng(2)
    B, M, A, Hkv, G, D, page, S, L = 3, 13, 6, 2, 4, 64, 16, 256, 2
    n_pages = 40
    t, e = (kv4.page_tables(B, S // page, n_pages, page) for _ in range(2))
    caches, eager, whole = ([kv4.empty_cache(*shape, Hkv, D) for _ in range(L)] for shape in ((n_pages, page), (n_pages, page), (B, S)))
    lens = np.array([40, 7, 90])
    for tab, cs in ((t, caches), (e, eager)):
        s = kv4.kv4_tables(tab, i32(lens), i32(lens), int(lens.sum()))
        torch.manual_seed(0)
        for c, w in zip(cs, whole):
            k, v = (torch.randn((int(lens.sum()), Hkv, D), device=DEV).bfloat16() for _ in range(2))
            kv4.kv4_write_slots(k, v, c, s.slots)
            for b in range(B):
                a, z = s.starts[b].item(), s.starts[b + 1].item()
                kv4.kv4_write(k[None, a:z], v[None, a:z], kv4.KV4(*(x[b:b + 1] for x in w)), i32([0]))
    ks, vs = (torch.randn((L, B * M, Hkv, D), device=DEV).bfloat16() for _ in range(2))
    q = torch.randn((L, B, M, Hkv * G, D), device=DEV).bfloat16()
    parents, path, dpos, new = i32(np.zeros((B, M))), i32(np.zeros((B, A))), i32(lens), i32([M] * B)

    def step(tab, cs):
        after = dpos + M
        s = kv4.kv4_tables(tab, after, new, B * M)
        tree, depth = kv4.tree_masks(parents)
        o = []
        for i, c in enumerate(cs):
            kv4.kv4_write_slots(ks[i], vs[i], c, s.slots)
            o.append(kv4.attn_decode4(q[i], c, dpos, tab.pages, tree=tree))
        kv4.kv4_keep(cs, dpos, path, tab.pages)
        kv4.kv4_tables(tab, dpos + (path >= 0).sum(1, dtype=torch.int32))
        return o, depth

    def inputs():
        p = random_parents(rng, B, M, empty=False)
        p[:, 1:] = np.maximum(p[:, 1:], 0)
        lines = [kv4_masks.line(p[b], int(rng.integers(M)))[::-1][:A] for b in range(B)]
        parents.copy_(i32(p))
        path.copy_(i32([x + [-1] * (A - len(x)) for x in lines]))
        for x in (ks, vs, q):
            x.normal_()
        return p, lines

    inputs()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    saved = [x.clone() for x in (*t[:4], *[y for c in caches for y in c])]
    with torch.cuda.stream(side):
        step(t, caches)
        with torch.cuda.graph(graph, stream=side):
            out, depth = step(t, caches)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for x, y in zip((*t[:4], *[y for c in caches for y in c]), saved):
        x.copy_(y)
    for i in range(6):
        p, lines = inputs()
        dpos.copy_(i32(lens))
        graph.replay()
        want, d = step(e, eager)
        assert all(torch.equal(a, b) for a, b in zip(out + [depth], want + [d]))
        # each draft's line as a sequence of its own, over the accepted tokens' cache
        for b in range(B):
            for m in range(M):
                line = kv4_masks.line(p[b], m)[::-1]
                at = [b * M + j for j in line]
                for l in range(L):
                    alone = kv4.KV4(*(x[b:b + 1].clone() for x in whole[l]))
                    kv4.kv4_write(ks[l, at][None], vs[l, at][None], alone, i32([lens[b]]))
                    see = (torch.arange(S, device=DEV) < int(lens[b]) + len(line)).view(1, 1, -1)
                    check(out[l][b:b + 1, m:m + 1], q[l, b:b + 1, m:m + 1], alone, see)
        for b in range(B):
            at = [b * M + j for j in lines[b]]
            for l in range(L):
                kv4.kv4_write(ks[l, at][None], vs[l, at][None], kv4.KV4(*(x[b:b + 1] for x in whole[l])), i32([lens[b]]))
            lens[b] += len(lines[b])
        for l in range(L):
            got = kv4.kv4_read(caches[l], int(lens.max()), pages=t.pages)
            for x, y in zip(got, kv4.kv4_read(whole[l], int(lens.max()))):
                assert all(torch.equal(x[b, :lens[b]], y[b, :lens[b]]) for b in range(B))
        assert int(t.state[0]) == n_pages - sum(-(-int(n) // page) for n in lens)
