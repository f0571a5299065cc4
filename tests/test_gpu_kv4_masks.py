"""GPU tests of attention over the MXFP4 cache with a window and sinks, and over trees of drafts (kv4.attn_decode4)."""
import numpy as np
import pytest
import torch

from moe_fused_inference_amd import _lib, kv4
from oracle import kv4_masks
from oracle import mxfp4 as fmt
from tests.gpu_helpers import DEV, np_
from tests.kv4_mask_helpers import DT, Call, check, i32, random_parents

pytestmark = pytest.mark.gpu

WINDOWS = [
    # B, M, Hkv, G, D, page, S, dpos, q, o, window, sinks
    (1, 1, 4, 8, 128, 0, 64, [37], "bf16", "fp32", 1, 0),                         # itself alone
    (1, 1, 4, 8, 128, 0, 64, [37], "bf16", "bf16", 7, 1),
    (1, 1, 2, 4, 64, 0, 4096, [4095], "fp16", "fp32", 100, 33),
    (1, 1, 4, 8, 128, 0, 8192, [8000], "bf16", "fp32", 4096, 4),                  # shares
    (1, 1, 4, 8, 128, 0, 8192, [5], "bf16", "fp32", 4096, 4),                     # fewer than the window
    (1, 1, 1, 16, 128, 0, 2048, [1999], "bf16", "fp32", 64, 700),                 # more sinks than window
    (1, 1, 1, 4, 64, 0, 2048, [1000], "bf16", "fp32", 500, 501),                  # they meet
    (1, 1, 1, 4, 64, 0, 2048, [1000], "bf16", "fp32", 500, 470),                  # or nearly
    (1, 9, 4, 8, 128, 0, 8192, [7771], "bf16", "fp32", 1000, 4),                  # more than 16 rows
    (1, 16, 1, 1, 64, 0, 1600, [1300], "bf16", "fp32", 5, 3),                     # fewer than the tokens
    (1, 40, 1, 3, 128, 0, 1600, [1300], "bf16", "fp16", 5, 3),
    (1, 4, 1, 3, 128, 0, 32, [-2], "bf16", "fp32", 2, 1),                         # tokens before the cache
    (1, 5, 2, 7, 128, 0, 112, [110], "bf16", "fp32", 30, 0),                      # and past it
    (1, 70, 2, 4, 64, 0, 512, [480], "bf16", "fp32", 30, 2),
    (1, 3, 2, 7, 128, 0, 256, [2 ** 31 - 2], "bf16", "fp32", 30, 9),
    (3, 1, 2, 4, 128, 16, 480, [0, 31, 479], "bf16", "fp32", 33, 16),
    (7, 3, 5, 3, 64, 16, 1360, [0, 15, 16, -3, 700, 1357, 64], "fp16", "fp32", 100, 1),
    (5, 2, 3, 12, 128, 64, 640, [638, 63, 64, -2, 127], "bf16", "bf16", 64, 64),
    (70, 1, 1, 2, 64, 32, 4096, [(i * 337) % 4096 - 3 * (i % 9 == 0) for i in range(70)], "bf16", "fp32", 300, 5),
    (48, 1, 4, 8, 128, 64, 2048, [(i * 731) % 2048 for i in range(48)], "bf16", "bf16", 500, 16),
    (2, 1, 8, 1, 128, 128, 1024, [1023, 2 ** 31 - 1], "bf16", "fp32", 129, 127),
    (33, 1, 4, 2, 128, 0, 544, [(i * 61) % 545 - 1 for i in range(33)], "bf16", "fp32", 200, 0),
    (32, 1, 4, 8, 128, 0, 2048, [(i * 611) % 2048 for i in range(32)], "bf16", "fp32", 1000, 4),      # sixteen waves
    (1, 200, 2, 4, 128, 64, 2048, [1600], "bf16", "bf16", 333, 4),                # pieces of a prompt
    (2, 130, 1, 8, 64, 0, 1024, [0, 800], "fp16", "fp32", 64, 1),
    (1, 512, 4, 8, 128, 0, 4096, [3584], "bf16", "bf16", 1024, 4),
    (3, 50, 1, 5, 64, 16, 4096, [-20, 3290, 100], "fp16", "bf16", 700, 40),       # a line of more than 16 rows
    (8, 33, 8, 16, 64, 0, 64, [0, 31, -33, 30, 5, -1, 60, 20], "bf16", "fp16", 9, 2),
]

TREES = [
    # B, M, Hkv, G, D, page, S, dpos, q, o, window, sinks
    (1, 1, 4, 8, 128, 0, 64, [37], "bf16", "fp32", None, 0),
    (1, 5, 1, 3, 128, 0, 64, [0], "bf16", "fp32", None, 0),                       # nothing before it
    (1, 26, 4, 8, 128, 0, 4096, [4000], "bf16", "fp32", None, 0),
    (1, 31, 1, 1, 64, 0, 4096, [33], "fp16", "fp32", None, 0),
    (1, 16, 1, 1, 64, 0, 16384, [16000], "bf16", "bf16", None, 0),
    (1, 33, 1, 1, 64, 0, 256, [95], "bf16", "fp32", None, 0),                     # two words
    (1, 100, 2, 4, 128, 32, 1024, [777], "bf16", "bf16", None, 0),
    (1, 9, 2, 1, 64, 0, 32, [-3], "bf16", "fp32", None, 0),                       # drafts before the cache
    (1, 9, 2, 8, 64, 0, 64, [60], "bf16", "fp32", None, 0),                       # and past it
    (7, 5, 5, 3, 64, 16, 1360, [0, 15, 16, -5, 700, 1355, 64], "fp16", "fp32", None, 0),
    (16, 64, 1, 8, 128, 64, 1024, [(i * 61) % 961 for i in range(16)], "bf16", "bf16", None, 0),
    (70, 2, 2, 2, 64, 32, 512, [(i * 37) % 500 - 3 * (i % 9 == 0) for i in range(70)], "bf16", "fp32", None, 0),
    (40, 3, 1, 4, 128, 16, 4096, [(i * 331) % 4090 for i in range(40)], "bf16", "fp32", None, 0),
    (1, 26, 4, 8, 128, 0, 4096, [4000], "bf16", "fp32", 500, 4),
    (1, 26, 1, 2, 128, 0, 4096, [4000], "bf16", "fp32", 26, 1),                   # no more than the tree
    (5, 7, 2, 2, 64, 16, 2048, [3, 500, 1999, -7, 1022], "fp16", "fp32", 100, 33),
    (3, 12, 1, 1, 128, 0, 512, [0, 100, 500], "bf16", "bf16", 12, 0),
    (1, 70, 1, 4, 64, 0, 2048, [1900], "bf16", "fp32", 333, 2),
]


def _call(case, tree, **kw):
    *shape, qt, _, window, sinks = case
    return Call(*shape, qt, window, sinks, tree, **kw)


@pytest.mark.parametrize("tree,case", [(False, c) for c in WINDOWS] + [(True, c) for c in TREES],
                         ids=["window%d" % i for i in range(len(WINDOWS))] + ["tree%d" % i for i in range(len(TREES))])
def test_attention(case, tree):
    c = _call(case, tree)
    dt = DT[case[9]]
    o = c.run(dt)
    check(o, c.q, c.cache, c.see, c.pages)
    assert torch.equal(o, c.run(dt))                                     # the same bits again
    o32 = c.run()
    oq, os_ = c.run_mx()
    wq, ws = fmt.quantize_rows(fmt.bf16_round(np_(o32)).reshape(oq.shape[0], -1))
    assert np.array_equal(np_(oq), wq) and np.array_equal(np_(os_), ws)
    # what no token sees is without effect, NaN included; rows that see nothing are zeros
    assert torch.equal(o, c.run(dt, cache=c.fill_unseen())) and torch.isfinite(o).all()
    assert not o[~c.see.any(-1)].any()


@pytest.mark.parametrize("B,M,Hkv,G,D,S", [(1, 1, 4, 8, 128, 8192), (1, 6, 1, 2, 64, 2000), (3, 9, 2, 4, 128, 4096), (1, 64, 2, 4, 64, 640)])
def test_masks_that_hide_nothing(B, M, Hkv, G, D, S):
    """A window that reaches everything, and a tree that is one line: the bits of the call without."""
    dpos = [S - M - 40 * b for b in range(B)]
    c = Call(B, M, Hkv, G, D, 0, S, dpos)
    want = c.run()
    words, depth = kv4_masks.tree_masks(np.tile(np.arange(-1, M - 1, dtype=np.int32), (B, 1)))
    assert (depth == np.arange(M)).all()
    for window, sinks, tree in ((S, 5, None), (S - 1 if M > 1 else S, 0, None), (2 ** 40, 0, None), (None, 0, i32(words)), (S + M, 3, i32(words))):
        got = kv4.attn_decode4(c.q, c.cache, c.dpos, window=window, sinks=sinks, tree=tree)
        if window == S - 1:
            check(got, c.q, c.cache, torch.from_numpy(kv4_masks.sees(dpos, M, S, window)).to(DEV))
        else:
            assert torch.equal(got, want)


@pytest.mark.parametrize("B,M,Hkv,G,D,page,S,window,sinks,tree", [
    (3, 1, 2, 4, 128, 16, 2048, 200, 5, False), (2, 1, 1, 16, 64, 64, 8192, 1000, 100, False), (2, 9, 2, 4, 128, 16, 2048, 90, 20, False),
    (1, 6, 2, 2, 64, 32, 4096, 77, 0, False), (2, 7, 1, 2, 64, 16, 2048, 100, 3, True), (1, 40, 1, 4, 128, 32, 4096, 100, 3, True)])
def test_pages_behind_the_window_are_gone(B, M, Hkv, G, D, page, S, window, sinks, tree):
    """A table without the pages that no token sees, whose rows are others' by now: the same bits."""
    dpos = [S - M - 333 * b for b in range(B)]
    c = Call(B, M, Hkv, G, D, page, S, dpos, window=window, sinks=sinks, tree=tree)
    need = c.see.any(1).view(B, -1, page).any(-1)
    assert not need.all()
    for dt in (torch.float32, torch.bfloat16):
        o = c.run(dt)
        for gone in (-1, c.cache[0].shape[0], -2 ** 31):
            pages = torch.where(need, c.pages, gone).to(torch.int32)
            assert torch.equal(o, c.run(dt, cache=c.fill_unseen(), pages=pages))


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("B,M,Hkv,G,D,page,S,holes", [(2, 2, 2, 4, 128, 16, 640, 12), (1, 7, 1, 5, 64, 32, 1024, 9), (2, 20, 1, 4, 128, 16, 640, 12)])
def test_holes(B, M, Hkv, G, D, page, S, holes, tree):
    """Pages that are none among those that are seen."""
    c = Call(B, M, Hkv, G, D, page, S, [S - M - 100 * b for b in range(B)], window=300, sinks=40, tree=tree, holes=holes)
    for dt in (torch.float32, torch.bfloat16):
        check(c.run(dt), c.q, c.cache, c.see, c.pages)


def test_masks_of_any_bits():
    """A tree's words may name any drafts, later ones and none; bits from M on are without effect."""
    rng = np.random.default_rng(5)
    for M, G, window in ((5, 2, None), (40, 2, None), (40, 2, 200), (5, 2, 9)):
        words = rng.integers(-2 ** 31, 2 ** 31, (2, M, (M + 31) // 32)).astype(np.int32)
        words[0, 1], words[1, 3] = 0, 0
        keep = words.copy()
        if M % 32:
            keep[..., -1] &= (1 << (M % 32)) - 1
        c = Call(2, M, 1, G, 64, 0, 768, [0, 600], words=keep, window=window, sinks=2 if window else 0)
        o = c.run()
        check(o, c.q, c.cache, c.see)
        assert not o[0, 1].any()                       # no position at all
        c.tree = i32(words)
        assert torch.equal(o, c.run())


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("M,Hkv,G,D,window", [(3, 1, 4, 128, 40), (6, 1, 2, 64, 33), (30, 1, 2, 128, 40), (30, 2, 4, 64, 100), (4, 1, 4, 64, 1000)])
def test_values_that_are_not_finite(M, Hkv, G, D, window, tree):
    """An infinity or NaN among values reaches exactly the tokens that see it; the others' bits stay."""
    S, base = 4096, 2000
    for at in (3, 34, base - window - 1, base - window + 1, base - window + 3, base - 5, base, base + 1, base + M - 1):
        c = Call(1, M, Hkv, G, D, 0, S, [base], window=window, sinks=35, tree=tree, seed=at)
        for dt in (torch.float32, torch.bfloat16):
            o = c.run(dt)
            bad = kv4.KV4(*(x.clone() for x in c.cache))
            col = at % D
            bad.vs[0, :, at, col // 32] = 254
            bad.vq[0, :, at, col // 32 * 16:col // 32 * 16 + 16] = 0        # (zeros of a large scale are zeros)
            clean = c.run(dt, cache=kv4.KV4(*bad))
            bad.vq[0, :, at, col // 2] = 0x07 << 4 * (col & 1)
            got = c.run(dt, cache=bad)
            hit = torch.zeros_like(o, dtype=torch.bool)
            hit[0, :, :, col] = c.see[0, :, at, None]
            assert not torch.isfinite(got[hit]).any()
            assert torch.equal(got[~hit], clean[~hit])
            assert torch.isfinite(clean).all() and torch.equal(o[~c.see[..., at]], clean[~c.see[..., at]])


def test_query_rows_of_infinities_and_nan():
    for M, tree in ((1, False), (5, False), (40, False), (5, True), (40, True)):
        c = Call(1, M, 2, 8, 128, 0, 512, [400], window=100, sinks=3, tree=tree)
        o = c.run()
        bad = c.q.clone()
        bad[0, 0, 0, 3], bad[0, M - 1, 9, 127], bad[0, M - 1, 15, 64] = float("inf"), float("-inf"), float("nan")
        ob = c.run(q=bad)
        rows = torch.zeros((1, M, 16), dtype=torch.bool, device=DEV)
        rows[0, 0, 0] = rows[0, M - 1, 9] = rows[0, M - 1, 15] = True
        assert torch.isnan(ob[rows]).all() and torch.equal(ob[~rows], o[~rows])


def test_a_window_far_in_a_cache_past_four_gigabytes():
    """Offsets of a long cache: a window and sinks at the ends of its last sequence."""
    B, Hkv, D, S, n = 9, 8, 128, 1 << 20, 700
    cache = kv4.empty_cache(B, S, Hkv, D)
    k, v = (torch.randn((B, n, Hkv, D), device=DEV).bfloat16() for _ in range(2))
    kv4.kv4_write(k, v, cache, i32([-n] * (B - 1) + [S - n]))
    kv4.kv4_write(k[:, :9], v[:, :9], cache, i32([-n] * (B - 1) + [0]))
    q = torch.randn((B, 1, 16, D), device=DEV).bfloat16()
    o = kv4.attn_decode4(q, cache, i32([-1] * (B - 1) + [S - 1]), window=500, sinks=7)
    assert not o[:-1].any()
    small = kv4.empty_cache(1, 512, Hkv, D)           # what it sees, side by side
    for x, y in zip(small, cache):
        x[0, :, :7], x[0, :, 7:507] = y[-1, :, :7], y[-1, :, S - 500:]
    check(o[-1:], q[-1:], small, (torch.arange(512, device=DEV) < 507).view(1, 1, -1))
    del cache
    torch.cuda.empty_cache()


@pytest.mark.parametrize("B,M,S,window,tree", [(1, 1, 8192, 3000, False), (1, 9, 8192, 500, False), (3, 6, 4096, 100, True), (40, 1, 4096, 700, False),
                                               (40, 1, 512, 100, False), (1, 26, 4096, None, True)])
def test_replays(B, M, S, window, tree):
    """Captured once and replayed over other lengths and trees, with eager work between, is the eager result."""
    rng = np.random.default_rng(23 + B)
    c = Call(B, M, 1, 8, 128, 0, S, [5] * B, window=window, sinks=3 if window else 0, tree=tree)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        c.run()
        with torch.cuda.graph(graph, stream=side):
            o = c.run()
    torch.cuda.current_stream().wait_stream(side)
    for hi in (S, 40, S // 2, 1):
        c.dpos.copy_(i32(rng.integers(-M, hi, B)))
        c.q.normal_()
        if tree:
            c.tree.copy_(i32(kv4_masks.tree_masks(random_parents(rng, B, M))[0]))
        graph.replay()
        assert torch.equal(o, c.run()) and torch.isfinite(o).all()


def test_two_at_once_on_other_streams():
    c = Call(2, 3, 4, 8, 128, 0, 4096, [4000, 2500], window=1000, sinks=4, tree=True)
    qs = [torch.randn_like(c.q) for _ in range(2)]
    want = [c.run(q=q) for q in qs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(c.run(q=qs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_rows_behind_the_outputs_and_the_workspace_stay():
    lib = _lib.load()
    for M, window, tree in ((1, 300, False), (9, 300, False), (9, None, True)):
        c = Call(2, M, 1, 4, 128, 0, 4096, [4000, 411], window=window, sinks=4 if window else 0, tree=tree)
        n = lib.mxfp4_attn_kv4_masked_workspace_size(2, M, 4, 1, 128, 4096, window or 0, c.sinks)
        ws = torch.full((n + 64,), 99, dtype=torch.uint8, device=DEV)
        o = torch.full((2 * M + 1, 4, 128), 77.0, device=DEV)
        _lib.check(lib.mxfp4_attn_kv4_masked(c.q.data_ptr(), 0, 512, *[t.data_ptr() for t in c.cache], None, 2, 4096, 0, c.dpos.data_ptr(),
                                             window or 0, c.sinks, None if c.tree is None else c.tree.data_ptr(), o.data_ptr(), 2, None, None,
                                             2, M, 4, 1, 128, ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream), "attn_kv4")
        assert torch.equal(o[:-1].view(2, M, 4, 128), c.run()) and (o[-1] == 77).all() and (ws[n:] == 99).all()


def test_shapes_without_work_and_refusals():
    cache, dp = kv4.empty_cache(2, 32, 2, 64), i32([3, 4])
    e = torch.empty((2, 0, 2, 64), dtype=torch.bfloat16, device=DEV)
    assert kv4.attn_decode4(e, cache, dp, window=5, sinks=1).shape == (2, 0, 2, 64)
    assert kv4.attn_decode4(e, cache, dp, tree=torch.empty((2, 0, 0), dtype=torch.int32, device=DEV)).shape == (2, 0, 2, 64)
    q = torch.zeros((2, 3, 2, 64), dtype=torch.bfloat16, device=DEV)
    t = torch.zeros((2, 3, 1), dtype=torch.int32, device=DEV)
    for bad in (dict(window=0), dict(window=-1), dict(sinks=1), dict(window=4, sinks=-1), dict(tree=t[:1]), dict(tree=t[:, :2]), dict(tree=t.long()),
                dict(tree=t[..., 0]), dict(tree=t.cpu()), dict(tree=t, window=2), dict(tree=t.expand(2, 3, 2)), dict(tree=t[..., :0])):
        for call in (kv4.attn_decode4, kv4.attn_decode4_mx):
            with pytest.raises(RuntimeError):
                call(q, cache, dp, **bad)
