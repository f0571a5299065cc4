"""What the entry points around the MXFP4 cache (trees, paths, tables, slots) refuse, on the CPU: the C ABI's checks by
addresses that are never read, and the torch binding's by CPU tensors."""
import pytest
import torch

from moe_fused_inference_amd import _lib, kv4

P = 1 << 20


def _refused(rc, text):
    assert rc == -1
    assert text in _lib.load().mxfp4_last_error().decode()


def test_tree_masks():
    def call(parents=P, tree=P, depth=P, B=2, M=5):
        return _lib.load().mxfp4_tree_masks(parents, tree, depth, B, M, None)

    for kw in (dict(parents=None), dict(tree=None), dict(depth=None)):
        _refused(call(**kw), "null pointer")
    for kw in (dict(B=0), dict(B=-1), dict(B=65536), dict(M=0), dict(M=-3), dict(M=4097), dict(M=2 ** 31 - 1)):
        _refused(call(**kw), "tree_masks: B=")


def test_keep():
    def call(kq=P, vs=P, layers=2, pages=None, n_pages=4, page=64, max_pages=0, dpos=P, path=P, B=2, A=3, Hkv=4, D=128, table=True):
        t = [_lib.ptr_array([x, x] if x is not None else [P, None]) for x in (kq, P, P, vs)]
        return _lib.load().mxfp4_kv4_keep(*(t if table else [None] * 4), layers, pages, n_pages, page, max_pages, dpos, path, B, A, Hkv, D, None)

    for kw in (dict(dpos=None), dict(path=None), dict(table=False)):
        _refused(call(**kw), "null pointer")
    _refused(call(kq=None), "null cache pointer")           # of the second layer
    _refused(call(vs=P + 4), "16-byte")
    _refused(call(layers=0), "n_layers=0")
    _refused(call(layers=65536), "n_layers")
    _refused(call(A=0), "A=0")
    _refused(call(B=0), "B=0")
    _refused(call(B=5), "as many pages")
    _refused(call(D=96), "D=96")
    _refused(call(page=24), "multiple of 16")
    _refused(call(pages=P, page=48, max_pages=2), "power of two")
    _refused(call(pages=P), "max_pages")
    _refused(call(B=65535, Hkv=300, pages=P, max_pages=1), "B*Hkv")


def test_tables():
    def call(pages=P, span=P, free=P, state=P, lens=P, news=P, window=0, sinks=0, B=4, max_pages=8, n_pages=32, page=64, starts=P, slots=P, seq=P,
             pos=P, T=9):
        return _lib.load().mxfp4_kv4_tables(pages, span, free, state, lens, news, window, sinks, B, max_pages, n_pages, page, starts, slots, seq,
                                            pos, T, None)

    for k in ("pages", "span", "free", "state", "lens"):
        _refused(call(**{k: None}), "null pointer")
    _refused(call(span=P + 4), "8-byte")
    _refused(call(state=P + 4), "8-byte")
    _refused(call(slots=P + 4), "8-byte")
    for b in (0, -1, 4097, 2 ** 31 - 1):
        _refused(call(B=b), "B=%d" % b)
    _refused(call(max_pages=0), "max_pages=0")
    _refused(call(n_pages=0), "n_pages=0")
    for page in (0, -16, 8, 24, 48):
        _refused(call(page=page), "page=%d" % page)
    _refused(call(max_pages=1 << 25), "2^30")
    _refused(call(max_pages=1 << 20, page=16, B=2048), "too large")
    _refused(call(window=-1), "window=-1")
    _refused(call(sinks=4), "sinks=4")
    _refused(call(window=5, sinks=-4), "sinks=-4")
    _refused(call(news=None), "go together")
    _refused(call(starts=None), "go together")
    _refused(call(T=-1), "T=-1")
    _refused(call(T=2 ** 30 + 1), "T=")
    for k in ("slots", "seq", "pos"):
        _refused(call(**{k: None}), "a place for them")
    _refused(call(news=None, starts=None), "a place for them")


def test_write_slots():
    def call(k=P, slots=P, dt=0, ld=512, page=48, n_pages=2, T=3, Hkv=4, D=128, kq=P):
        return _lib.load().mxfp4_kv4_write_slots(k, P, dt, ld, ld, kq, P, P, P, n_pages, page, slots, T, Hkv, D, None)

    _refused(call(k=None), "null")
    _refused(call(slots=None), "null")
    _refused(call(kq=None), "null cache")
    _refused(call(dt=3), "dtype")
    _refused(call(ld=511), "stride")
    _refused(call(page=24), "multiple of 16")
    _refused(call(n_pages=0), "n_pages")
    _refused(call(T=0), "T=0")
    _refused(call(D=96), "D=96")
    _refused(call(T=2 ** 31 - 1), "too large")
    _refused(call(n_pages=1 << 20, page=1 << 12), "head rows")


def test_binding():
    cache = kv4.empty_cache(2, 32, 4, 128, device="cpu")
    d, x = torch.zeros(2, dtype=torch.int32), torch.zeros((3, 4, 128))
    t = kv4.page_tables(2, 4, 8, 16, device="cpu")
    assert t.pages.tolist() == [[-1] * 4] * 2 and t.free.tolist() == [7, 6, 5, 4, 3, 2, 1, 0] and t.state.tolist() == [8, 0] and t.page == 16
    for call in (lambda: kv4.tree_masks(torch.zeros((2, 3), dtype=torch.int32)), lambda: kv4.kv4_keep(cache, d, torch.zeros((2, 3), dtype=torch.int32)),
                 lambda: kv4.kv4_tables(t, d), lambda: kv4.kv4_write_slots(x, x, cache, torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="must be cuda"):
            call()
    for bad in (dict(B=0), dict(max_pages=0), dict(n_pages=0), dict(page=8), dict(page=24), dict(page=0), dict(window=0), dict(sinks=3),
                dict(window=4, sinks=-1)):
        a = dict(B=2, max_pages=4, n_pages=8, page=16)
        a.update(bad)
        with pytest.raises(RuntimeError):
            kv4.page_tables(**a, device="cpu")
