"""What the masked attention's entry points refuse, on the CPU: by addresses that are never read, and CPU tensors."""
import pytest
import torch

from moe_fused_inference_amd import _lib, kv4

P = 1 << 20


def _attn(window=0, sinks=0, tree=None, B=2, M=3, Hq=8, Hkv=4, D=128, page=8192, ws=P, wsb=1 << 40, o=P, q=P, dpos=P):
    return _lib.load().mxfp4_attn_kv4_masked(q, 0, Hq * D, P, P, P, P, None, 4, page, 0, dpos, window, sinks, tree, o, 2, None, None, B, M, Hq, Hkv,
                                             D, ws, wsb, None)


def _refused(rc, text):
    assert rc == -1
    assert text in _lib.load().mxfp4_last_error().decode()


def test_refusals():
    _refused(_attn(window=-1), "window=-1")
    _refused(_attn(window=5, sinks=-1), "sinks=-1")
    _refused(_attn(sinks=1), "without a window")
    _refused(_attn(window=2, tree=P), "for a tree of 3")
    _refused(_attn(tree=P + 2), "4-byte aligned")
    for kw in (dict(), dict(window=4000, sinks=4), dict(tree=P)):
        _refused(_attn(**kw, ws=None), "workspace")
        _refused(_attn(**kw, wsb=16), "workspace")
        _refused(_attn(**kw, o=None), "no output")
        _refused(_attn(**kw, q=None), "null")
        _refused(_attn(**kw, dpos=None), "null")
        _refused(_attn(**kw, M=65536), "M=65536" if not kw.get("tree") else "M=65536")
        _refused(_attn(**kw, Hq=6), "Hq=6")


def test_workspace_sizes():
    plain, size = _lib.load().mxfp4_attn_kv4_workspace_size, _lib.load().mxfp4_attn_kv4_masked_workspace_size
    for a in ((1, 1, 32, 4, 128, 32768), (3, 9, 32, 4, 128, 4096), (1, 1, 8, 4, 128, 64), (0, 1, 8, 4, 128, 64)):
        assert size(*a, 0, 0) == plain(*a)
        assert size(*a, 2 ** 31 - 1, 2 ** 31 - 1) == plain(*a)
    assert 0 < size(1, 1, 32, 4, 128, 32768, 1024, 4) <= plain(1, 1, 32, 4, 128, 32768)
    assert size(1, 1, 32, 4, 128, 32768, 1, 0) <= size(1, 1, 32, 4, 128, 32768, 1024, 4)
    for a in ((1, 1, 32, 4, 128, 32768, -1, 0), (1, 1, 32, 4, 128, 32768, 5, -1), (1, 1 << 30, 128, 1, 128, 4096, 5, 0), (1, 1, 7, 4, 128, 64, 5, 0),
              (2 ** 31 - 1,) * 8):
        assert size(*a) == 0, a


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that are never read: needs a machine without a GPU")
@pytest.mark.parametrize("B,M,Hq,Hkv", [(1, 1, 32, 4), (8, 1, 32, 4), (8, 2, 16, 8), (100, 1, 8, 8), (1, 40, 32, 4), (3, 9, 8, 2)])
@pytest.mark.parametrize("tree", [None, P])
def test_the_workspace_that_a_call_asks_for(B, M, Hq, Hkv, tree):
    """What the size function says is enough, and a byte less is not: at every window, also those that reach everything."""
    page, size = 4096, _lib.load().mxfp4_attn_kv4_masked_workspace_size
    for window in [0] + sorted({max(M, 1 << i) + j for i in range(14) for j in (0, 1)} | {page + j for j in (-70, -33, -1, 0, M - 1, M, M + 1)}):
        for sinks in (0, 4) if window else (0,):
            n = size(B, M, Hq, Hkv, 128, page, window, sinks)
            kw = dict(window=window, sinks=sinks, tree=tree, B=B, M=M, Hq=Hq, Hkv=Hkv, page=page)
            args = lambda wsb: _lib.load().mxfp4_attn_kv4_masked(P, 0, Hq * 128, P, P, P, P, None, B, page, 0, P, window, sinks, tree, P, 2, None, None, B, M,
                                                                 Hq, Hkv, 128, P if wsb else None, wsb, None)
            assert args(n) == 100, kw         # hipErrorNoDevice: it came to the launch
            if n:
                assert args(n - 1) == -1, kw


def test_binding():
    cache = kv4.empty_cache(2, 32, 4, 128, device="cpu")
    d, q = torch.zeros(2, dtype=torch.int32), torch.zeros((2, 3, 4, 128), dtype=torch.bfloat16)
    for call in (kv4.attn_decode4, kv4.attn_decode4_mx):
        with pytest.raises(RuntimeError, match="must be cuda"):
            call(q, cache, d, window=4, sinks=1)
