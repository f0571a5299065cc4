"""What the MXFP4 cache's entry points refuse, on the CPU: the C ABI's checks by addresses that are never
read, and the torch binding's by CPU tensors."""
import ctypes

import pytest
import torch

from moe_fused_inference_amd import _lib, kv4

P = 1 << 20      # an aligned address; every call below is refused before a launch


def _cache(**kw):
    a = dict(kq=P, ks=P, vq=P, vs=P, pages=None, n_pages=4, page=64, max_pages=0)
    a.update(kw)
    return [a[k] for k in ("kq", "ks", "vq", "vs", "pages", "n_pages", "page", "max_pages")]


BAD_CACHE = [({"kq": None}, "null cache"), ({"vs": P + 4}, "16-byte"), ({"n_pages": 0}, "n_pages"), ({"page": 24}, "multiple of 16"),
             ({"page": 0}, "multiple of 16"), ({"page": 48, "pages": P, "max_pages": 2}, "power of two"),
             ({"pages": P, "max_pages": 0}, "max_pages"), ({"n_pages": 1}, "as many pages"),
             ({"pages": P, "page": 1 << 16, "max_pages": 1 << 15}, "2^30")]


def _write(cache=None, D=128, B=2, M=1, Hkv=4, dt=0, k=P, dpos=P, ld=None):
    return _lib.load().mxfp4_kv4_write(k, P, dt, ld or Hkv * D, ld or Hkv * D, *(cache or _cache()), dpos, B, M, Hkv, D, None)


def _read(cache=None, D=128, B=2, n=1, Hkv=4, dt=0, k=P):
    return _lib.load().mxfp4_kv4_read(*(cache or _cache()), None, k, P, dt, B, n, Hkv, D, None)


def _attn(cache=None, D=128, B=2, M=1, Hq=8, Hkv=4, qdt=0, odt=2, q=P, o=P, oq=None, os_=None, ldq=None, ws=P, wsb=1 << 40, dpos=P):
    return _lib.load().mxfp4_attn_kv4(q, qdt, ldq or Hq * D, *(cache or _cache(page=8192)), dpos, o, odt, oq, os_, B, M, Hq, Hkv, D,
                                      ws, wsb, None)


def _rope(cache=None, D=128, B=2, M=1, Hq=8, Hkv=4, qkv=P, dpos=P):
    return _lib.load().mxfp4_qk_norm_rope_kv4(qkv, P, P, 1e-6, 1e6, *(cache or _cache()), dpos, B, M, Hq, Hkv, D, P, None)


def _refused(rc, text):
    assert rc == -1
    assert text in _lib.load().mxfp4_last_error().decode()


@pytest.mark.parametrize("kw,text", BAD_CACHE)
@pytest.mark.parametrize("call", [_write, _read, _attn, _rope])
def test_bad_caches(call, kw, text):
    _refused(call(_cache(**kw)), text)


@pytest.mark.parametrize("call", [_write, _read, _attn, _rope])
def test_bad_sizes(call):
    _refused(call(D=96), "D=96")
    _refused(call(B=0), "B=0")
    _refused(call(Hkv=0), "Hkv=0")
    _refused(call(**({"n": 0} if call is _read else {"M": 0})), "n=0" if call is _read else "M=0")


def test_write_refuses():
    _refused(_write(dt=3), "dtype")
    _refused(_write(k=None), "null")
    _refused(_write(dpos=None), "null")
    _refused(_write(ld=100), "stride")
    _refused(_write(M=1 << 30, B=4), "too large")


def test_read_refuses():
    _refused(_read(dt=-1), "dtype")
    _refused(_read(k=None), "null")
    _refused(_read(k=P + 8), "16-byte")
    _refused(_read(n=1 << 30, B=4), "too large")


def test_attn_refuses():
    _refused(_attn(qdt=2), "q dtype")
    _refused(_attn(odt=5), "o dtype")
    _refused(_attn(Hq=6), "Hq=6")
    _refused(_attn(q=None), "null")
    _refused(_attn(dpos=None), "null")
    _refused(_attn(q=P + 2), "aligned")
    _refused(_attn(ldq=8 * 128 + 4), "16-byte")
    _refused(_attn(ldq=8 * 64), "apart")
    _refused(_attn(o=None), "no output")
    _refused(_attn(oq=P), "together")
    _refused(_attn(o=P + 4), "aligned")
    _refused(_attn(ws=None), "workspace")
    _refused(_attn(ws=P + 4), "workspace")
    _refused(_attn(wsb=16), "workspace")
    _refused(_attn(M=65536), "M=65536")


def test_rope_refuses():
    _refused(_rope(D=64), "D=64")
    _refused(_rope(Hq=6), "Hq=6")
    _refused(_rope(qkv=None), "null")


def test_workspace_size():
    size = _lib.load().mxfp4_attn_kv4_workspace_size
    assert size.restype is ctypes.c_size_t
    assert size(0, 1, 8, 4, 128, 64) == 0 and size(1, 1, 7, 4, 128, 64) == 0
    assert size(1, 1, 8, 4, 128, 128) == 0                       # one share: nothing to merge
    assert size(1, 1, 32, 4, 128, 32768) % (32 * 132 * 4) == 16       # records, and a sequence's place
    assert size(1, 1, 32, 4, 128, 32768) <= (512 // 4 + 1) * 32 * 132 * 4


def test_binding_refuses_cpu_tensors_and_bad_allocations():
    t = kv4.empty_cache(2, 32, 4, 128, device="cpu")
    d = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros((2, 1, 4, 128), dtype=torch.bfloat16)
    for call in (lambda: kv4.kv4_write(x, x, t, d), lambda: kv4.kv4_read(t, 4), lambda: kv4.attn_decode4(x, t, d),
                 lambda: kv4.attn_decode4_mx(x, t, d)):
        with pytest.raises(RuntimeError, match="must be cuda"):
            call()
    for bad in (dict(D=96), dict(page=24), dict(page=0), dict(n_pages=0), dict(Hkv=0)):
        a = dict(n_pages=1, page=32, Hkv=4, D=128)
        a.update(bad)
        with pytest.raises(RuntimeError, match="cache needs"):
            kv4.empty_cache(a["n_pages"], a["page"], a["Hkv"], a["D"], device="cpu")


@pytest.mark.parametrize("call", [_write, _read, _attn, _rope])
def test_more_head_rows_than_32_bits(call):
    _refused(call(_cache(n_pages=1 << 15, page=1 << 15)), "head rows")      # times four heads: 2^32


def _on_cpu(Hkv=4, D=128, n_pages=2, pages=None):
    """Every entry of the binding on CPU tensors: (name, call).  What is refused by its shape is refused before
    the device is looked at."""
    cache = [torch.zeros((n_pages, Hkv, 32, w), dtype=torch.uint8) for w in (D // 2, D // 32) * 2]
    d = torch.zeros(n_pages if pages is None else pages.shape[0], dtype=torch.int32)
    x = torch.zeros((d.numel(), 1, Hkv, D), dtype=torch.bfloat16)
    q = torch.zeros((d.numel(), 1, 8, D), dtype=torch.bfloat16)
    return [("write", lambda: kv4.kv4_write(x, x, cache, d, pages)), ("read", lambda: kv4.kv4_read(cache, 4, d, pages)),
            ("attn", lambda: kv4.attn_decode4(q, cache, d, pages)), ("attn_mx", lambda: kv4.attn_decode4_mx(q, cache, d, pages))]


@pytest.mark.parametrize("pages", [torch.zeros((2, 0), dtype=torch.int32), torch.zeros((2, 3), dtype=torch.int32)[:, :0].contiguous()])
def test_binding_refuses_a_table_of_no_columns(pages):
    """It has no address, and no address means that sequence b is page b."""
    for _, call in _on_cpu(pages=pages):
        with pytest.raises(RuntimeError, match="a column at least"):
            call()


def test_binding_refuses_a_cache_of_no_heads():
    """The query heads would be divided by none, which ends the process."""
    for _, call in _on_cpu(Hkv=0):
        with pytest.raises(RuntimeError, match="a kv head at least"):
            call()


def test_workspace_size_of_calls_that_are_refused():
    """0, whatever the sizes: groups of rows past 32 bits were divided by (2^32 of them are none)."""
    size, top = _lib.load().mxfp4_attn_kv4_workspace_size, 2 ** 31 - 1
    assert size(1, 65535, 16, 1, 128, 4096) >= 0 and size(2, 512, 32, 4, 128, 1 << 30) > 0
    for a in ((1, 1 << 30, 128, 1, 128, 4096), (1, top, 64, 1, 128, 4096), (1, 65536, 1, 1, 128, 4096), (1, 65535, 17, 1, 128, 4096),
              (1, 1, 65536, 1, 128, 4096), (65536, 1, 8, 8, 128, 4096), (2, 1, 8, 4, 128, top), (2, 1, 8, 4, 96, 4096),
              (2, 1, 8, 4, 128, -5), (-1, 1, 8, 4, 128, 64), (top, top, top, 1, 128, top)):
        assert size(*a) == 0, a


def test_launches_of_more_threads_than_32_bits():
    """Refused by name before a launch: rows of 2^32 threads of eight values, and head counts past 31 bits."""
    big = _cache(n_pages=64, page=1 << 14, pages=P, max_pages=1 << 10)
    for D, M in ((128, 1 << 22), (64, 1 << 23)):                   # times 64 sequences: 2^28 (2^29) tokens, 2^32 threads a head
        _refused(_write(big, D=D, B=64, M=M, Hkv=1), "too large")
        _refused(_read(big, D=D, B=64, n=M, Hkv=1), "too large")
    _refused(_rope(big, B=64, M=1 << 18), "M=262144")              # 2^24 workgroups of 256
    _refused(_rope(Hq=2 ** 31 - 4, Hkv=4), "Hq=2147483644")
    # rows to merge, a workgroup each (two sequences of 2^24 positions, 2^24 rows of q)
    _refused(_attn(_cache(n_pages=2, page=1 << 14, pages=P, max_pages=1 << 10), B=2, M=65535, Hq=257, Hkv=257, wsb=1 << 60), "too large")


def test_binding_takes_an_empty_batch_whatever_its_table():
    """No sequence, no work: what is left to refuse is the device."""
    for shape in ((0, 0), (0, 3)):
        for _, call in _on_cpu(pages=torch.zeros(shape, dtype=torch.int32)):
            with pytest.raises(RuntimeError, match="must be cuda"):
                call()
