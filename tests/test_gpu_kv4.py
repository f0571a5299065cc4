"""GPU tests of the MXFP4 KV cache: write, read-back and attention (kv4.py, the kv4 entries of the C ABI).

Bytes and values are compared exactly; attention against 64 bits within the bound that oracle/kv4.py derives from the
operands, plus half a step of the output type.
"""
import numpy as np
import pytest
import torch

from moe_fused_inference_amd import _lib, kv4
from oracle import kv4 as ref
from oracle import mxfp4 as fmt
from tests.gpu_helpers import DEV, np_

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _values(rng, shape):
    """Keys or values whose blocks differ in size, with zeros, ties and signed zeros."""
    x = rng.standard_normal(shape).astype(np.float32) * np.exp(rng.standard_normal(shape[-2:])).astype(np.float32)
    x.reshape(-1)[:8] = [0.0, -0.0, 0.25, -0.75, 2.5, -5.0, 6.0, 1e-3]
    return x


def _host_cache(rng, n_pages, Hkv, page, D):
    """Random rows: every nibble, scales of a factor 2^8."""
    def half():
        return [rng.integers(0, 256, (n_pages, Hkv, page, D // 2), dtype=np.uint8),
                rng.integers(121, 130, (n_pages, Hkv, page, D // 32), dtype=np.uint8)]
    return half() + half()


def _dev(cache):
    return kv4.KV4(*(torch.from_numpy(c).to(DEV) for c in cache))


def _i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def _table(rng, B, max_pages, n_pages, holes=0):
    t = rng.permutation(n_pages)[:B * max_pages].reshape(B, max_pages).astype(np.int32)
    for i in range(holes):
        t[rng.integers(B), rng.integers(max_pages)] = (-1, n_pages, -2 ** 31, 2 ** 31 - 1)[i % 4]
    return t


# ------------------------------------------------------------------ write and read
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,M,Hkv,D,page,dpos", [
    (1, 1, 4, 128, 0, [5]), (1, 37, 4, 128, 0, [0]), (3, 9, 5, 64, 16, [0, 11, 43]), (4, 3, 1, 128, 32, [-3, -1, 94, 95]),
    (2, 20, 3, 128, 64, [50, 2 ** 31 - 5]), (2, 1, 2, 64, 0, [-2 ** 31, 15])])
def test_write_and_read_back(dtype, B, M, Hkv, D, page, dpos):
    rng = np.random.default_rng(B * 100 + M + D)
    n_pages, P = (B * 3 + 2, page) if page else (B, 48)
    cache = _host_cache(rng, n_pages, Hkv, P, D)
    pages = _table(rng, B, 3, n_pages, holes=2) if page else None
    k, v = (torch.from_numpy(_values(rng, (B, M, Hkv, D))).to(DT[dtype]) for _ in range(2))
    dev, dp, tab = _dev(cache), _i32(dpos), None if pages is None else _i32(pages)
    kv4.kv4_write(k.to(DEV), v.to(DEV), dev, dp, tab)
    ref.write(k.float().numpy(), v.float().numpy(), cache, dpos, pages)
    for got, want in zip(dev, cache):
        assert np.array_equal(np_(got), want)
    for start in (dpos, None):
        rk, rv, _ = ref.read(cache, M, dpos if start else [0] * B, pages)
        gk, gv = kv4.kv4_read(dev, M, None if start is None else dp, tab, DT[dtype])
        assert gk.dtype == DT[dtype] and gk.shape == (B, M, Hkv, D)
        # the values fit all three types
        assert np.array_equal(np_(gk.float()), rk) and np.array_equal(np_(gv.float()), rv)


def test_write_of_strange_values():
    """Infinities, NaN, denormals, the largest values and exact ties: the quantizer's own codes."""
    rng = np.random.default_rng(1)
    x = _values(rng, (1, 6, 2, 64))
    x[0, 0, 0, :4] = [np.inf, -np.inf, np.nan, 3.0]
    x[0, 1] = 0.0
    x[0, 2] = -0.0
    x[0, 3] = rng.choice(np.array([1e-40, -3e-39, 0.0], np.float32), (2, 64))
    x[0, 4] = rng.choice(np.array([3.38e38, -1.7e38, 1e30], np.float32), (2, 64))
    x[0, 5] = rng.choice(fmt.E2M1_MIDPOINTS.astype(np.float32), (2, 64)) * rng.choice([-1, 1], (2, 64))
    for dt in ("fp32", "bf16"):
        t = torch.from_numpy(x).to(DT[dt]).to(DEV)
        dev = kv4.empty_cache(1, 16, 2, 64)
        kv4.kv4_write(t, t, dev, _i32([0]))
        lib = _lib.load()
        q, s = torch.empty((12, 32), dtype=torch.uint8, device=DEV), torch.empty((12, 2), dtype=torch.uint8, device=DEV)
        _lib.check(lib.mxfp4_quantize_rows(t.data_ptr(), 2 if dt == "fp32" else 0, 0, 64, 12, 64, 64, q.data_ptr(), s.data_ptr(),
                                           torch.cuda.current_stream().cuda_stream), "quantize_rows")
        assert torch.equal(dev.kq[0, :, :6].transpose(0, 1).reshape(12, 32), q)
        assert torch.equal(dev.vs[0, :, :6].transpose(0, 1).reshape(12, 2), s)


def test_read_of_every_code():
    """Every byte under every scale code: exact in fp32 and bf16 (255: NaN), fp16 to nearest."""
    page = 4096
    host = np.zeros((1, 1, page, 32), np.uint8)
    codes = np.zeros((1, 1, page, 2), np.uint8)
    # 256 scales x 16 rows of 16 bytes, twice a row
    for c in range(256):
        for r in range(16):
            host[0, 0, c * 16 + r] = np.tile(np.arange(r * 16, r * 16 + 16, dtype=np.uint8), 2)
            codes[0, 0, c * 16 + r] = c
    dev = _dev([host, codes, host, codes])
    want = fmt.dequant_rows(host.reshape(-1, 32), codes.reshape(-1, 2))
    want[255 * 16:] = np.nan
    for dt in DT.values():
        k, v = kv4.kv4_read(dev, page, dtype=dt)
        w = torch.from_numpy(want).to(dt)
        assert torch.equal(torch.isnan(w), torch.isnan(k[0, :, 0].cpu()))
        ok = ~torch.isnan(w)
        assert torch.equal(w[ok], k[0, :, 0].cpu()[ok]) and torch.equal(w[ok], v[0, :, 0].cpu()[ok])


def test_write_of_views():
    """Slices of a fused projection (one token stride), of odd alignment, and views that have to be copied."""
    rng = np.random.default_rng(2)
    B, M, Hq, Hkv, D = 2, 3, 4, 2, 64
    qkv = torch.randn((B * M, (Hq + 2 * Hkv) * D), device=DEV)
    part = qkv.view(B, M, Hq + 2 * Hkv, D)
    odd = torch.randn(B * M * Hkv * D + 1, device=DEV).bfloat16()[1:].view(B, M, Hkv, D)
    views = [(part[:, :, Hq:Hq + Hkv], part[:, :, Hq + Hkv:]), (odd, odd.clone()),
             (part.transpose(0, 1).contiguous().transpose(0, 1)[:, :, :Hkv], part[:, :, ::2][:, :, :Hkv]),
             (part[:, :, :1].expand(B, M, Hkv, D), part[:, :, :Hkv])]
    for k, v in views:
        a, b = kv4.empty_cache(B, 32, Hkv, D), kv4.empty_cache(B, 32, Hkv, D)
        dp = _i32(rng.integers(0, 28, B))
        kv4.kv4_write(k, v, a, dp)
        kv4.kv4_write(k.contiguous().clone(), v.contiguous().clone(), b, dp)
        assert all(torch.equal(x, y) for x, y in zip(a, b)) and any(bool(x.any()) for x in a)


# ------------------------------------------------------------------ attention
def _check(o, q, cache, dpos, pages=None):
    want, bound = ref.attention(np_(q.float()), cache, dpos, pages)
    got = np_(o.double())
    half = torch.finfo(o.dtype).eps / 2
    lim = bound + (half if o.dtype != torch.float32 else 0) * (np.abs(want) + bound) + (2.0 ** -25 if o.dtype == torch.float16 else 0)
    bad = np.abs(got - want) > lim
    assert not bad.any(), (int(bad.sum()), float((np.abs(got - want) / np.maximum(lim, 1e-300)).max()))


CASES = [
    # B, M, Hkv, G, D, page (0: none), positions a sequence has room for, dpos, q, o
    (1, 1, 4, 8, 128, 0, 16, [0], "bf16", "fp32"),
    (1, 1, 4, 8, 128, 0, 64, [37], "bf16", "bf16"),
    (1, 1, 1, 1, 64, 0, 16, [15], "fp16", "fp16"),
    (1, 1, 4, 8, 128, 0, 4096, [499], "bf16", "fp32"),
    (1, 1, 2, 16, 128, 0, 4096, [4095], "fp16", "fp32"),
    (1, 9, 4, 8, 128, 0, 2000, [1771], "bf16", "fp32"),
    (1, 16, 2, 5, 64, 0, 1600, [0], "bf16", "fp32"),
    (1, 5, 2, 7, 128, 0, 112, [110], "bf16", "fp32"),            # two tokens past the cache
    (1, 4, 1, 3, 128, 0, 32, [-2], "bf16", "fp32"),              # two before it
    (3, 1, 2, 4, 128, 16, 480, [0, 31, 479], "bf16", "fp32"),
    (7, 3, 5, 3, 64, 16, 336, [0, 15, 16, -3, 200, 331, 64], "fp16", "fp32"),
    (5, 2, 3, 12, 128, 64, 640, [638, 63, 64, -2, 127], "bf16", "bf16"),
    (70, 1, 1, 2, 64, 32, 256, [(i * 37) % 256 - 3 * (i % 9 == 0) for i in range(70)], "bf16", "fp32"),
    (2, 1, 8, 1, 128, 128, 1024, [1023, 2 ** 31 - 1], "bf16", "fp32"),
    (1, 33, 2, 4, 128, 32, 256, [100], "bf16", "fp32"),
    (2, 70, 1, 2, 64, 0, 160, [0, 77], "fp16", "fp32"),
    (1, 200, 2, 4, 128, 64, 1024, [600], "bf16", "fp32"),                                      # pieces of a prompt
    (3, 50, 1, 5, 64, 16, 336, [-20, 290, 100], "fp16", "bf16"),
    (8, 33, 8, 16, 64, 0, 64, [0, 31, -33, 30, 5, -1, 60, 20], "bf16", "fp16"),
    (1, 130, 1, 1, 128, 0, 144, [0], "fp16", "fp32"),
    (33, 1, 4, 2, 128, 0, 544, [(i * 61) % 545 - 1 for i in range(33)], "bf16", "fp32"),      # one workgroup a head
    (66, 2, 2, 3, 64, 16, 672, [(i * 97) % 670 - 2 * (i % 7 == 0) for i in range(66)], "fp16", "bf16"),
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_attention(case):
    B, M, Hkv, G, D, page, S, dpos, qt, ot = case
    rng = np.random.default_rng(S + M + B)
    n_pages, P = (B * (S // page) + 1, page) if page else (B, S)
    cache = _host_cache(rng, n_pages, Hkv, P, D)
    pages = _table(rng, B, S // page, n_pages) if page else None
    q = torch.from_numpy(rng.standard_normal((B, M, Hkv * G, D))).to(DT[qt]).to(DEV)
    dev, dp, tab = _dev(cache), _i32(dpos), None if pages is None else _i32(pages)
    o = kv4.attn_decode4(q, dev, dp, tab, DT[ot])
    _check(o, q, cache, dpos, pages)
    assert torch.equal(o, kv4.attn_decode4(q, dev, dp, tab, DT[ot]))           # the same bits again
    # its MXFP4 rows are those of bf16(o)
    oq, os_ = kv4.attn_decode4_mx(q, dev, dp, tab)
    o32 = np_(kv4.attn_decode4(q, dev, dp, tab))
    wq, ws = fmt.quantize_rows(fmt.bf16_round(o32).reshape(B * M, -1))
    assert np.array_equal(np_(oq), wq) and np.array_equal(np_(os_), ws)


@pytest.mark.parametrize("B,M,Hkv,G,D,S", [(700, 1, 2, 3, 64, 8192), (250, 5, 1, 8, 128, 8192), (250, 7, 1, 5, 64, 4096), (70, 2, 1, 8, 128, 2048),
                                          (3, 1, 4, 8, 128, 8192)])
def test_long_and_short_sequences_together(B, M, Hkv, G, D, S):
    """One long sequence among many of a few positions, some slots empty: several sequences in a share, and a
    sequence in several shares."""
    rng = np.random.default_rng(B)
    dpos = rng.integers(0, 60, B)
    dpos[rng.permutation(B)[:B // 8]] = -M
    dpos[B // 3] = S - M - 100
    need = (np.maximum(dpos + M, 0) + 15) // 16
    ids = iter(rng.permutation(int(need.sum()) + 3))
    pages = np.full((B, S // 16), -1, np.int32)
    for b in range(B):
        pages[b, :need[b]] = [next(ids) for _ in range(need[b])]
    cache = _host_cache(rng, int(need.sum()) + 3, Hkv, 16, D)
    q = torch.from_numpy(rng.standard_normal((B, M, Hkv * G, D))).bfloat16().to(DEV)
    dev, dp, tab = _dev(cache), _i32(dpos), _i32(pages)
    for dt in (torch.float32, torch.float16):
        o = kv4.attn_decode4(q, dev, dp, tab, dt)
        _check(o, q, cache, dpos, pages)
        assert torch.equal(o, kv4.attn_decode4(q, dev, dp, tab, dt))


def test_pages_that_are_none():
    """Holes in a table are positions that no token sees; rows with nothing else are zeros."""
    rng = np.random.default_rng(8)
    B, M, Hkv, G, D, page = 4, 2, 2, 4, 128, 16
    cache = _host_cache(rng, 30, Hkv, page, D)
    pages = _table(rng, B, 7, 30, holes=9)
    pages[2] = (-1, 30, 31, 2 ** 31 - 1, -2 ** 31, -5, -1)
    pages[3, :2] = -1
    dpos = [100, 75, 90, 20]
    q = torch.randn((B, M, Hkv * G, D), device=DEV).bfloat16()
    o = kv4.attn_decode4(q, _dev(cache), _i32(dpos), _i32(pages))
    _check(o, q, cache, dpos, pages)
    assert not o[2].any() and not o[3].any() and o[0].any()


@pytest.mark.parametrize("M,Hkv,G,D", [(1, 1, 8, 128), (5, 1, 8, 128), (1, 2, 3, 64), (7, 2, 5, 64)])
def test_holes_in_long_tables(M, Hkv, G, D):
    rng = np.random.default_rng(M + G)
    cache = _host_cache(rng, 90, Hkv, 16, D)
    pages = rng.integers(0, 90, (2, 128)).astype(np.int32)
    pages[rng.random((2, 128)) < 0.4] = -1
    pages[1, 40:70] = 90
    dpos = [2040, 1300]
    q = torch.from_numpy(rng.standard_normal((2, M, Hkv * G, D))).bfloat16().to(DEV)
    for dt in (torch.float32, torch.bfloat16):
        _check(kv4.attn_decode4(q, _dev(cache), _i32(dpos), _i32(pages), dt), q, cache, dpos, pages)


@pytest.mark.parametrize("M,Hkv,G,D", [(1, 4, 8, 64), (1, 1, 4, 128), (9, 1, 8, 128), (16, 2, 1, 64), (40, 1, 1, 128)])
def test_a_long_context(M, Hkv, G, D):
    """More shares than four waves merge at once."""
    rng = np.random.default_rng(M + D)
    S = 16384
    cache = _host_cache(rng, 1, Hkv, S, D)
    q = torch.from_numpy(rng.standard_normal((1, M, Hkv * G, D))).bfloat16().to(DEV)
    for at in (S - M, 9000, 4200, 3, -M):
        _check(kv4.attn_decode4(q, _dev(cache), _i32([at])), q, cache, [at])


def test_one_share_for_two_sequences():
    """So many kv heads and rows that a workgroup has both sequences, one after the other."""
    rng = np.random.default_rng(20)
    Hkv, M, D = 256, 33, 64
    cache = _host_cache(rng, 8, Hkv, 64, D)
    pages = np.full((2, 160), -1, np.int32)            # 10240 positions
    pages[0, :3], pages[1, :4] = (5, 1, 7), (0, 2, 3, 6)
    q = torch.from_numpy(rng.standard_normal((2, M, Hkv, D))).bfloat16().to(DEV)
    for dpos in ([150, 200], [-M, 200], [120, -M], [-10, -M]):
        _check(kv4.attn_decode4(q, _dev(cache), _i32(dpos), _i32(pages)), q, cache, dpos, pages)


def test_views_of_q():
    """Slices of a projection, at strides and addresses that loads of 16 bytes take and that they do not."""
    rng = np.random.default_rng(21)
    Hkv, D = 2, 128
    cache = _host_cache(rng, 3, Hkv, 256, D)
    dev, dp = _dev(cache), _i32([200, 17, 100])
    for M, G, dt in ((1, 4, torch.bfloat16), (3, 4, torch.float16), (7, 5, torch.bfloat16)):
        Hq = Hkv * G
        for off, extra in ((0, 2 * Hkv * D), (8, 64), (3, 5), (0, 4)):
            proj = torch.from_numpy(rng.standard_normal((3, M, Hq * D + extra + off))).to(dt).to(DEV)
            q = proj[..., off:off + Hq * D].unflatten(-1, (Hq, D))
            for o, w in zip((kv4.attn_decode4(q, dev, dp), *kv4.attn_decode4_mx(q, dev, dp)),
                            (kv4.attn_decode4(q.contiguous(), dev, dp), *kv4.attn_decode4_mx(q.contiguous(), dev, dp))):
                assert torch.equal(o, w)
        q = torch.from_numpy(rng.standard_normal((M, 3, Hq, D))).to(dt).to(DEV).transpose(0, 1)      # tokens before sequences
        assert torch.equal(kv4.attn_decode4(q, dev, dp), kv4.attn_decode4(q.contiguous(), dev, dp))
        q = torch.from_numpy(rng.standard_normal((1, 1, Hq, D))).to(dt).to(DEV).expand(3, M, Hq, D)
        assert torch.equal(kv4.attn_decode4(q, dev, dp), kv4.attn_decode4(q.contiguous(), dev, dp))


@pytest.mark.parametrize("M", [2, 9])
def test_both_outputs_of_one_call(M):
    """o and oq, os together are what each is alone (o in fp32; bf16 its rounding), and rows behind them stay."""
    lib, rng = _lib.load(), np.random.default_rng(22)
    B, Hkv, G, D, S = 2, 1, 4, 128, 1024
    cache = _dev(_host_cache(rng, B, Hkv, S, D))
    dp, q = _i32([1000, 411]), torch.from_numpy(rng.standard_normal((B, M, Hkv * G, D))).bfloat16().to(DEV)
    n = lib.mxfp4_attn_kv4_workspace_size(B, M, Hkv * G, Hkv, D, S)
    assert n > 0
    for code, dt in ((0, torch.bfloat16), (1, torch.float16), (2, torch.float32)):
        ws = torch.full((n + 64,), 99, dtype=torch.uint8, device=DEV)
        o = torch.full((B * M + 1, Hkv * G, D), 77.0, dtype=dt, device=DEV)
        oq, os_ = (torch.full((B * M + 1, Hkv * G * w), 55, dtype=torch.uint8, device=DEV) for w in (D // 2, D // 32))
        _lib.check(lib.mxfp4_attn_kv4(q.data_ptr(), 0, Hkv * G * D, *[t.data_ptr() for t in cache], None, B, S, 0, dp.data_ptr(),
                                      o.data_ptr(), code, oq.data_ptr(), os_.data_ptr(), B, M, Hkv * G, Hkv, D, ws.data_ptr(), n,
                                      torch.cuda.current_stream().cuda_stream), "attn_kv4")
        wq, wsc = kv4.attn_decode4_mx(q, cache, dp)
        assert torch.equal(oq[:-1], wq) and torch.equal(os_[:-1], wsc)
        assert torch.equal(o[:-1].view(B, M, Hkv * G, D), kv4.attn_decode4(q, cache, dp).to(dt))
        assert (o[-1] == 77).all() and (oq[-1] == 55).all() and (os_[-1] == 55).all() and (ws[n:] == 99).all()


@pytest.mark.parametrize("B,M,S", [(1, 9, 8192), (3, 6, 4096), (40, 1, 4096), (40, 1, 512)])
def test_replays_with_other_positions(B, M, S):
    """Every path captured once and replayed over other lengths, with eager work between, is the eager result."""
    rng = np.random.default_rng(23 + B)
    dev = _dev(_host_cache(rng, B, 1, S, 128))
    q, dp = torch.randn((B, M, 8, 128), device=DEV).bfloat16(), _i32([5] * B)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        kv4.attn_decode4(q, dev, dp)
        with torch.cuda.graph(graph, stream=side):
            o = kv4.attn_decode4(q, dev, dp)
    torch.cuda.current_stream().wait_stream(side)
    for hi in (S, 40, S // 2, 1):
        dp.copy_(_i32(rng.integers(-M, hi, B)))
        q.normal_()
        graph.replay()
        assert torch.equal(o, kv4.attn_decode4(q, dev, dp))
        assert torch.isfinite(o).all()


def test_shared_pages():
    """A prefix that two sequences share."""
    rng = np.random.default_rng(9)
    cache = _host_cache(rng, 9, 1, 32, 64)
    pages = np.array([[4, 2, 0, 1], [4, 2, 7, 8], [4, 4, 4, 4]], np.int32)
    q = torch.randn((3, 1, 8, 64), device=DEV).bfloat16()
    _check(kv4.attn_decode4(q, _dev(cache), _i32([127, 99, 70]), _i32(pages)), q, cache, [127, 99, 70], pages)


@pytest.mark.parametrize("page", [0, 16])
@pytest.mark.parametrize("M", [1, 6, 40])
def test_what_lies_past_the_last_token_is_without_effect(M, page):
    rng = np.random.default_rng(M)
    B, Hkv, G, D, S = 2, 2, 4, 128, 320
    n_pages, P = (B * (S // page), page) if page else (B, S)
    cache = _host_cache(rng, n_pages, Hkv, P, D)
    pages = _table(rng, B, S // page, n_pages) if page else None
    dpos = [163, 240]
    q = torch.randn((B, M, Hkv * G, D), device=DEV).bfloat16()
    tab = None if pages is None else _i32(pages)
    o = kv4.attn_decode4(q, _dev(cache), _i32(dpos), tab)
    for b in range(B):
        for pos in range(dpos[b] + M, S):
            pid, r = ref.place(cache, pages, b, pos)
            for c in cache:
                c[pid, :, r] = 255          # -6 * NaN
    assert torch.equal(o, kv4.attn_decode4(q, _dev(cache), _i32(dpos), tab))
    assert torch.isfinite(o).all()


def test_query_rows_of_infinities_and_nan():
    """They give rows of NaN and leave the others' bits alone."""
    rng = np.random.default_rng(10)
    for M, dt in ((1, "bf16"), (5, "bf16"), (5, "fp16"), (40, "bf16")):
        cache = _dev(_host_cache(rng, 1, 2, 512, 128))
        q = torch.randn((1, M, 16, 128), device=DEV).to(DT[dt])
        dp = _i32([400])
        o = kv4.attn_decode4(q, cache, dp)
        bad = q.clone()
        bad[0, 0, 0, 3], bad[0, M - 1, 9, 127], bad[0, M - 1, 15, 64] = float("inf"), float("-inf"), float("nan")
        ob = kv4.attn_decode4(bad, cache, dp)
        rows = torch.zeros((1, M, 16), dtype=torch.bool, device=DEV)
        rows[0, 0, 0] = rows[0, M - 1, 9] = rows[0, M - 1, 15] = True
        assert torch.isnan(ob[rows]).all() and torch.equal(ob[~rows], o[~rows])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [30.0, 3e3, 1e30])
def test_large_scores(size, D):
    """Scores far apart, one row's maximum late and early: the softmax is the one-hot or the few that are near."""
    rng = np.random.default_rng(11)
    S = 700
    cache = _host_cache(rng, 1, 1, S + 4, D)
    q = torch.from_numpy(rng.standard_normal((1, 3, 4, D)) * size).to(torch.bfloat16).to(DEV)
    o = kv4.attn_decode4(q, _dev(cache), _i32([S - 3]))
    want, bound = ref.attention(np_(q.float()), cache, [S - 3])
    got = np_(o).astype(np.float64)
    big = bound > 0.1 * np.abs(want).max()          # the exponents' rounding is more than a term: nothing to compare
    assert np.isfinite(got).all()
    off = np.where(big, 0.0, np.abs(got - want) / bound)
    assert off.max() <= 1, (off.max(), want.reshape(-1)[off.argmax()], got.reshape(-1)[off.argmax()])
    k, v, _ = ref.read(cache, S, [0])
    s = np.einsum("mhd,nd->mhn", np_(q.float()).astype(np.float64)[0], k[0, :, 0].astype(np.float64))
    top = np.sort(s, -1)
    sure = (top[..., -1] - top[..., -2]) / np.sqrt(D) > 40 + 1e-4 * np.abs(s).max() / np.sqrt(D)     # one-hot
    for m in range(3):
        for h in range(4):
            n = S - 2 + m
            i = int(np.argmax(s[m, h, :n]))
            if sure[m, h] and top[m, h, -1] == s[m, h, i]:
                assert np.allclose(got[0, m, h], v[0, i, 0], rtol=1e-6)


def test_small_terms_beside_one_large_score():
    """Many positions far below one whose value is tiny: their sum keeps its bits."""
    D, S = 64, 16384
    kq, ks = np.zeros((1, 1, S, 32), np.uint8), np.full((1, 1, S, 2), 127, np.uint8)
    vq, vs = np.full((1, 1, S, 32), 0x77, np.uint8), np.full((1, 1, S, 2), 133, np.uint8)     # 6 * 64
    kq[0, 0, 5, 0] = 0x07                        # one key 6 in dimension 0
    vq[0, 0, 5], vs[0, 0, 5] = 0x11, 118          # its value 2^-10
    cache = [kq, ks, vq, vs]
    q = torch.zeros((1, 1, 1, D), device=DEV)
    q[..., 0] = 17.5 * 8 / 6
    q = q.bfloat16()
    o = kv4.attn_decode4(q, _dev(cache), _i32([S - 1]))
    _check(o, q, cache, [S - 1])


def test_a_cache_past_two_and_four_gigabytes():
    """Offsets of a long cache: rows at the end of its last sequence."""
    B, Hkv, D, S = 9, 8, 128, 1 << 20                  # 4.5 GiB of keys
    cache = kv4.empty_cache(B, S, Hkv, D)
    n = 700
    k, v = (torch.randn((B, n, Hkv, D), device=DEV).bfloat16() for _ in range(2))
    at = S - n
    dp = _i32([-n] * (B - 1) + [at])
    kv4.kv4_write(k, v, cache, dp)
    rk, rv = kv4.kv4_read(cache, n, dp)
    want = torch.from_numpy(fmt.dequant_rows(*fmt.quantize_rows(np_(k[-1].float()).reshape(-1, D)))).view(n, Hkv, D)
    assert torch.equal(rk[-1].float().cpu(), want) and not rk[:-1].any()
    assert not cache.kq[:-1].any() and not cache.kq[-1, :, :at].any()
    q = torch.randn((B, 1, 16, D), device=DEV).bfloat16() * 8
    o = kv4.attn_decode4(q, cache, _i32([-1] * (B - 1) + [S - 1]))
    # the rows before `at` are zeros: scores 0, values 0
    s = torch.einsum("hgd,nhd->hgn", q[-1, 0].view(Hkv, 2, D).double(), rk[-1].double()) / D ** 0.5
    w = torch.exp(s)
    want = torch.einsum("hgn,nhd->hgd", w, rv[-1].double()) / (w.sum(-1, keepdim=True) + at)
    assert not o[:-1].any()
    assert (o[-1, 0].view(Hkv, 2, D).double() - want).abs().max() <= 1e-4 * want.abs().max()


def test_together_over_steps_in_a_graph_and_out_of_it():
    """A prompt's write, then steps of write + attention: captured and replayed with the positions moved on the
    device, beside eager steps on another cache; the bits are the same, and right."""
    rng = np.random.default_rng(12)
    B, Hkv, G, D, page, S = 3, 2, 4, 128, 32, 512
    Hq = Hkv * G
    pages = _table(rng, B, S // page, B * (S // page))
    tab, first = _i32(pages), [0, 100, 331]
    caches = [kv4.empty_cache(B * (S // page), page, Hkv, D) for _ in range(2)]
    k, v = (torch.randn((B, 40, Hkv, D), device=DEV).bfloat16() for _ in range(2))
    for c in caches:
        kv4.kv4_write(k, v, c, _i32(first), tab)
    start = [f + 40 for f in first]
    kn, vn = (torch.randn((6, B, 1, Hkv, D), device=DEV).bfloat16() for _ in range(2))
    qn = torch.randn((6, B, 1, Hq, D), device=DEV).bfloat16()
    k1, v1, q1, dp = kn[0].clone(), vn[0].clone(), qn[0].clone(), _i32(start)

    def step():
        kv4.kv4_write(k1, v1, caches[0], dp, tab)
        o = kv4.attn_decode4(q1, caches[0], dp, tab)
        dp.add_(1)
        return o

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()                                  # step 0, then the capture
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.current_stream().wait_stream(side)
    host = [np_(c) for c in caches[1]]
    for i in range(6):
        if i:
            k1.copy_(kn[i])
            v1.copy_(vn[i])
            q1.copy_(qn[i])
            graph.replay()
        at = [s + i for s in start]
        kv4.kv4_write(kn[i], vn[i], caches[1], _i32(at), tab)
        eager = kv4.attn_decode4(qn[i], caches[1], _i32(at), tab)
        ref.write(np_(kn[i].float()), np_(vn[i].float()), host, at, pages)
        if i:
            assert torch.equal(out, eager)
        _check(eager, qn[i], host, at, pages)
    for a, b, h in zip(*caches, host):
        assert torch.equal(a, b) and np.array_equal(np_(a), h)


def test_on_another_stream_and_two_at_once():
    """Calls queued on side streams, two at a time, have workspaces of their own."""
    rng = np.random.default_rng(13)
    cache = _dev(_host_cache(rng, 2, 4, 4096, 128))
    dp = _i32([4000, 2500])
    qs = [torch.randn((2, 3, 32, 128), device=DEV).bfloat16() for _ in range(2)]
    want = [kv4.attn_decode4(q, cache, dp) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(kv4.attn_decode4(qs[i], cache, dp))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_shapes_without_work():
    cache = kv4.empty_cache(2, 32, 2, 64)
    dp = _i32([3, 4])
    e = torch.empty((2, 0, 2, 64), dtype=torch.bfloat16, device=DEV)
    kv4.kv4_write(e, e, cache, dp)
    assert kv4.kv4_read(cache, 0)[0].shape == (2, 0, 2, 64)
    assert kv4.attn_decode4(e, cache, dp).shape == (2, 0, 2, 64)
    assert kv4.attn_decode4_mx(e, cache, dp)[0].shape == (0, 64)


def test_refusals_of_tensors():
    cache = kv4.empty_cache(2, 32, 2, 64)
    dp = _i32([3, 4])
    x = torch.zeros((2, 1, 2, 64), dtype=torch.bfloat16, device=DEV)
    tab = _i32([[0], [1]])
    for bad in (dict(k=x[:1]), dict(k=x.double(), v=x.double()), dict(v=x.float()), dict(k=x[..., :32], v=x[..., :32]), dict(k=x.cpu()),
                dict(dp=dp[:1]), dict(dp=dp.long()), dict(dp=dp.cpu()), dict(cache=cache._replace(ks=cache.kq)),
                dict(cache=cache._replace(kq=cache.kq.float())), dict(cache=cache._replace(vs=cache.vs.cpu())),
                dict(cache=cache._replace(kq=cache.kq.transpose(1, 2))), dict(pages=tab.long()), dict(pages=tab[:1]),
                dict(pages=tab[0])):
        a = dict(k=x, v=x, cache=cache, dp=dp, pages=None)
        a.update(bad)
        with pytest.raises(RuntimeError):
            kv4.kv4_write(a["k"], a["v"], a["cache"], a["dp"], a["pages"])
    q = torch.zeros((2, 1, 4, 64), dtype=torch.bfloat16, device=DEV)
    for bad in (q.float(), q[:, :, :3], q[:1], q[..., :32], q[0], q.cpu()):
        with pytest.raises(RuntimeError):
            kv4.attn_decode4(bad, cache, dp)
    with pytest.raises(RuntimeError):
        kv4.attn_decode4(q, cache, dp, dtype=torch.float64)
    with pytest.raises(RuntimeError):
        kv4.kv4_read(cache, -1)
    with pytest.raises(RuntimeError):
        kv4.kv4_read(cache, 4, dtype=torch.uint8)
    with pytest.raises(RuntimeError):
        kv4.kv4_read(cache, 4, start=dp[:1])


def test_a_table_of_no_columns():
    """Refused, with the pool as it was: its pages are someone's."""
    cache, before = (_dev(_host_cache(np.random.default_rng(30), 3, 2, 32, 64)) for _ in range(2))
    x, q = torch.ones((2, 1, 2, 64), device=DEV), torch.ones((2, 1, 4, 64), device=DEV).bfloat16()
    tab = _i32([[0, 1], [2, 0]])[:, :0]
    for t in (tab, tab.contiguous(), torch.empty((2, 0), dtype=torch.int32, device=DEV)):
        for call in (lambda: kv4.kv4_write(x, x, cache, _i32([0, 0]), t), lambda: kv4.kv4_read(cache, 1, pages=t),
                     lambda: kv4.attn_decode4(q, cache, _i32([0, 0]), t), lambda: kv4.attn_decode4_mx(q, cache, _i32([0, 0]), t)):
            with pytest.raises(RuntimeError):
                call()
    assert all(torch.equal(a, b) for a, b in zip(cache, before))


def test_a_cache_of_no_heads():
    cache = kv4.KV4(*(torch.empty((2, 0, 32, w), dtype=torch.uint8, device=DEV) for w in (32, 2, 32, 2)))
    x, q, dp = torch.empty((2, 1, 0, 64), device=DEV), torch.ones((2, 1, 4, 64), device=DEV).bfloat16(), _i32([0, 0])
    for call in (lambda: kv4.kv4_write(x, x, cache, dp), lambda: kv4.kv4_read(cache, 1), lambda: kv4.attn_decode4(q, cache, dp),
                 lambda: kv4.attn_decode4_mx(q, cache, dp)):
        with pytest.raises(RuntimeError, match="a kv head at least"):
            call()


def test_an_empty_batch():
    cache, dp = kv4.empty_cache(3, 32, 2, 64), torch.empty(0, dtype=torch.int32, device=DEV)
    x, q = torch.empty((0, 2, 2, 64), device=DEV), torch.empty((0, 2, 4, 64), device=DEV).bfloat16()
    for cols in (0, 3):
        t = torch.empty((0, cols), dtype=torch.int32, device=DEV)
        kv4.kv4_write(x, x, cache, dp, t)
        assert kv4.kv4_read(cache, 5, dp, t)[0].shape == (0, 5, 2, 64)
        assert kv4.attn_decode4(q, cache, dp, t).shape == (0, 2, 4, 64) and kv4.attn_decode4_mx(q, cache, dp, t)[1].shape == (0, 8)
    assert not any(c.any() for c in cache)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("M,G", [(1, 2), (2, 16)])
def test_the_smallest_keys_and_values(M, G, D):
    """Scale code 0: keys and values below bf16's normal numbers, which the products must not take for zeros."""
    cache = kv4.empty_cache(1, 64, 1, D)
    cache.kq[0, 0, 0, 0], cache.vq[0, 0, 0] = 0x01, 0x11            # 2^-128 in dimension 0, and everywhere
    cache.vq[0, 0, 1] = 0x32                                        # 2^-127 and 1.5 * 2^-127
    q = torch.zeros((1, M, G, D), device=DEV).bfloat16()
    q[..., 0] = 2.0 ** 127                                          # a score of 1/2 at position 0, 0 at the others
    q[0, 0, 0, 0] = 2.0 ** 120                                      # 2^-8
    o = kv4.attn_decode4(q, cache, _i32([1]))
    host = [np_(c) for c in cache]
    want, bound = ref.attention(np_(q.float()), host, [1])
    assert (want != 0).all() and (np.abs(np_(o).astype(np.float64) - want) <= bound + 2.0 ** -148).all()
