"""The MXFP4 cache oracle against itself and against plain numpy, on the CPU."""
import numpy as np
import pytest

from oracle import kv4
from oracle import mxfp4 as fmt


def _cache(rng, n_pages, Hkv, page, D):
    def half():
        return [rng.integers(0, 256, (n_pages, Hkv, page, D // 2), dtype=np.uint8),
                rng.integers(120, 130, (n_pages, Hkv, page, D // 32), dtype=np.uint8)]

    return half() + half()


@pytest.mark.parametrize("paged", [False, True])
def test_write_then_read_gives_the_rounded_rows(paged):
    rng = np.random.default_rng(3)
    D, Hkv, M = 64, 2, 5
    pages = np.array([[3, 0], [1, -1]], np.int32) if paged else None
    cache = _cache(rng, 4 if paged else 2, Hkv, 16 if paged else 32, D)
    before = [c.copy() for c in cache]
    dpos = [14, 13]                       # both cross row 16: the second runs off its pages
    k, v = (rng.standard_normal((2, M, Hkv, D)).astype(np.float32) for _ in range(2))
    kv4.write(k, v, cache, dpos, pages)
    rk, rv, there = kv4.read(cache, M, dpos, pages)
    assert there.tolist() == [[True] * 5, [True] * 3 + [not paged] * 2]
    want = fmt.dequant_rows(*fmt.quantize_rows(k.reshape(-1, D))).reshape(k.shape)
    assert np.array_equal(rk[there], want[there])
    want = fmt.dequant_rows(*fmt.quantize_rows(v.reshape(-1, D))).reshape(v.shape)
    assert np.array_equal(rv[there], want[there])
    changed = sum(int((a != b).any(-1).sum()) for a, b in zip(cache[:1], before[:1]))
    assert changed <= there.sum() * Hkv


def test_attention_is_the_softmax_of_the_visible_rows():
    rng = np.random.default_rng(4)
    cache = _cache(rng, 3, 1, 16, 64)
    pages = np.array([[2, -1, 0]], np.int32)          # positions 16..31 are on no page
    q = rng.standard_normal((1, 2, 3, 64))
    o, bound = kv4.attention(q, cache, [36], pages)
    k = fmt.dequant_rows(cache[0][[2, 0], 0].reshape(-1, 32), cache[1][[2, 0], 0].reshape(-1, 2)).astype(np.float64)
    v = fmt.dequant_rows(cache[2][[2, 0], 0].reshape(-1, 32), cache[3][[2, 0], 0].reshape(-1, 2)).astype(np.float64)
    for m, n in ((0, 16 + 5), (1, 16 + 6)):
        w = np.exp(q[0, m] @ k[:n].T / 8.0)
        assert np.allclose(o[0, m], w @ v[:n] / w.sum(-1, keepdims=True), rtol=1e-12, atol=1e-12)
    assert (bound[0] > 0).all() and bound.max() < 1e-2 * np.abs(o).max()
    assert not kv4.attention(q, cache, [-2], pages)[0].any()      # an empty slot
    assert not kv4.attention(q, cache, [20], np.array([[-1, 7, -9]], np.int32))[0].any()   # no page at all


def test_two_parts_of_a_probability_would_show():
    """What the bound of the probabilities' bits is good for: p in two bf16 parts passes it, in three it does not."""
    import torch

    from tests.kv4_helpers import P_BITS, p_rows
    for D in (64, 128):
        p = torch.exp2(-p_rows(256, D).double() * np.log2(np.e) / np.sqrt(D)).float()
        rest, off = p.clone(), []
        for _ in range(3):
            rest = rest - rest.bfloat16().float()
            off.append(float((rest.abs() / p).max()))
        assert off[1] > P_BITS and off[2] == 0


def test_the_proven_bound_is_above_the_tolerance():
    """rounding() counts more than attention()'s tolerance does, at any size."""
    u = 2.0 ** -24
    for D, n, big, size in ((64, 1, 1.0, 1.0), (128, 4096, 30.0, 8.0), (128, 32768, 100.0, 90.0)):
        e = np.log(2) * (1.4427 * (D + 2) * u * big + 2 * u * 1.4427 * size) + 4 * u
        assert kv4.rounding(D, n, big, size) > 2 * e + 2 * (n / 128 + 40) * u
    assert kv4.rounding(128, 4096, 0.0, 8.0) < 3e-4
