"""GPU tests of page tables whose sequences outgrow their rows (kv4.kv4_tables) against oracle/kv4_tables.py."""
import numpy as np
import pytest

from moe_fused_inference_amd import kv4
from oracle.kv4_tables import Tables
from tests.gpu_helpers import np_
from tests.kv4_mask_helpers import i32

pytestmark = pytest.mark.gpu


# (one workgroup, and past its 32768 entries)
@pytest.mark.parametrize("B,max_pages", [(1, 4), (9, 4), (300, 120)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 0), (20, 100), (50, 2000), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_pages_past_the_row_are_counted(B, max_pages, window, sinks):
    rng = np.random.default_rng([B, sinks])
    t, want = kv4.page_tables(B, max_pages, B * max_pages, 16, window, sinks), Tables(B, max_pages, B * max_pages, 16, window, sinks)
    room, some = max_pages * 16, False
    for top in (room, room + 1, room + 40, 3 * room, 2 ** 31 - 1, room // 2, room + 70):
        lens = np.where(rng.random(B) < 0.5, top, rng.integers(0, top + 1, B))
        new = np.minimum(lens, rng.integers(0, 90, B))
        T = int(new.sum()) + 3
        got, said = kv4.kv4_tables(t, i32(lens), i32(new), T), want.update(lens, new, T)
        n = len(want.free)
        assert t.state.tolist() == [n, min(want.lacked, 2 ** 30)] and t.free[:n].tolist() == want.free
        assert np.array_equal(np_(t.pages), want.pages) and np.array_equal(np_(t.span), want.span)
        assert all(np.array_equal(np_(x), y) for x, y in zip(got, said))
        some |= (lens > room).any()
        assert want.lacked > 0 or not (lens > room).any()
    assert some
