"""The oracle's page table (oracle/kv4_tables.py) by a case that can be written down, and by what must always hold."""
import numpy as np

from oracle.kv4_tables import Tables


def test_by_hand():
    t = Tables(2, 4, 5, 16)
    slots, seq, pos, starts = t.update([17, 3], [17, 3], 22)
    assert t.pages.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1]] and t.free == [4, 3] and t.span.tolist() == [[0, 2], [0, 1]]
    assert slots.tolist() == list(range(17)) + [32, 33, 34, -1, -1] and starts.tolist() == [0, 17, 20]
    assert pos.tolist() == list(range(17)) + [0, 1, 2, -1, -1] and seq.tolist() == [0] * 17 + [1] * 3 + [-1] * 2
    t.update([0, 40])                                   # two come back (0 last, on top) and two are taken
    assert t.pages.tolist() == [[-1] * 4, [2, 0, 1, -1]] and t.free == [4, 3]
    t.update([64, 40])
    assert t.pages.tolist() == [[3, 4, -1, -1], [2, 0, 1, -1]] and t.lacked == 2 and t.span.tolist() == [[0, 2], [0, 3]]
    t.update([64, 0])
    assert t.pages.tolist() == [[3, 4, 2, 0], [-1] * 4] and t.lacked == 0 and t.free == [1]


def test_a_window():
    t = Tables(1, 8, 8, 16, window=20, sinks=17)
    t.update([100], [100], 100)
    assert t.span.tolist() == [[0, 7]] and (t.pages[0, :7] >= 0).all()
    t.update([100])                                     # the next token's window begins at 81
    assert t.span.tolist() == [[5, 7]] and [i for i in range(8) if t.pages[0, i] >= 0] == [0, 1, 5, 6]
    t.update([110], [10], 10)                           # the first new one's at 81
    t.update([102])
    assert [i for i in range(8) if t.pages[0, i] >= 0] == [0, 1, 5, 6]
    t.update([0])
    assert len(t.free) == 8 and t.span.tolist() == [[0, 0]]


def test_no_page_is_lost_or_given_twice():
    rng = np.random.default_rng(0)
    for window, sinks in ((None, 0), (40, 0), (40, 20), (1, 1), (500, 64)):
        B, max_pages, n_pages = 6, 9, 30
        t = Tables(B, max_pages, n_pages, 16, window, sinks)
        lens = np.zeros(B, np.int64)
        for _ in range(200):
            new = rng.integers(0, 30, B)
            lens = np.where(rng.random(B) < 0.1, 0, lens + new)
            t.update(lens, np.where(lens == 0, 0, new), 40)
            used = t.pages[t.pages >= 0].tolist()
            assert sorted(used + t.free) == list(range(n_pages))
            for b in range(B):
                assert [i for i in range(max_pages) if t.pages[b, i] >= 0] == t.has(*t.span[b])
