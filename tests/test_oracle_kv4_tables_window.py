"""The oracle's page table (oracle/kv4_tables.py) where a window has had pages given back, by cases that can be written down."""
import numpy as np

from oracle.kv4_tables import Tables


def test_a_sequence_that_begins_in_the_place_of_another():
    """No call with length 0 between them: the new one has all its pages, the old one's go back."""
    for sinks, held in ((0, [31, 32, 33, 34, 35, 36, 37]), (17, [0, 1, 31, 32, 33, 34, 35, 36, 37])):
        t = Tables(1, 40, 40, 16, window=100, sinks=sinks)
        t.update([600], [600], 600)
        t.update([600])
        assert t.span.tolist() == [[31, 38]] and [i for i in range(40) if t.pages[0, i] >= 0] == held
        slots, _, pos, _ = t.update([40], [40], 40)
        assert t.span.tolist() == [[0, 3]] and (t.pages[0, :3] >= 0).all() and (t.pages[0, 3:] < 0).all() and t.lacked == 0
        assert (slots >= 0).all() and pos.tolist() == list(range(40)) and len(t.free) == 37
        t.update([0])
        assert sorted(t.free) == list(range(40)) and t.span.tolist() == [[0, 0]]


def test_a_sequence_that_steps_back_behind_its_window():
    """Pages that are gone stay gone, and are counted while a token needs them: a new one, or one whose window reaches them."""
    t = Tables(1, 40, 40, 16, window=100)
    t.update([600], [600], 600)
    t.update([600])
    slots = t.update([520], [3], 3)[0]                      # 517 .. 519, and the first's window from 418 on: pages 26 .. 30 are gone
    assert t.span.tolist() == [[31, 33]] and t.lacked == 5 and (slots >= 0).all()
    slots = t.update([497], [3], 3)[0]                      # 494, 495 and 496, whose page alone is there; pages 24 .. 30
    assert t.lacked == 7 and (slots >= 0).tolist() == [False, False, True] and t.span.tolist() == [[31, 32]]
    t.update([400])                                         # pages 18 .. 24
    assert t.lacked == 7 and t.span.tolist() == [[25, 25]] and len(t.free) == 40
    t.update([520], [20], 0)                                # the first new one's window begins at 401, on the first page that is not gone
    assert t.lacked == 0 and t.span.tolist() == [[25, 33]]


def test_drafts_that_are_rejected_are_not_counted():
    t = Tables(1, 40, 40, 16, window=100, sinks=5)
    t.update([600], [600], 600)
    for n in range(600, 620):
        t.update([n + 18], [18], 18)
        assert t.lacked == 0
        t.update([n + 1])
        assert t.lacked == 0


def test_no_page_is_lost_or_given_twice():
    """Lengths that go anywhere, in pools that do not hold them all; where nothing lacks, every position that is needed has a page."""
    rng = np.random.default_rng(0)
    for window, sinks in ((40, 0), (40, 20), (1, 1), (100, 64)):
        B, max_pages, n_pages = 6, 9, 30
        t = Tables(B, max_pages, n_pages, 16, window, sinks)
        for _ in range(300):
            lens = rng.integers(0, max_pages * 16 + 1, B)
            new = np.where(rng.random(B) < 0.5, lens, np.minimum(lens, rng.integers(0, 30, B)))
            slots, _, _, starts = t.update(lens, new, 500)
            used = t.pages[t.pages >= 0].tolist()
            assert sorted(used + t.free) == list(range(n_pages))
            lacks = 0
            for b in range(B):
                there = t.pages[b] >= 0
                assert [i for i in range(max_pages) if there[i]] == t.has(*t.span[b])
                first = max(0, lens[b] - new[b] - window + 1) // 16
                needs = [i for i in range(-(-lens[b] // 16)) if i >= first or i < t.sink_pages]
                lacks += sum(not there[i] for i in needs)
                if all(there[i] for i in needs):
                    assert (slots[starts[b]:starts[b + 1]] >= 0).all()
            assert lacks == t.lacked
