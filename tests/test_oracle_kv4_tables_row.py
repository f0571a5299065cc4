"""The oracle's page table (oracle/kv4_tables.py) for lengths past a sequence's row, by cases that can be written down."""
import pytest

from oracle.kv4_tables import Tables


# four pages of 16: 70 positions need a fifth, 100 seven in all
@pytest.mark.parametrize("window,sinks,lens,new,lacked", [
    (None, 0, 64, 64, 0), (None, 0, 65, 65, 1), (None, 0, 70, 6, 1), (None, 0, 100, 100, 3), (None, 0, 2 ** 31 - 1, 5, 2 ** 27 - 4),
    (20, 0, 70, 70, 1), (20, 0, 200, 1, 2),              # the window of position 199 begins at 180, in page 11 of 0 .. 12
    (20, 100, 200, 1, 5),                                # and pages 4, 5 and 6 of the sinks
    (20, 1000, 200, 1, 9)])                              # sinks past the row's end: pages 4 .. 12
def test_pages_past_the_row_are_counted(window, sinks, lens, new, lacked):
    t = Tables(1, 4, 9, 16, window, sinks)
    t.update([lens], [new], 0)
    assert t.lacked == lacked
    t.update([0])
    assert t.lacked == 0 and len(t.free) == 9
