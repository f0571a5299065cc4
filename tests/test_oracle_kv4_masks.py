"""The oracle's masks (oracle/kv4_masks.py) by cases that can be written down."""
import numpy as np

from oracle import kv4_masks


def _rows(a):
    return ["".join("x" if v else "." for v in r) for r in a]


def test_windows():
    assert _rows(kv4_masks.sees([3], 3, 8)[0]) == ["xxxx....", "xxxxx...", "xxxxxx.."]
    assert _rows(kv4_masks.sees([3], 3, 8, window=2)[0]) == ["..xx....", "...xx...", "....xx.."]
    assert _rows(kv4_masks.sees([3], 3, 8, window=2, sinks=1)[0]) == ["x.xx....", "x..xx...", "x...xx.."]
    assert _rows(kv4_masks.sees([-1, 7], 2, 8, window=3, sinks=1).reshape(4, 8)) == ["........", "x.......", "x....xxx", "........"]
    assert _rows(kv4_masks.sees([0], 1, 4, window=1, sinks=9)[0]) == ["x..."]


def test_trees():
    words, depth = kv4_masks.tree_masks(np.array([[-1, 0, 0, 1, 3, -2, 5, -1]]))
    assert [int(w) for w in words[0, :, 0]] == [1, 3, 5, 11, 27, 0, 0, 128] and list(depth[0]) == [0, 1, 1, 2, 3, -1, -1, 0]
    see = kv4_masks.sees([2], 8, 10, tree=words)[0]
    assert _rows(see) == ["xxx.......", "xxxx......", "xxx.x.....", "xxxx.x....", "xxxx.xx...", "xx........", "xx........", "xx.......x"]
    # draft 4 stands at 2 + 3, its window of 4 begins at 2; a draft that sees none of them at 1
    see = kv4_masks.sees([2], 8, 10, window=4, tree=words)[0]
    assert _rows(see) == ["xxx.......", "xxxx......", "xxx.x.....", ".xxx.x....", "..xx.xx...", "xx........", "xx........", "xx.......x"]
    words, depth = kv4_masks.tree_masks(np.arange(-1, 69)[None])
    assert words.shape == (1, 70, 3) and list(words[0, 69]) == [-1, -1, 63] and depth[0, 69] == 69
    assert np.array_equal(kv4_masks.sees([5], 70, 80, tree=words), kv4_masks.sees([5], 70, 80))
    for bad in (-2, 1, 2, 7, 2 ** 31 - 1, -2 ** 31):
        words, depth = kv4_masks.tree_masks(np.array([[-1, bad, 1]]))
        assert list(words[0, :, 0]) == [1, 0, 0] and list(depth[0]) == [0, -1, -1]
