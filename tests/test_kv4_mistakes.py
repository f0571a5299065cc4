"""What the GPU tests of moving references are good for, on the CPU: the running softmax of one row, right and with the
mistakes that they are there to find."""
import numpy as np
import pytest

from oracle import kv4 as ref
from tests.test_gpu_kv4_units import SHAPES, STEPS

MOST, NONE = 2048.0, -3e38


def _row(score, v, lanes, mistake):
    """A wave's units, score (units, 32) in log 2 and v (units, 32, columns), lanes a row of 32 / lanes terms each."""
    m, l, acc = NONE, 0.0, 0.0
    with np.errstate(over="ignore"):
        for s, x in zip(score, v):
            t = np.exp2(s - m)
            if (t.reshape(lanes, -1).sum(1) > MOST).any():
                mn = max(m, s.max())
                al = np.exp2(m - mn)
                l *= al if mistake != "l kept" else 1.0
                acc *= {"acc kept": 1.0, "twice": al * al}.get(mistake, al)
                if mistake == "both twice":
                    l, acc = l * al, acc * al
                m = mn
                if mistake != "old terms" or l == 0.0:
                    t = np.exp2(s - m)
            l += t.sum()
            acc += t @ x
    return m, l, acc


def _off(shape, step, units, lanes, mistake):
    """|o - the softmax| over the bound, for four waves of `units` units, the GPU tests' levels, eighths and signs."""
    rng = np.random.default_rng(units)
    level = np.array(SHAPES[shape])[np.arange(units) * 4 // units]
    s = step * (level[None, :, None] + rng.choice([0, .5, 1, 1.5, 2, 3, 4, 6], (4, units, 32)) / 8)
    v = rng.choice([0, .5, 1, 1.5, 2, 3, 4, 6], (*s.shape, 64)) * (1 - 2 * (level % 2))[None, :, None, None]
    waves = [_row(s[w], v[w], lanes, mistake) for w in range(4)]
    top = max(m for m, _, _ in waves)
    den, num = (sum(np.exp2(w[0] - top) * w[i] for w in waves) for i in (1, 2))
    p = np.exp2(s - s.max())
    want, size = (np.tensordot(p, x, 3) / p.sum() for x in (v, np.abs(v)))
    return (np.abs(num / den - want) / (ref.rounding(64, s.size, 0.0, np.log(2) * s.max()) * size)).max()


@pytest.mark.parametrize("units,lanes", [(4, 4), (16, 4), (4, 2), (16, 2)])
def test_mistakes_exceed_the_bound(units, lanes):
    every = [(shape, step) for shape in SHAPES for step in STEPS]
    assert max(_off(*c, units, lanes, None) for c in every) < 1e-6
    for mistake in ("l kept", "acc kept", "twice", "both twice", "old terms"):
        assert max(_off(*c, units, lanes, mistake) for c in every) > 2, mistake
