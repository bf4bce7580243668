"""How far an element of the 8-bit cache is off, by the oracle (64 bits): at most 2^-4 of its value plus 2^-9
of the largest scale S that its block has had since it was written. The first rounding is off by 2^-4 |x| or
2^-10 S_0. A later one happens only where a scale rises above all before it (the value is a multiple of
2^-9 of the largest so far, or has 4 significant bits, both exact at any scale up to that), is off by at
most 2^-10 S_i, and such scales at least double: 2^-10 (S_0 + S_1 + ... + S) <= 2^-9 S."""
import numpy as np
import pytest

from oracle import kv8 as okv


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("block", [16, 64])
def test_bound_over_random_writes(seed, block):
    """Rows of very different size, chunks and single tokens, taken back now and then."""
    g = np.random.default_rng(seed)
    r = okv.Ring(1, 70, 8, 6, block)
    true, big = {}, {}          # by slot: the value written, the largest scale since
    at = -6
    for _ in range(120):
        T = int(g.choice([1, 1, 1, 5, 20]))
        x = g.standard_normal((T, 1, 8)) * 2.0 ** g.uniform(-14, 14, (T, 1, 1))
        r.write(x, at)
        for t in range(T):
            true[r.slot(at + t)], big[r.slot(at + t)] = x[t, 0], 0.0
        at += T
        w = r.window()
        for s in w:
            big[s] = max(big[s], r.scale[0, s // block])
            err = np.abs(r.val[0, s] * r.scale[0, s // block] - true[s])
            assert (err <= 2.0 ** -4 * np.abs(true[s]) + 2.0 ** -9 * big[s]).all()
        if at < 60 and g.random() < 0.3:  # before the ring comes round
            at = max(0, at - int(g.integers(1, 8)))


def test_a_loud_padding_costs_the_rows_that_stay():
    """Padding of 3e6 in the block of rows of 1.0: its scale is 2^13, under whose half smallest code 1.0 falls; the
    scale comes down again when the padding is taken back and overwritten, the rows do not come back."""
    r = okv.Ring(1, 22, 8, 0, 16)
    r.write(np.ones((8, 1, 8)), 0)
    r.write(np.full((8, 1, 8), 3e6), 8)
    assert r.scale[0, 0] == 2.0 ** 13
    for p in range(8, 16):
        r.write(np.ones((1, 1, 8)), p)
    assert r.scale[0, 0] == 2.0 ** -8
    rows = r.rows()[0]
    assert (rows[:8] == 0).all() and (rows[8:] == 1).all()
    quiet = okv.Ring(1, 22, 8, 0, 16)  # zeros as padding
    quiet.write(np.ones((8, 1, 8)), 0)
    quiet.write(np.zeros((8, 1, 8)), 8)
    assert (quiet.rows()[0, :8] == 1).all() and quiet.scale[0, 0] == 2.0 ** -8
