"""Attention over 4-bit pages: which of its two forms a tile of 64 keys takes is a matter of that
tile's own values and of what the same rows have met before, and of nothing else."""
import numpy as np
import pytest

from q4ref import KB, Call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("model", ["qwen25_1p5b", "qwen25_7b", "qwen25_14b"])
@pytest.mark.parametrize("rows,past", [(70, 100), (70, 20), (12, 2000)])
def test_values_past_fp16_stay_with_their_session(model, rows, past):
    """Every other session's values are 2^20 times as large, past fp16: the sessions between them, which
    share workgroups with them, have the bits that they have beside values of their own size."""
    n = 60
    c = Call(model, [past + 3 * (i % 5) for i in range(n)], [rows] * n, seed=21, behind=0, scale=0.5)
    still = c.run().reshape(n, -1)
    p = c.parts()
    for i in range(1, n, 2):
        p[3][c.table[i, :-(-int(c.keys[i]) // KB)]] += 20
    c.set_parts(p)
    loud = c.run().reshape(n, -1)
    changed = [i for i in range(0, n, 2) if not np.array_equal(still[i], loud[i])]
    assert not changed, f"sessions {changed}"
    assert not any(np.array_equal(still[i], loud[i]) for i in range(1, n, 2))


@pytest.mark.parametrize("byte", [104, 107, 110, 113, 114, 120, 140, 141])
@pytest.mark.parametrize("rows,keys", [(0, 40), (0, 900), (4, 300), (70, 900)])
def test_a_mean_of_equal_values_is_the_value(rows, keys, byte):
    """Every value is half of one power of two, those that fp16 holds as subnormal numbers among them.  Numerator and
    denominator are sums of the same weights.  In the numerator a weight is held to 2^-22 of itself or to 2^-26 of
    the largest of its 64, at most 2^-20 of their sum; each sum runs through chains of at most 3 n / 32 + 64
    additions of 2^-24; the quotient and its product take 2^-23."""
    c = Call("qwen25_7b", [keys - rows] * 3, [rows] * 3 if rows else None, seed=22, behind=0, poison=False)
    p = c.parts()
    p[2][:], p[3][:] = 1, byte
    c.set_parts(p)
    off = c.run() / 2.0 ** (byte - 128) - 1
    bound = 2.0 ** -22 + 2.0 ** -20 + 2 * (3 * keys / 32 + 64) * 2.0 ** -24 + 2.0 ** -23
    assert np.abs(off).max() <= bound, np.abs(off).max() / bound


@pytest.mark.parametrize("power", [-10, -4, 9])
@pytest.mark.parametrize("rows,keys", [(0, 1), (0, 40), (0, 200), (4, 40), (4, 133), (12, 40), (12, 61)])
def test_a_tile_that_keys_fill_in_part_takes_its_form_from_them(rows, keys, power):
    """Values 2^power times as large, as exact in fp16 as they were: the result is 2^power times what it was, bit
    by bit, as no product, sum or weight of either is rounded differently.  What fills the slots behind
    the last key has no say in it."""
    past = [keys - rows] * 3
    c = Call("qwen25_7b", past, [rows] * 3 if rows else None, seed=22, behind=0, scale=0.5)
    one = c.run()
    p = c.parts()
    held = np.unique(np.concatenate([c.table[i, :-(-keys // KB)] for i in range(3)]))
    e = p[3][held]
    # (the poison behind the last key has powers of its own)
    live = np.ones(e.shape, bool)
    last = [int(np.flatnonzero(held == c.table[i, (keys - 1) // KB])[0]) for i in range(3)]
    if keys % KB:
        live[last, :, keys % KB:] = False
    assert 124 <= e[live].min() and e[live].max() <= 128                         # normal numbers of fp16 at -10 and 9 as well
    e[live] = (e[live].astype(int) + power).astype(np.uint8)
    p[3][held] = e
    c.set_parts(p)
    assert np.array_equal(c.run(), one * np.float32(2.0 ** power))
