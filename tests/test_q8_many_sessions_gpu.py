"""Attention over 8-bit pages with so many sessions that the batch is read 64 at a time
and its long sessions are cut."""
import numpy as np
import pytest

from q8ref import KB, assert_within, attention, values
from test_q8_attn_gpu import MODELS, Chunk, Decode

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_sess", [33, 60, 64, 65])
@pytest.mark.parametrize("model", MODELS)
def test_one_long_session_among_short_ones_is_cut(model, n_sess):
    """however many sessions stand beside it: its parts are at most six tiles of 64 keys
    each (the work split's share here is four, and half as much again at most)"""
    n_keys = np.random.default_rng(n_sess).integers(1, 64, n_sess)
    n_keys[n_sess - 3] = 12000
    d = Decode(model, n_keys, seed=71)
    d.launch()
    d.nova.dev_sync()
    info = d.nova.download(d.ws, (n_sess, 4), np.int32)       # first slot, parts, rows, first row
    assert (info[:, 2] == 1).all() and list(info[:, 3]) == list(range(n_sess))
    assert (np.delete(info[:, 1], n_sess - 3) == 1).all()
    assert info[n_sess - 3, 1] >= -(-12000 // 64) // 6
    d.check(f"{model} {n_sess}")


def _check(x, n_keys, first_row, count, first_key):
    """every session against the formula; rows of session i from first_row[i], the first
    of them seeing first_key[i] keys"""
    got, worst = x.result(), 0.0
    for i, n in enumerate(n_keys):
        if count[i] == 0:
            continue
        a, b = int(first_row[i]), int(first_row[i] + count[i])
        pages = x.table[i, :-(-int(n) // KB)]
        k, v = values(x.pool.rec[pages], np.arange(len(pages)), int(n))
        ref, tol = attention(x.q[a:b], k, v, int(first_key[i]), x.nova.group)
        worst = max(worst, assert_within(got[a:b], ref, tol, f"session {i} of {n} keys"))
    print(f"  {worst:.3f} of the bound")


def _lengths(n_sess, seed):
    """short sessions, an empty one in between, and long ones in the first and the last
    batch of 64"""
    n = np.random.default_rng(seed).integers(1, 120, n_sess)
    n[::17] = 0
    n[[2, 63, n_sess - 1]] = 4500, 900, 5000
    return n


@pytest.mark.parametrize("n_sess", [65, 130, 200])
@pytest.mark.parametrize("model", MODELS)
def test_decode_batches_of_64(model, n_sess):
    d = Decode(model, _lengths(n_sess, n_sess), seed=72)
    assert d.table.shape[1] > 48                             # not the form without a join
    d.launch()
    d.nova.dev_sync()
    info = d.nova.download(d.ws, (n_sess, 4), np.int32)
    assert info[2, 1] > 1 and info[n_sess - 1, 1] > 1
    _check(d, d.n_keys, np.arange(n_sess), np.ones(n_sess, int), d.n_keys)


@pytest.mark.parametrize("n_sess", [65, 130, 200])
@pytest.mark.parametrize("max_q", [1, 4, 11])
@pytest.mark.parametrize("model", MODELS)
def test_chunk_batches_of_64(model, max_q, n_sess):
    """one 16-column block, two, and groups of 64 columns"""
    rng = np.random.default_rng(n_sess + max_q)
    count = rng.integers(0, max_q + 1, n_sess)
    count[[2, 63, n_sess - 1]] = max_q
    c = Chunk(model, _lengths(n_sess, max_q), count, seed=73)
    c.launch()
    c.nova.dev_sync()
    _check(c, c.past + c.count, c.off, c.count, c.past + 1)
    assert (c.result()[c.off[-1]:] == 3).all()               # rows behind the last session's
