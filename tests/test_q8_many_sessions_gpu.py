"""Attention over 8-bit pages with so many sessions that the batch is read 64 at a time
and its long sessions are cut."""
import numpy as np
import pytest

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
