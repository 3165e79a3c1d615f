"""Attention over 4-bit pages with so many sessions that the batch is read 64 at a time
and its long sessions are cut."""
import numpy as np
import pytest

from q4ref import HD, Call, Q4Pool, assert_within, attention, values

pytestmark = pytest.mark.gpu
MODELS = ["qwen25_1p5b", "qwen25_7b", "qwen25_14b"]


def _lengths(n_sess, seed):
    """short sessions, an empty one in between, and long ones in the first and the last
    batch of 64"""
    n = np.random.default_rng(seed).integers(1, 120, n_sess)
    n[::17] = 0
    n[[2, 63, n_sess - 1]] = 4500, 900, 5000
    return n


def _parts(c):
    return c.nova.download(c.ws, (len(c.past), 4), np.int32)     # first slot, parts, rows, first row


@pytest.mark.parametrize("n_sess", [33, 64, 65])
@pytest.mark.parametrize("model", MODELS)
def test_one_long_session_among_short_ones_is_cut(model, n_sess):
    n_keys = np.random.default_rng(n_sess).integers(1, 64, n_sess)
    n_keys[n_sess - 3] = 12000
    d = Call(model, n_keys, seed=71)
    d.run()
    info = _parts(d)
    assert (info[:, 2] == 1).all() and list(info[:, 3]) == list(range(n_sess))
    assert (np.delete(info[:, 1], n_sess - 3) == 1).all()
    assert info[n_sess - 3, 1] >= 12000 // 64 // 12
    d.check(f"{model} {n_sess}")


@pytest.mark.parametrize("n_sess", [65, 130, 200])
@pytest.mark.parametrize("model", MODELS)
def test_decode_batches_of_64(model, n_sess):
    d = Call(model, _lengths(n_sess, n_sess), seed=72)
    d.run()
    info = _parts(d)
    assert info[2, 1] > 1 and info[n_sess - 1, 1] > 1
    d.check(f"{model} {n_sess}")


@pytest.mark.parametrize("n_sess", [65, 150])
@pytest.mark.parametrize("max_q", [1, 4, 11])
@pytest.mark.parametrize("model", MODELS)
def test_chunk_batches_of_64(model, max_q, n_sess):
    """one 16-column block, two, and groups of 64 columns"""
    rng = np.random.default_rng(n_sess + max_q)
    count = rng.integers(0, max_q + 1, n_sess)
    count[[2, 63, n_sess - 1]] = max_q
    c = Call(model, _lengths(n_sess, max_q), count, seed=73)
    c.run()
    c.check(f"{model} {n_sess}")


@pytest.mark.parametrize("stride", [1, 49])
@pytest.mark.parametrize("decode", [True, False])
def test_as_many_sessions_as_a_call_takes(decode, stride):
    """65535 sessions over 40 pages that many of them read, with and without a joining launch"""
    import nova_amd
    nova = nova_amd.load("qwen25_1p5b")
    n, nb = 65535, 40
    print(f"[case] {n} sessions stride={stride} decode={decode}", flush=True)
    pool = Q4Pool(nova, nb, 0, 5)
    rng = np.random.default_rng(stride)
    table = np.full((n, stride), -1, np.int32)
    table[:, 0] = rng.integers(0, nb, n)
    keys = rng.integers(0 if decode else 1, 17, n).astype(np.int32)
    past = keys if decode else keys - 1
    q = rng.standard_normal((n, nova.nh, HD)).astype(np.float32)
    dt, dp, dq, o = nova.upload(table), nova.upload(past), nova.upload(q), nova.alloc(q.nbytes)
    if decode:
        ws = nova.alloc(nova.attn_decode_q4_workspace_bytes(n))
        nova.launch_attn_decode_q4_batch(dq.ptr, pool.dev.ptr, dt.ptr, stride, dp.ptr, n, 0, nb, o.ptr, ws.ptr, None)
    else:
        ws = nova.alloc(nova.attn_chunk_q4_workspace_bytes(n, n, 1))
        nova.launch_attn_chunk_q4_batch(dq.ptr, pool.dev.ptr, dt.ptr, stride, dp.ptr, None, n, n, 1, 0, nb, o.ptr, ws.ptr, None)
    nova.dev_sync()
    got = o.numpy(q.shape, np.float32)
    assert np.isfinite(got).all() and not got[keys == 0].any()
    for i in [0, 1, 63, 64, 65, 255, 256, 32767, 65279, 65280, 65281, n - 2, n - 1]:
        k, v = values(pool.rec, table[i], int(keys[i]))
        ref, tol = attention(q[i:i + 1], k, v, int(keys[i]), nova.group)
        assert_within(got[i:i + 1], ref, tol, f"session {i}")
