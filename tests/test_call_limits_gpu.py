"""Calls at the limits of what their arguments may be."""
import numpy as np
import pytest

import q8ref
from q8ref import HD, Q8Pool

pytestmark = pytest.mark.gpu


def _nova(model):
    import nova_amd
    return nova_amd.load(model)


@pytest.mark.parametrize("stride", [1, 49])
@pytest.mark.parametrize("rows", [0, 1, 3])
def test_8_bit_attention_of_as_many_sessions_as_a_call_takes(rows, stride):
    """65535 sessions over 40 pages that many of them read, with and without a joining launch: a decode
    (rows 0), one row each, and three rows of every 512th and of the last"""
    nova, n, nb = _nova("qwen25_1p5b"), 65535, 40
    print(f"[case] 8-bit, {n} sessions stride={stride} rows={rows}", flush=True)
    pool = Q8Pool(nova, nb, 0, 5)
    rng = np.random.default_rng(stride)
    table = np.full((n, stride), -1, np.int32)
    table[:, 0] = rng.integers(0, nb, n)
    keys = rng.integers(rows, 17, n).astype(np.int32)        # with the rows
    past = keys - rows
    count = np.ones(n, np.int64)
    if rows == 3:
        count = np.where(np.arange(n) % 512 == 510, 3, 0)    # 65534, the last, among them
    off = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    total = int(off[-1])
    q = rng.standard_normal((total, nova.nh, HD)).astype(np.float32)
    dt, dp, dq, doff, o = nova.upload(table), nova.upload(past), nova.upload(q), nova.upload(off), nova.alloc(q.nbytes)
    if rows == 0:
        ws = nova.alloc(nova.attn_decode_q8_workspace_bytes(n))
        nova.launch_attn_decode_q8_batch(dq.ptr, pool.dev.ptr, dt.ptr, stride, dp.ptr, n, 0, nb, o.ptr, ws.ptr, None)
    else:
        ws = nova.alloc(nova.attn_chunk_q8_workspace_bytes(n, total, rows))
        nova.launch_attn_chunk_q8_batch(dq.ptr, pool.dev.ptr, dt.ptr, stride, dp.ptr, doff.ptr, n, total, rows, 0, nb, o.ptr,
                                        ws.ptr, None)
    nova.dev_sync()
    got = o.numpy(q.shape, np.float32)
    assert np.isfinite(got).all()
    if rows == 0:
        assert not got[keys == 0].any()
    some = [i for i in (0, 1, 63, 64, 65, 255, 256, 510, 32767, 32766, 65279, 65280, 65281, n - 2, n - 1) if count[i]]
    assert n - 1 in some
    for i in some:
        a, b = off[i], off[i + 1]
        k, v = q8ref.values(pool.rec, table[i], int(keys[i]))
        ref, tol = q8ref.attention(q[a:b], k, v, int(past[i]) + (1 if rows else 0), nova.group)
        q8ref.assert_within(got[a:b], ref, tol, f"session {i}")
