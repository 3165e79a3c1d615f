"""Calls at the limits of what their arguments may be."""
import numpy as np
import pytest

import q8ref
from q8ref import HD, Q8Pool
from test_q4_store_gpu import _angles, _turn

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


def test_rotation_of_many_rows():
    """rows past 65536, some of them empty, into other buffers and in place"""
    nova, rows, rot = _nova("qwen25_1p5b"), 65536 + 41, 96
    print(f"[case] rope rows {rows}", flush=True)
    rng = np.random.default_rng(rows)
    q, k = (rng.standard_normal((rows, n, HD), np.float32) for n in (nova.nh, nova.nkv))
    c, s = _angles(rng, rows, rot)
    pos = np.arange(rows, dtype=np.int32)
    pos[[7, 65535, 65536 + 7, 65536 + 40]] = -1
    dq, dk, dc, ds, dp = (nova.upload(x) for x in (q, k, c, s, pos))
    oq, ok = (nova.upload(np.full(x.shape, 7, np.float32)) for x in (q, k))
    some = np.concatenate([np.arange(40), np.arange(65500, rows)])
    for to_q, to_k, rest in ((oq, ok, None), (dq, dk, 0)):
        nova.launch_rope_rows(dq.ptr, dk.ptr, dp.ptr, dc.ptr, ds.ptr, rows, rot, 0, to_q.ptr, to_k.ptr, None)
        nova.dev_sync()
        for to, x in ((to_q, q), (to_k, k)):
            want = _turn(x[some], c[some], s[some], rot, 0)
            want[pos[some] < 0] = 7 if rest is None else x[some][pos[some] < 0]
            assert np.array_equal(to.numpy(x.shape, np.float32)[some], want)


def test_rotation_of_as_many_rows_as_a_call_takes():
    """2^24 rows, all but the first of them empty"""
    nova, rows, rot = _nova("qwen25_1p5b"), 1 << 24, 128
    print(f"[case] rope rows {rows}", flush=True)
    rng = np.random.default_rng(1)
    q, k = (rng.standard_normal((3, n, HD), np.float32) for n in (nova.nh, nova.nkv))
    c, s = _angles(rng, 3, rot)
    pos = np.full(rows, -1, np.int32)
    pos[:2] = 5
    dq, dk, dc, ds, dp = (nova.upload(x) for x in (q, k, c, s, pos))     # (empty rows are not read)
    nova.launch_rope_rows(dq.ptr, dk.ptr, dp.ptr, dc.ptr, ds.ptr, rows, rot, 0, dq.ptr, dk.ptr, None)
    nova.dev_sync()
    for dev, x in ((dq, q), (dk, k)):
        got = dev.numpy(x.shape, np.float32)
        assert np.array_equal(got[:2], _turn(x, c, s, rot, 0)[:2]) and np.array_equal(got[2], x[2])


@pytest.mark.parametrize("rot", [128, 6])
def test_rotation_of_more_rows_than_a_launch_takes(rot):
    """2^20 rows and 41, of which the first ones and those around 2^20 turn, in place; the others are empty"""
    nova, border = _nova("qwen25_1p5b"), 1 << 20
    rows = border + 41
    print(f"[case] rope rows {rows} rot={rot}", flush=True)
    rng = np.random.default_rng(rot)
    some = np.concatenate([np.arange(3), np.arange(border - 4, border + 41)])
    c, s = _angles(rng, len(some), rot)
    pos = np.full(rows, -1, np.int32)
    pos[some] = 9
    pos[[border - 2, border + 3, rows - 1]] = -1
    dp = nova.upload(pos)
    dc, ds = (nova.alloc(rows * rot // 2 * 4) for _ in range(2))
    dev = {n: nova.alloc(rows * n * HD * 4) for n in (nova.nh, nova.nkv)}
    host = {n: rng.standard_normal((len(some), n, HD), np.float32) for n in dev}
    # (the rows that turn lie in two runs)
    for lo, hi, at in ((0, 3, 0), (3, len(some), border - 4)):
        for d, x in ((dc, c), (ds, s), *((dev[n], host[n]) for n in dev)):
            part = np.ascontiguousarray(x[lo:hi])
            nova.dev_upload(d.ptr + at * part[0].nbytes, part.ctypes.data, part.nbytes)
    q, k = dev[nova.nh].ptr, dev[nova.nkv].ptr
    nova.launch_rope_rows(q, k, dp.ptr, dc.ptr, ds.ptr, rows, rot, 0, q, k, None)
    nova.dev_sync()
    for n, x in host.items():
        want = np.where((pos[some] >= 0)[:, None, None], _turn(x, c, s, rot, 0), x)
        got = np.concatenate([nova.download(dev[n], (hi - lo, n, HD), np.float32, at * n * HD * 4)
                              for lo, hi, at in ((0, 3, 0), (3, len(some), border - 4))])
        assert np.array_equal(got, want)
