"""8-bit pages: append with quantisation, RoPE + append, read back, page copies,
page clears, against the format and the quantiser in numpy: every byte."""
import ctypes as C

import numpy as np
import pytest

from q8ref import HD, KB, Q8Pool, pack, quantise, unpack, values

pytestmark = pytest.mark.gpu
LAYER = 2


def _nova(model):
    import nova_amd
    return nova_amd.load(model)


def _expected(pool, table, pos0, off, k, v):
    """the pool's records after the append, with every other byte as it was"""
    rec = pool.rec.copy()
    kc, ks, vc, vs = (np.array(x) for x in unpack(rec))
    qk, qks = quantise(k)
    qv, qvs = quantise(v)
    for i in range(len(pos0)):
        for r in range(off[i], off[i + 1]):
            pos = pos0[i] + r - off[i]
            page, slot = table[i, pos // KB], pos % KB
            kc[page, :, slot], ks[page, :, slot] = qk[r], qks[r]
            vc[page, :, slot], vs[page, :, slot] = qv[r], qvs[r]
    return pack(kc, ks, vc, vs)


def _rows(rng, n, nkv):
    k = rng.standard_normal((n, nkv, HD)).astype(np.float32)
    k[..., 5] *= 8
    v = (rng.standard_normal((n, nkv, HD)) * np.exp(rng.standard_normal((n, nkv, 1)))).astype(np.float32)
    return k, v


CASES = [
    ("one token each", [0, 15, 16, 31, 100], [1, 1, 1, 1, 1]),
    ("inside a page", [3], [7]),
    ("whole pages", [0, 16, 32], [16, 32, 48]),
    ("ragged, some empty", [5, 0, 16, 15, 33, 7], [0, 40, 1, 18, 0, 0]),
    ("none but the last", [0, 0, 9], [0, 0, 23]),
    ("many sessions", [(7 * i) % 50 for i in range(131)], [(5 * i) % 4 for i in range(131)]),
]


@pytest.mark.parametrize("model", ["qwen25_1p5b", "qwen25_7b", "qwen25_14b"])
@pytest.mark.parametrize("name,pos0,count", CASES)
def test_store_and_read_back(model, name, pos0, count):
    nova = _nova(model)
    print(f"[case] q8 store {model} {name}", flush=True)
    pos0, count = np.array(pos0, np.int32), np.array(count)
    off = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    n = int(off[-1])
    pages = (pos0 + count + KB - 1) // KB
    pool = Q8Pool(nova, int(pages.sum()) + 3, LAYER, seed=len(name))
    table = pool.tables(pages)
    k, v = _rows(pool.rng, n + 2, nova.nkv)               # two rows behind the last session's
    want = _expected(pool, table, pos0, off, k, v)
    dt, dp, doff, dk, dv = (nova.upload(x) for x in (table, pos0, off, k, v))
    stream = nova.dev_stream_create()
    nova.launch_kv_q8_store_batch(pool.dev.ptr, dt.ptr, table.shape[1], dp.ptr, doff.ptr, len(pos0), n + 2, LAYER,
                                  pool.nb, dk.ptr, dv.ptr, stream)
    ko = nova.upload(np.full(k.shape, 7, np.float32))
    vo = nova.upload(np.full(v.shape, 7, np.float32))
    nova.launch_kv_q8_load_batch(pool.dev.ptr, dt.ptr, table.shape[1], dp.ptr, doff.ptr, len(pos0), n + 2, LAYER,
                                 pool.nb, ko.ptr, vo.ptr, stream)
    nova.dev_stream_sync(stream)
    nova.dev_stream_destroy(stream)
    assert np.array_equal(pool.pull(), want)
    for got, x in ((ko.numpy(k.shape, np.float32), k), (vo.numpy(v.shape, np.float32), v)):
        c, s = quantise(x[:n])
        assert np.array_equal(got[:n], c.astype(np.float32) * s[..., None])
        assert (got[n:] == 7).all()                       # rows behind the last sequence: left as they were


@pytest.mark.parametrize("n_sess,n", [(3, 1), (2, 37), (1, 16)])
def test_store_without_offsets(n_sess, n):
    """row_off NULL: n rows per session"""
    nova = _nova("qwen25_7b")
    pos0 = np.arange(n_sess, dtype=np.int32) * 11 + 2
    off = np.arange(n_sess + 1) * n
    pages = (pos0 + n + KB - 1) // KB
    pool = Q8Pool(nova, int(pages.sum()) + 1, LAYER, seed=n)
    table = pool.tables(pages)
    k, v = _rows(pool.rng, n_sess * n, nova.nkv)
    want = _expected(pool, table, pos0, off, k, v)
    dt, dp, dk, dv = (nova.upload(x) for x in (table, pos0, k, v))
    nova.launch_kv_q8_store_batch(pool.dev.ptr, dt.ptr, table.shape[1], dp.ptr, None, n_sess, n_sess * n, LAYER,
                                  pool.nb, dk.ptr, dv.ptr, None)
    nova.dev_sync()
    assert np.array_equal(pool.pull(), want)


def test_quantiser_borders():
    """Quotients exactly between two codes, one step to either side of it, rows of
    zeros, of tiny and of huge values, infinities and NaN."""
    nova = _nova("qwen25_1p5b")
    rng = np.random.default_rng(3)
    rows = []
    for top in (127.0, 1.0, 3.7, 1e-3, 0.99999994, 5e4):
        s = np.float32(np.float32(top) / np.float32(127))
        mid = ((np.arange(127) - 63).astype(np.float64) + 0.5) * np.float64(s)
        for step in (0, -1, 1):
            x = mid.astype(np.float32)
            x = np.nextafter(x, np.float32(step * np.inf), dtype=np.float32) if step else x
            rows.append(np.concatenate([[np.float32(top)], x]).astype(np.float32))
    rows.append(np.zeros(HD, np.float32))
    rows.append(np.full(HD, 2.0 ** -120, np.float32))                 # scale below the smallest normal number
    rows.append(np.full(HD, 127 * 2.0 ** -126, np.float32))           # scale exactly that
    rows.append((rng.standard_normal(HD) * 1e37).astype(np.float32))
    rows.append(np.full(HD, np.finfo(np.float32).max, np.float32))
    rows.append(np.full(HD, -1e-45, np.float32))
    for bad in (np.inf, -np.inf, np.nan):
        x = rng.standard_normal(HD).astype(np.float32)
        x[77] = bad
        rows.append(x)
    x = np.stack(rows)
    x = x[: len(x) // nova.nkv * nova.nkv].reshape(-1, nova.nkv, HD) if len(x) % nova.nkv == 0 else \
        np.concatenate([x, x[:nova.nkv - len(x) % nova.nkv]]).reshape(-1, nova.nkv, HD)
    n = len(x)
    v = np.ascontiguousarray(x[::-1])
    pool = Q8Pool(nova, 4, LAYER, seed=1)
    table = pool.tables([(n + KB - 1) // KB])
    pos0 = np.zeros(1, np.int32)
    want = _expected(pool, table, pos0, [0, n], x, v)
    dt, dp, dk, dv = (nova.upload(a) for a in (table, pos0, x, v))
    nova.launch_kv_q8_store_batch(pool.dev.ptr, dt.ptr, table.shape[1], dp.ptr, None, 1, n, LAYER, pool.nb, dk.ptr,
                                  dv.ptr, None)
    ko, vo = nova.alloc(x.nbytes), nova.alloc(x.nbytes)
    nova.launch_kv_q8_load_batch(pool.dev.ptr, dt.ptr, table.shape[1], dp.ptr, None, 1, n, LAYER, pool.nb, ko.ptr,
                                 vo.ptr, None)
    nova.dev_sync()
    for a, b in zip(unpack(pool.pull()), unpack(want)):
        assert np.array_equal(a, b, equal_nan=a.dtype.kind == "f")    # a NaN's payload is not fixed
    got = ko.numpy(x.shape, np.float32)
    bad = ~np.isfinite(x).all(-1)
    assert bad.sum() >= 3 and np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
    # a value is off by at most half a step: s / 2, plus the rounding of c * s and of s itself (127 ulps)
    _, s = quantise(x[~bad])
    lim = s[..., None].astype(np.float64) * (0.5 + 128 * 2.0 ** -23) + np.where(s == 0, 2.0 ** -119, 0)[..., None]
    assert (np.abs(got[~bad].astype(np.float64) - x[~bad]) <= lim).all()


@pytest.mark.parametrize("model", ["qwen25_1p5b", "qwen25_7b", "qwen25_14b"])
def test_rope_store_is_rope_then_store(model):
    """q rotated with the bits of launch_rope_batch, and the pages those of the
    plain append of the rotated k; k's buffer is left as passed."""
    nova = _nova(model)
    pos0, count = np.array([0, 30, 5, 17], np.int32), np.array([16, 1, 0, 23])
    off = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    n = int(off[-1])
    pages = (pos0 + count + KB - 1) // KB
    pool = Q8Pool(nova, int(pages.sum()) + 1, LAYER, seed=9)
    table = pool.tables(pages)
    k, v = _rows(pool.rng, n + 1, nova.nkv)
    q = pool.rng.standard_normal((n + 1, nova.nh, HD)).astype(np.float32)
    cs, sn = nova.alloc(64 * 64 * 4), nova.alloc(64 * 64 * 4)
    nova.launch_rope_table_rows(cs.ptr, sn.ptr, 64, None)
    dq, dk = nova.upload(q), nova.upload(k)
    for i in range(len(pos0)):
        nova.launch_rope_batch(dq.ptr + int(off[i]) * nova.nh * HD * 4, dk.ptr + int(off[i]) * nova.kvw * 4, int(count[i]),
                               int(pos0[i]), cs.ptr, sn.ptr, None)
    nova.dev_sync()
    want_q, rot_k = dq.numpy(q.shape, np.float32), dk.numpy(k.shape, np.float32)
    want = _expected(pool, table, pos0, off, rot_k, v)
    dt, dp, doff, dq, dk, dv = (nova.upload(x) for x in (table, pos0, off, q, k, v))
    nova.launch_rope_kv_q8_store_batch(dq.ptr, dk.ptr, dv.ptr, cs.ptr, sn.ptr, pool.dev.ptr, dt.ptr, table.shape[1],
                                       dp.ptr, doff.ptr, len(pos0), n + 1, LAYER, pool.nb, None)
    nova.dev_sync()
    assert np.array_equal(dq.numpy(q.shape, np.float32), want_q)
    assert np.array_equal(dk.numpy(k.shape, np.float32), k)
    assert np.array_equal(pool.pull(), want)


def test_rows_outside_the_table_are_left_out():
    """positions behind a session's table and pages outside the pool: nothing is
    written for them"""
    nova = _nova("qwen25_7b")
    pool = Q8Pool(nova, 6, LAYER, seed=4)
    table = np.array([[4, 1], [99, -1]], np.int32)
    pos0 = np.array([20, 0], np.int32)
    k, v = _rows(pool.rng, 48, nova.nkv)                  # 24 rows each: 20 .. 43 of a 32-token table, 0 .. 23
    want = _expected(pool, table, pos0[:1], [0, 12], k, v)
    dt, dp, dk, dv = (nova.upload(x) for x in (table, pos0, k, v))
    nova.launch_kv_q8_store_batch(pool.dev.ptr, dt.ptr, 2, dp.ptr, None, 2, 48, LAYER, pool.nb, dk.ptr, dv.ptr, None)
    nova.dev_sync()
    assert np.array_equal(pool.pull(), want)


def _ops(nova_amd, ops):
    return (nova_amd.CowOp * len(ops))(*[nova_amd.CowOp(s, d, t) for s, d, t in ops])


@pytest.mark.parametrize("model,n_ops", [("qwen25_1p5b", 1), ("qwen25_7b", 7), ("qwen25_14b", 3), ("qwen25_1p5b", 150)])
def test_cow_copies_every_layer(model, n_ops):
    import nova_amd
    nova = _nova(model)
    nb = 2 * n_ops + 5
    rng = np.random.default_rng(n_ops)
    host = rng.integers(0, 256, (nova.n_layers, nb, nova.kv_q8_page_bytes()), dtype=np.uint8)
    pages = rng.permutation(nb)
    ops = [(int(pages[e // 3]), int(pages[n_ops + 2 + e]), 2 * e + 1) for e in range(n_ops)]    # sources are shared
    table = rng.integers(0, nb, 2 * n_ops + 1).astype(np.int32)
    dev, dt = nova.upload(host), nova.upload(table)
    nova.launch_kv_q8_cow_apply(dev.ptr, nb, dt.ptr, _ops(nova_amd, ops), n_ops, None)
    nova.dev_sync()
    for s, d, t in ops:
        host[:, d] = host[:, s]
        table[t] = d
    assert np.array_equal(dev.numpy(host.shape, np.uint8), host)
    assert np.array_equal(dt.numpy(table.shape, np.int32), table)


def test_zero_pages():
    nova = _nova("qwen25_7b")
    nb = 9
    host = np.random.default_rng(5).integers(0, 256, (nova.n_layers, nb, nova.kv_q8_page_bytes()), dtype=np.uint8)
    pages = np.array([8, 0, 3, 3, 77, -2], np.int32)       # a page twice; pages that are not there
    dev, dp = nova.upload(host), nova.upload(pages)
    nova.launch_kv_q8_zero_pages(dev.ptr, nb, dp.ptr, len(pages), None)
    nova.dev_sync()
    host[:, [8, 0, 3]] = 0
    assert np.array_equal(dev.numpy(host.shape, np.uint8), host)


def test_pool_beyond_32_bit_offsets():
    """the last layer of a pool of 5 GB"""
    nova = _nova("qwen25_7b")
    nb, layer = 11000, 27
    page = nova.kv_q8_page_bytes()
    assert layer * nb * page > 2 ** 32
    dev = nova.alloc((layer + 1) * nb * page)
    k, v = _rows(np.random.default_rng(6), 16, nova.nkv)
    table, pos0 = np.array([[nb - 1]], np.int32), np.zeros(1, np.int32)
    dt, dp, dk, dv = (nova.upload(x) for x in (table, pos0, k, v))
    ko, vo = nova.alloc(k.nbytes), nova.alloc(v.nbytes)
    nova.launch_kv_q8_store_batch(dev.ptr, dt.ptr, 1, dp.ptr, None, 1, 16, layer, nb, dk.ptr, dv.ptr, None)
    nova.launch_kv_q8_load_batch(dev.ptr, dt.ptr, 1, dp.ptr, None, 1, 16, layer, nb, ko.ptr, vo.ptr, None)
    nova.dev_sync()
    rec = nova.download(dev, (nova.nkv, 4224), np.uint8, (layer * nb + nb - 1) * page)
    kq, ks = quantise(k.transpose(1, 0, 2))
    vq, vs = quantise(v.transpose(1, 0, 2))
    assert np.array_equal(rec, pack(kq, ks, vq, vs))
    want_k, want_v = values(rec[None], np.zeros(1, int), 16)
    assert np.array_equal(ko.numpy(k.shape, np.float32), want_k.astype(np.float32))
    assert np.array_equal(vo.numpy(v.shape, np.float32), want_v.astype(np.float32))
