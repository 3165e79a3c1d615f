"""4-bit pages: append with quantisation, rotation + append, read back, page copies, page
clears, against the format and the quantiser in numpy: every byte."""
import numpy as np
import pytest

from q4ref import HD, KB, Q4Pool, decode, pack, quantise, unpack, values

pytestmark = pytest.mark.gpu
LAYER = 2
MODELS = ["qwen25_1p5b", "qwen25_7b", "qwen25_14b"]


def _nova(model):
    import nova_amd
    return nova_amd.load(model)


def _expected(pool, table, pos0, off, k, v):
    """the pool's records after the append, with every other byte as it was"""
    kc, ke, vc, ve = (np.array(x) for x in unpack(pool.rec))
    qk, qke = quantise(k)
    qv, qve = quantise(v)
    for i in range(len(pos0)):
        for r in range(off[i], off[i + 1]):
            pos = pos0[i] + r - off[i]
            page, slot = table[i, pos // KB], pos % KB
            kc[page, :, slot], ke[page, :, slot] = qk[r], qke[r]
            vc[page, :, slot], ve[page, :, slot] = qv[r], qve[r]
    return pack(kc, ke, vc, ve)


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


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("name,pos0,count", CASES)
def test_store_and_read_back(model, name, pos0, count):
    nova = _nova(model)
    print(f"[case] q4 store {model} {name}", flush=True)
    pos0, count = np.array(pos0, np.int32), np.array(count)
    off = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    n = int(off[-1])
    pages = (pos0 + count + KB - 1) // KB
    pool = Q4Pool(nova, int(pages.sum()) + 3, LAYER, seed=len(name))
    table = pool.tables(pages)
    k, v = _rows(pool.rng, n + 2, nova.nkv)               # two rows behind the last session's
    want = _expected(pool, table, pos0, off, k, v)
    dt, dp, doff, dk, dv = (nova.upload(x) for x in (table, pos0, off, k, v))
    stream = nova.dev_stream_create()
    nova.launch_kv_q4_store_batch(pool.dev.ptr, dt.ptr, table.shape[1], dp.ptr, doff.ptr, len(pos0), n + 2, LAYER,
                                  pool.nb, dk.ptr, dv.ptr, stream)
    ko = nova.upload(np.full(k.shape, 7, np.float32))
    vo = nova.upload(np.full(v.shape, 7, np.float32))
    nova.launch_kv_q4_load_batch(pool.dev.ptr, dt.ptr, table.shape[1], dp.ptr, doff.ptr, len(pos0), n + 2, LAYER,
                                 pool.nb, ko.ptr, vo.ptr, stream)
    nova.dev_stream_sync(stream)
    nova.dev_stream_destroy(stream)
    assert np.array_equal(pool.pull(), want)
    for got, x in ((ko.numpy(k.shape, np.float32), k), (vo.numpy(v.shape, np.float32), v)):
        assert np.array_equal(got[:n], decode(*quantise(x[:n])))
        assert (got[n:] == 7).all()                       # rows behind the last sequence: left as they were


@pytest.mark.parametrize("n_sess,n", [(3, 1), (2, 37), (1, 16)])
def test_store_without_offsets(n_sess, n):
    """row_off NULL: n rows per session"""
    nova = _nova("qwen25_7b")
    pos0 = np.arange(n_sess, dtype=np.int32) * 11 + 2
    off = np.arange(n_sess + 1) * n
    pages = (pos0 + n + KB - 1) // KB
    pool = Q4Pool(nova, int(pages.sum()) + 1, LAYER, seed=n)
    table = pool.tables(pages)
    k, v = _rows(pool.rng, n_sess * n, nova.nkv)
    want = _expected(pool, table, pos0, off, k, v)
    dt, dp, dk, dv = (nova.upload(x) for x in (table, pos0, k, v))
    nova.launch_kv_q4_store_batch(pool.dev.ptr, dt.ptr, table.shape[1], dp.ptr, None, n_sess, n_sess * n, LAYER,
                                  pool.nb, dk.ptr, dv.ptr, None)
    nova.dev_sync()
    assert np.array_equal(pool.pull(), want)


def test_quantiser_borders():
    """Values exactly between two of the format's, one step to either side of it, at powers
    from the smallest to the largest; zeros, infinities and NaN in either half of a row."""
    nova = _nova("qwen25_1p5b")
    rng = np.random.default_rng(3)
    mid = np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 7], np.float32)
    rows = []
    for power in (-126, -102, -101, -100, -99, -60, -1, 0, 3, 95, 96, 97, 125):
        for top in (7.0, 3.6, 6.0):
            with np.errstate(over="ignore"):
                x = np.ldexp(np.concatenate([[np.float32(top)], mid, -mid]).astype(np.float32), power)
                # (the neighbours of 7 change the power: they get blocks of their own)
                block = [x, np.nextafter(x, np.float32(np.inf)), np.nextafter(x, np.float32(0))]
            row = np.zeros((4, 32), np.float32)
            for j, b in enumerate(block):
                row[j, :len(b)] = np.where(np.isfinite(b), b, 0)
            row[3] = rng.uniform(-1, 1, 32) * np.ldexp(np.float32(1), min(power, 120))
            rows.append(row.ravel())
    rows.append(np.zeros(HD, np.float32))
    rows.append(np.full(HD, np.finfo(np.float32).max, np.float32))
    rows.append(np.full(HD, -1e-45, np.float32))
    for bad, at in ((np.inf, 77), (-np.inf, 3), (np.nan, 127), (-np.nan, 32)):
        x = rng.standard_normal(HD).astype(np.float32)
        x[at] = bad
        rows.append(x)
    rows += rows[:len(rows) % nova.nkv]
    x = np.stack(rows).astype(np.float32).reshape(-1, nova.nkv, HD)
    n = len(x)
    v = np.ascontiguousarray(x[::-1])
    pool = Q4Pool(nova, 6, LAYER, seed=1)
    table = pool.tables([(n + KB - 1) // KB])
    pos0 = np.zeros(1, np.int32)
    want = _expected(pool, table, pos0, [0, n], x, v)
    dt, dp, dk, dv = (nova.upload(a) for a in (table, pos0, x, v))
    nova.launch_kv_q4_store_batch(pool.dev.ptr, dt.ptr, table.shape[1], dp.ptr, None, 1, n, LAYER, pool.nb, dk.ptr,
                                  dv.ptr, None)
    ko, vo = nova.alloc(x.nbytes), nova.alloc(x.nbytes)
    nova.launch_kv_q4_load_batch(pool.dev.ptr, dt.ptr, table.shape[1], dp.ptr, None, 1, n, LAYER, pool.nb, ko.ptr,
                                 vo.ptr, None)
    nova.dev_sync()
    got = pool.pull()
    for name, a, b in zip(("K codes", "K exponents", "V codes", "V exponents"), unpack(got), unpack(want)):
        assert np.array_equal(a, b), (name, np.argwhere(a != b)[:5], a[a != b][:5], b[a != b][:5])
    for out, src in ((ko, x), (vo, v)):
        assert np.array_equal(out.numpy(x.shape, np.float32), decode(*quantise(src)), equal_nan=True)


FORMS = [(128, 0), (128, 1), (64, 0), (64, 1), (96, 0), (24, 0), (20, 0), (20, 1), (2, 0), (2, 1), (6, 1), (126, 0), (100, 0)]


def _angles(rng, n, rot):
    a = rng.uniform(-50, 50, (n, rot // 2))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def _turn(x, c, s, rot, beside):
    """fp32, every product rounded; x [n][heads][128]"""
    y = x.copy()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if beside else (slice(0, rot // 2), slice(rot // 2, rot))
    c, s = c[:, None], s[:, None]
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


@pytest.mark.parametrize("rot,beside", FORMS)
def test_rope_store_is_rope_then_store(rot, beside):
    """q turned with the bits of the formula in fp32, out of place and in place, and the pages
    those of the plain append of the turned k; k's buffer is left as passed."""
    nova = _nova(MODELS[rot % 3])
    print(f"[case] rope + q4 store rot={rot} beside={beside}", flush=True)
    pos0, count = np.array([0, 30, 5, 17], np.int32), np.array([16, 1, 0, 23])
    off = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    n = int(off[-1])
    pages = (pos0 + count + KB - 1) // KB
    pool = Q4Pool(nova, int(pages.sum()) + 1, LAYER, seed=9)
    table = pool.tables(pages)
    k, v = _rows(pool.rng, n + 1, nova.nkv)
    q = pool.rng.standard_normal((n + 1, nova.nh, HD)).astype(np.float32)
    c, s = _angles(pool.rng, n + 1, rot)
    want_q = _turn(q, c, s, rot, beside)
    want_q[n] = q[n]                                      # a row behind the last session's
    want = _expected(pool, table, pos0, off, _turn(k, c, s, rot, beside), v)
    dt, dp, doff, dq, dk, dv, dc, ds = (nova.upload(x) for x in (table, pos0, off, q, k, v, c, s))
    out = nova.upload(np.full(q.shape, 7, np.float32))
    for to in (out, dq):
        nova.launch_rope_rows_kv_q4_store_batch(dq.ptr, dk.ptr, dv.ptr, dc.ptr, ds.ptr, rot, beside, pool.dev.ptr, dt.ptr,
                                                table.shape[1], dp.ptr, doff.ptr, len(pos0), n + 1, LAYER, pool.nb, to.ptr,
                                                None)
        nova.dev_sync()
        got = to.numpy(q.shape, np.float32)
        assert np.array_equal(got[:n], want_q[:n])
        assert (got[n] == 7).all() if to is out else np.array_equal(got[n], q[n])
        assert np.array_equal(pool.pull(), want)
    assert np.array_equal(dk.numpy(k.shape, np.float32), k)


def test_rows_outside_the_table_are_left_out():
    """positions behind a session's table, pages outside the pool, a session that starts below 0:
    nothing is written for them"""
    nova = _nova("qwen25_7b")
    pool = Q4Pool(nova, 6, LAYER, seed=4)
    table = np.array([[4, 1], [99, -1], [0, 2]], np.int32)
    pos0 = np.array([20, 0, -3], np.int32)
    k, v = _rows(pool.rng, 72, nova.nkv)                  # 24 rows each: 20 .. 43 of a 32-token table, 0 .. 23
    want = _expected(pool, table, pos0[:1], [0, 12], k, v)
    dt, dp, dk, dv = (nova.upload(x) for x in (table, pos0, k, v))
    nova.launch_kv_q4_store_batch(pool.dev.ptr, dt.ptr, 2, dp.ptr, None, 3, 72, LAYER, pool.nb, dk.ptr, dv.ptr, None)
    nova.dev_sync()
    assert np.array_equal(pool.pull(), want)


@pytest.mark.parametrize("model,n_ops", [("qwen25_1p5b", 1), ("qwen25_7b", 7), ("qwen25_14b", 3), ("qwen25_1p5b", 150)])
def test_cow_copies_every_layer(model, n_ops):
    import nova_amd
    nova = _nova(model)
    nb = 2 * n_ops + 5
    rng = np.random.default_rng(n_ops)
    host = rng.integers(0, 256, (nova.n_layers, nb, nova.kv_q4_page_bytes()), dtype=np.uint8)
    pages = rng.permutation(nb)
    ops = [(int(pages[e // 3]), int(pages[n_ops + 2 + e]), 2 * e + 1) for e in range(n_ops)]    # sources are shared
    table = rng.integers(0, nb, 2 * n_ops + 1).astype(np.int32)
    dev, dt = nova.upload(host), nova.upload(table)
    arr = (nova_amd.CowOp * n_ops)(*[nova_amd.CowOp(*o) for o in ops])
    nova.launch_kv_q4_cow_apply(dev.ptr, nb, dt.ptr, arr, n_ops, None)
    nova.dev_sync()
    for s, d, t in ops:
        host[:, d] = host[:, s]
        table[t] = d
    assert np.array_equal(dev.numpy(host.shape, np.uint8), host)
    assert np.array_equal(dt.numpy(table.shape, np.int32), table)


def test_zero_pages():
    nova = _nova("qwen25_7b")
    nb = 9
    host = np.random.default_rng(5).integers(0, 256, (nova.n_layers, nb, nova.kv_q4_page_bytes()), dtype=np.uint8)
    pages = np.array([8, 0, 3, 3, 77, -2], np.int32)       # a page twice; pages that are not there
    dev, dp = nova.upload(host), nova.upload(pages)
    nova.launch_kv_q4_zero_pages(dev.ptr, nb, dp.ptr, len(pages), None)
    nova.dev_sync()
    host[:, [8, 0, 3]] = 0
    assert np.array_equal(dev.numpy(host.shape, np.uint8), host)


def test_pool_beyond_32_bit_offsets():
    """the last layer of a pool of 5 GB"""
    nova = _nova("qwen25_7b")
    nb, layer = 21000, 27
    page = nova.kv_q4_page_bytes()
    assert layer * nb * page > 2 ** 32
    dev = nova.alloc((layer + 1) * nb * page)
    k, v = _rows(np.random.default_rng(6), 16, nova.nkv)
    table, pos0 = np.array([[nb - 1]], np.int32), np.zeros(1, np.int32)
    dt, dp, dk, dv = (nova.upload(x) for x in (table, pos0, k, v))
    ko, vo = nova.alloc(k.nbytes), nova.alloc(v.nbytes)
    nova.launch_kv_q4_store_batch(dev.ptr, dt.ptr, 1, dp.ptr, None, 1, 16, layer, nb, dk.ptr, dv.ptr, None)
    nova.launch_kv_q4_load_batch(dev.ptr, dt.ptr, 1, dp.ptr, None, 1, 16, layer, nb, ko.ptr, vo.ptr, None)
    nova.dev_sync()
    rec = nova.download(dev, (nova.nkv, 2176), np.uint8, (layer * nb + nb - 1) * page)
    assert np.array_equal(rec, pack(*quantise(k.transpose(1, 0, 2)), *quantise(v.transpose(1, 0, 2))))
    want_k, want_v = values(rec[None], np.zeros(1, int), 16)
    assert np.array_equal(ko.numpy(k.shape, np.float32), want_k)
    assert np.array_equal(vo.numpy(v.shape, np.float32), want_v)
