"""Attention over 4-bit pages against the formula in float64 over the values the
codes stand for, with the bound derived in q4ref.attention."""
import numpy as np
import pytest

from q4ref import HD, KB, NAN, Call, assert_within, attention, decode, quantise, values

pytestmark = pytest.mark.gpu
MODELS = ["qwen25_1p5b", "qwen25_7b", "qwen25_14b"]

LENGTHS = [
    ("one", [1]),
    ("borders", [15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129]),
    ("with none", [0, 5, 0, 300, 0]),
    ("none at all", [0, 0]),
    ("one long", [5003]),
    ("ragged", [700, 1, 4097, 64, 2000, 333]),
    ("many", [(37 * i) % 200 for i in range(150)]),
    ("few and long", [16384, 9001]),
]


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("name,n_keys", LENGTHS)
def test_decode(model, name, n_keys):
    print(f"[case] q4 decode {model} {name}", flush=True)
    d = Call(model, n_keys, seed=len(name))
    d.run()
    d.check(f"{model} {name}")


CHUNKS = [
    ("one row each", [0, 15, 16, 63, 64, 500], [1, 1, 1, 1, 1, 1]),
    ("drafts", [900, 33, 0, 4000, 127], [2, 8, 5, 3, 1]),
    ("drafts behind a long one", [16000], [4]),
    ("some empty", [0, 100, 7, 0, 12], [0, 30, 0, 17, 0]),
    ("from nothing", [0, 0, 0], [1, 16, 65]),
    ("middle", [100, 0, 700, 48], [64, 100, 33, 129]),
    ("prompt", [0], [300]),
    ("behind a prefix", [1500], [77]),
    ("many", [(13 * i) % 90 for i in range(90)], [(7 * i) % 11 for i in range(90)]),
]


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("name,past,count", CHUNKS)
def test_chunk(model, name, past, count):
    print(f"[case] q4 chunk {model} {name}", flush=True)
    c = Call(model, past, count, seed=len(name))
    c.run()
    c.check(f"{model} {name}")


@pytest.mark.parametrize("model,past,count", [
    ("qwen25_7b", [0, 900, 333, 64, 1023, 500], [512, 300, 511, 256, 400, 513]),       # enough rows to fill the chip
    ("qwen25_7b", [30000], [8]),                             # one group in as many pieces as there are stretches
    ("qwen25_14b", [9000, 9000, 70], [12, 7, 9]),
    ("qwen25_7b", [12000] + [40] * 12, [5] + [6] * 12),      # one long, many short
    ("qwen25_1p5b", [(7 * i) % 4 for i in range(300)], [10] + [(11 * i) % 11 for i in range(299)]),
], ids=["wide", "one", "two of three", "one of many", "tiny"])
def test_work_cut_in_many_ways(model, past, count):
    c = Call(model, past, count, seed=60 + len(past))
    c.run()
    c.check("pieces")


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1.0, 30.0, 1e4])
def test_query_sizes(scale):
    """from scores that are all alike to one key that takes everything"""
    for c in (Call("qwen25_7b", [1, 100, 900], seed=5, scale=scale), Call("qwen25_7b", [50, 200], [40, 3], seed=22, scale=scale)):
        c.run()
        c.check(f"scale {scale}")


@pytest.mark.parametrize("n", [1, 6, 50])
def test_chunk_without_offsets(n):
    c = Call("qwen25_14b", [0, 77, 15], [n] * 3, seed=23, behind=0, offsets=False)
    c.run()
    c.check("uniform")


def test_chunk_larger_max_q():
    c = Call("qwen25_7b", [40, 900], [3, 5], seed=24, max_q=10, behind=8)
    c.run()
    c.check("max_q")


def test_rows_behind_max_q_are_left_unwritten():
    c = Call("qwen25_7b", [100, 20], [9, 4], seed=66, max_q=5, behind=0)
    got = c.run()
    assert (got[5:9] == 3).all()
    for i, (a, n) in enumerate(((0, 5), (9, 4))):
        k, v = values(c.pool.rec, c.table[i], int(c.past[i]) + n)
        ref, tol = attention(c.q[a:a + n], k, v, int(c.past[i]) + 1, c.nova.group)
        assert_within(got[a:a + n], ref, tol, f"session {i}")


@pytest.mark.parametrize("n_keys", [[33, 500, 1], [1], [767, 768]])
def test_short_tables(n_keys):
    """tables of up to 48 pages take one launch without a join"""
    d = Call("qwen25_7b", n_keys, seed=64)
    d.table = np.ascontiguousarray(d.table[:, :48])
    d.upload()
    d.run()
    d.check("short")


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("stride", [40, 41, 64, 65, 96, 97])
def test_tables_at_the_one_launch_limits(model, stride):
    """few sessions and enough for longer tables, with some of no keys and no rows"""
    most = stride * KB
    lengths = [most, 0, most - 1, 1, 700 % most]
    d = Call(model, lengths, seed=75)
    c = Call(model, [most - 4, 9, 0, 500, most - 20], [3, 0, 1, 2, 0], seed=76, behind=2)
    many = 64 // d.nova.nkv
    e = Call(model, (lengths * many)[:many], seed=77)
    f = Call(model, [most - 4] + [40 + i for i in range(many - 1)], [3] + [i % 3 for i in range(many - 1)], seed=78, behind=2)
    for x in (d, c, e, f):
        assert x.table.shape[1] >= stride
        x.table = np.ascontiguousarray(x.table[:, :stride])
        x.upload()
        x.run()
        x.check(f"{stride} pages")


def test_keys_behind_the_table_are_left_out():
    d = Call("qwen25_1p5b", [64, 40], seed=65, poison=False)
    d.table = np.ascontiguousarray(d.table[:, :3])           # 48 tokens each
    d.upload()
    d.run()
    d.keys = np.array([48, 40])
    d.past = np.array([48, 40])
    d.check("cut")


def test_zero_rows():
    """a query of zeros weighs all keys alike; keys and values of zeros count in the sum; sessions of zeros only"""
    d = Call("qwen25_7b", [200, 130, 40], seed=6, poison=False)
    kc, ke, vc, ve = d.parts()
    for t in (d.table[0, :5], d.table[1, 2:3], d.table[2, :3]):
        kc[t], ke[t], vc[t], ve[t] = 0, 0, 0, 0
    d.set_parts((kc, ke, vc, ve))
    d.q[1] = 0
    d.upload()
    got = d.run()
    d.check("zeros")
    assert not got[2].any()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_non_finite_query_stays_in_its_row_and_head(bad):
    for x, row, head in ((Call("qwen25_7b", [70, 900], seed=61), 1, 9),
                         (Call("qwen25_7b", [30, 500], [70, 3], seed=62, behind=0), 40, 27),
                         (Call("qwen25_7b", [30, 500], [2, 3], seed=62, behind=0), 4, 27)):
        x.q[row, head, 77] = bad
        x.upload()
        wrong = ~np.isfinite(x.run())
        assert wrong[row, head].all()
        wrong[row, head] = False
        assert not wrong.any()


def test_non_finite_rows_of_a_decode():
    """A key or value row stored from an infinity or NaN makes every head of its kv head that sees it
    NaN, and no other."""
    d = Call("qwen25_7b", [100, 100, 100], seed=8)
    kc, ke, vc, ve = d.parts()
    ke[d.table[0, 2], 1, 4] = NAN                            # key 36 of session 0, kv head 1
    ve[d.table[1, 6], 3, 3] = NAN                            # the last key of session 1, kv head 3
    d.set_parts((kc, ke, vc, ve))
    bad = np.isnan(d.run()).reshape(3, d.nova.nkv, -1)
    assert bad[0, 1].all() and bad[1, 3].all()
    bad[0, 1] = bad[1, 3] = False
    assert not bad.any()


@pytest.mark.parametrize("rows", [4, 90])
def test_non_finite_rows_are_seen_by_later_rows_only(rows):
    """and the rows before them are what they are without"""
    c = Call("qwen25_7b", [30], [rows], seed=25, behind=0)
    kc, ke, vc, ve = c.parts()
    a, b = 30 + rows // 2, 30 + rows // 2 + 1
    ke[c.table[0, a // KB], 2, a % KB] = NAN                 # kv head 2: rows from rows / 2 on see it
    ve[c.table[0, b // KB], 0, b % KB] = NAN                 # kv head 0: one row later
    c.set_parts((kc, ke, vc, ve))
    got = c.run()
    bad = np.isnan(got).reshape(rows, c.nova.nkv, -1)
    assert bad[rows // 2:, 2].all() and bad[rows // 2 + 1:, 0].all()
    bad[rows // 2:, 2] = bad[rows // 2 + 1:, 0] = False
    assert not bad.any()
    k, v = values(c.pool.rec, c.table[0], 30 + rows)
    ref, tol = attention(c.q[:rows // 2], k, v, 31, c.nova.group)
    assert_within(got[:rows // 2], ref, tol, "rows before")


# rows of a session: 1 and 4 take the kernels of few columns, 70 that of many
FORMS = [(1, True), (1, False), (4, False), (70, False)]


def _call(keys, rows, decode, seed, **kw):
    if decode:
        return Call("qwen25_1p5b", keys, seed=seed, poison=False, **kw)
    return Call("qwen25_1p5b", [n - rows for n in keys], [rows] * len(keys), seed=seed, behind=0, poison=False, **kw)


def _towards(c, parts, sess, key, score):
    """all of the session's queries share a direction, and this key is a multiple of it with about `score`"""
    u = np.where(np.arange(HD) % 3 == 0, 1.0, -1.0).astype(np.float32)
    a, b = c.off[sess], c.off[sess + 1]
    c.q[a:b] += 2 * u - (c.q[a:b] @ u)[..., None] * u / HD
    at = c.table[sess, key // KB], slice(None), key % KB
    code, byte = quantise(u * np.float32(score * np.sqrt(HD) / (2 * HD)))
    parts[0][at], parts[1][at] = code, byte
    return at


@pytest.mark.parametrize("power", [14, 30, 60, 100])
@pytest.mark.parametrize("rows,decode", FORMS)
def test_large_value_of_small_weight(rows, decode, power):
    """a key that all rows see, its value 2^power times the others', its weight 2^-90 or so"""
    c = _call([900, 130], rows, decode, seed=2, scale=0.5)
    p = c.parts()
    for sess, key in ((0, 333), (1, 3)):
        p[3][_towards(c, p, sess, key, -60.0)] += power
    c.set_parts(p)
    c.upload()
    c.run()
    c.check()


@pytest.mark.parametrize("score", [8.0, 40.0])
@pytest.mark.parametrize("power", [-127, -60, -20])
@pytest.mark.parametrize("rows,decode", FORMS)
def test_small_value_of_large_weight(rows, decode, power, score):
    """a key that takes nearly all of the weight, its value zero or small: the others' count"""
    c = _call([900, 130], rows, decode, seed=3, scale=0.5)
    p = c.parts()
    for sess, key in ((0, 333), (1, 3)):
        at = _towards(c, p, sess, key, score)
        p[3][at] = np.maximum(p[3][at].astype(int) + power, 0)
    c.set_parts(p)
    c.upload()
    c.run()
    c.check()


@pytest.mark.parametrize("power", [20, 60, 100])
@pytest.mark.parametrize("rows", [4, 70])
def test_later_tokens_do_not_touch_earlier_rows(rows, power):
    c = _call([230, 34 + rows], rows, False, seed=1)
    p = c.parts()
    for sess in (0, 1):
        key = int(c.past[sess]) + rows // 2
        p[3][c.table[sess, key // KB], :, key % KB] += power
    c.set_parts(p)
    c.run()
    c.check()


@pytest.mark.parametrize("keys", [40, 3000])
@pytest.mark.parametrize("rows,decode", FORMS)
@pytest.mark.parametrize("byte", [27, 100, 200, 223])
def test_values_of_any_power(rows, decode, keys, byte):
    """all values of a size, under weights that are nearly equal"""
    c = _call([max(keys, rows)], rows, decode, seed=4, scale=0.01)
    p = c.parts()
    p[3] = np.where(p[3] > 0, p[3].astype(int) - p[3].max() + byte, 0).clip(0, 252).astype(np.uint8)
    c.set_parts(p)
    c.run()
    c.check()


@pytest.mark.parametrize("power", [-90, 90])
@pytest.mark.parametrize("rows,decode", FORMS)
def test_large_keys_and_small_queries(rows, decode, power):
    """keys 2^power times, queries 2^-power times as large: the same scores"""
    c = _call([700], rows, decode, seed=5, scale=0.5)
    p = c.parts()
    p[1] = (p[1].astype(int) + power).astype(np.uint8)
    c.set_parts(p)
    c.q *= np.float32(2.0 ** -power)
    c.upload()
    c.run()
    c.check()


@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("keys", [1, 90, 2000])
@pytest.mark.parametrize("rows,decode", FORMS)
def test_scores_of_any_size(rows, decode, keys, sign):
    """Scores of 2^90 to 2^113, key j's 1, 1.5, 1, 1.5 .. and twice that every eighth key: the largest
    (or the first) take everything, and a row's result lies between their values."""
    keys = max(keys, rows)
    c = _call([keys], rows, decode, seed=6)
    p = c.parts()
    u = np.where(np.arange(HD) % 3 == 0, 0, 8).astype(np.uint8)
    for j in range(keys):
        at = c.table[0, j // KB], slice(None), j % KB
        p[0][at] = u | (2 + j % 2)                           # 1 or 1.5
        p[1][at] = 127 + 45 + min(j, 80) // 4
    c.set_parts(p)
    c.q[:] = np.float32(sign * 2.0 ** 40) * np.where(u > 0, -1, 1)
    c.upload()
    got = c.run()
    k, v = values(c.pool.rec, c.table[0], keys)
    for r in range(rows):
        m = keys if decode else int(c.past[0]) + r + 1
        s = c.q[r, 0].astype(np.float64) @ k[:m, 0].T
        best = np.flatnonzero(s == s.max())                  # alike: the same codes and powers
        # A score of 2^113 in fp32, added up in five steps of 2^-23 of it, is off by up to 2^93, and less
        # the reference it is a number of that size: of keys that are alike by their codes, in tiles
        # with another reference, any may take any part of the whole.  The others' scores are a
        # sixteenth and more below, 2^104: they take nothing.
        lo, hi = (np.repeat(f(v[best], axis=0), c.nova.group, 0) for f in (np.min, np.max))
        slack = 2.0 ** -20 * np.repeat(np.abs(v[best]).max(0), c.nova.group, 0)
        assert ((got[r] >= lo - slack) & (got[r] <= hi + slack)).all(), r


def test_the_same_every_time():
    for c in (Call("qwen25_7b", [3000, 17, 900], seed=9), Call("qwen25_7b", [3000, 17], [200, 9], seed=9, behind=0)):
        first = c.run()
        for _ in range(3):
            assert np.array_equal(first, c.run())


@pytest.mark.parametrize("make", [
    lambda: Call("qwen25_7b", [2000, 40, 700], seed=31), lambda: Call("qwen25_7b", [900, 100], [5, 8], seed=32),
    lambda: Call("qwen25_7b", [300, 0], [120, 200], seed=33)], ids=["decode", "drafts", "chunk"])
def test_graph_replays(make):
    """A captured call replayed with eager work and other inputs between the replays: every replay gives
    the bits of the eager call."""
    c = make()
    n, live = c.nova, c.off[-1]
    s = n.dev_stream_create()
    c.launch(s)
    n.dev_stream_sync(s)
    want = c.result()
    n.dev_graph_begin(s)
    c.launch(s)
    graph = n.dev_graph_end(s)
    for _ in range(3):
        n.dev_zero(c.o.ptr, c.q.nbytes, s)
        n.dev_zero(c.ws.ptr, c.ws.nbytes, s)
        n.dev_graph_launch(graph, s)
        n.dev_stream_sync(s)
        assert np.array_equal(want[:live], c.result()[:live])
        c.launch(s)
        n.dev_stream_sync(s)
    c.q = (c.q[::-1] * 0.5).copy()
    n.dev_upload(c.dq.ptr, c.q.ctypes.data, c.q.nbytes)
    fresh = np.full(c.q.shape, 3, np.float32)
    n.dev_upload(c.o.ptr, fresh.ctypes.data, fresh.nbytes)
    n.dev_graph_launch(graph, s)
    n.dev_stream_sync(s)
    c.check("replay on new inputs")
    n.dev_graph_destroy(graph)
    n.dev_stream_destroy(s)


def test_two_calls_at_once():
    """calls on two streams with a workspace each"""
    a, b = Call("qwen25_7b", [4000, 300, 9], seed=41), Call("qwen25_7b", [2000, 5], [8, 3], seed=42)
    s1, s2 = a.nova.dev_stream_create(), a.nova.dev_stream_create()
    for _ in range(5):
        a.launch(s1)
        b.launch(s2)
    a.nova.dev_sync()
    a.check("decode beside a chunk")
    b.check("chunk beside a decode")
    a.nova.dev_stream_destroy(s1)
    a.nova.dev_stream_destroy(s2)


def test_workspace_is_enough():
    """nothing is written behind the workspace's size, whatever it held before"""
    for x in (Call("qwen25_1p5b", [5000, 3, 900], seed=67), Call("qwen25_14b", [3000, 0], [6, 3], seed=68),
              Call("qwen25_7b", [2000, 0], [50, 200], seed=69)):
        n, size = x.nova, x.ws.nbytes
        x.ws = n.upload(np.full(size + 65536, 0xff, np.uint8))               # NaN bits
        x.run()
        x.check("poisoned workspace")
        assert (n.download(x.ws, (65536,), np.uint8, size) == 0xff).all()


def test_beyond_32_bit_offsets():
    """the last layer and the last pages of a pool of 5 GB: append, decode, chunk"""
    import nova_amd
    nova = nova_amd.load("qwen25_7b")
    nb, layer, n = 21000, 27, 40
    rng = np.random.default_rng(63)
    dev = nova.alloc((layer + 1) * nb * nova.kv_q4_page_bytes())
    k, v = (rng.standard_normal((n, nova.nkv, HD)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((n, nova.nh, HD)).astype(np.float32)
    table, zero, keys = np.array([[nb - 1, 3, nb - 2]], np.int32), np.zeros(1, np.int32), np.array([n], np.int32)
    dt, dz, dn, dk, dv, dq = (nova.upload(x) for x in (table, zero, keys, k, v, q))
    nova.launch_kv_q4_store_batch(dev.ptr, dt.ptr, 3, dz.ptr, None, 1, n, layer, nb, dk.ptr, dv.ptr, None)
    o, o1 = nova.alloc(q.nbytes), nova.alloc(q[:1].nbytes)
    ws = nova.alloc(nova.attn_chunk_q4_workspace_bytes(1, n, n))
    nova.launch_attn_chunk_q4_batch(dq.ptr, dev.ptr, dt.ptr, 3, dz.ptr, None, 1, n, n, layer, nb, o.ptr, ws.ptr, None)
    ws1 = nova.alloc(nova.attn_decode_q4_workspace_bytes(1))
    nova.launch_attn_decode_q4_batch(dq.ptr, dev.ptr, dt.ptr, 3, dn.ptr, 1, layer, nb, o1.ptr, ws1.ptr, None)
    nova.dev_sync()
    kk, vv = (decode(*quantise(x)) for x in (k, v))
    ref, tol = attention(q, kk, vv, 1, nova.group)
    assert_within(o.numpy(q.shape, np.float32), ref, tol, "chunk")
    ref, tol = attention(q[:1], kk, vv, n, nova.group)
    assert_within(o1.numpy(q[:1].shape, np.float32), ref, tol, "decode")


@pytest.mark.parametrize("rows,decode", FORMS)
@pytest.mark.parametrize("spread", [7, 8, 30])
def test_value_powers_within_a_tile(rows, decode, spread):
    """powers that lie a window apart, one more, and far apart, in some tiles or all"""
    c = _call([700, 333], rows, decode, seed=11, scale=0.5)
    p = c.parts()
    rng = np.random.default_rng(spread)
    p[3] = (120 + rng.integers(0, spread + 1, p[3].shape)).astype(np.uint8)
    some = c.table[0, 8:20]
    p[3][some] = 126
    c.set_parts(p)
    c.run()
    c.check()


@pytest.mark.parametrize("rows,decode", FORMS)
@pytest.mark.parametrize("powers", [(-40, 0, 40), (-100, -20, -100, 13, -14, 90), (14, 10, 14, 13, 12, -23, -24)])
def test_value_powers_change_between_tiles(rows, decode, powers):
    """every two tiles of another size: in fp16's reach and past it, up and down"""
    c = _call([64 * 2 * len(powers) * 3 + 5], rows, decode, seed=12, scale=0.02)
    p = c.parts()
    n = c.table.shape[1] - 3
    for i in range(n):
        p[3][c.table[0, i]] = 127 + powers[i // 8 % len(powers)] - (np.arange(4) % 2)
    c.set_parts(p)
    c.run()
    c.check()


@pytest.mark.parametrize("rows,decode", FORMS)
@pytest.mark.parametrize("size", [3.0, 20.0, 80.0, 200.0])
@pytest.mark.parametrize("first", ["high", "low", "by turns"])
def test_scores_rise_and_fall_between_tiles(rows, decode, size, first):
    """tiles whose scores lie `size` apart, so that the reference goes up and down, and values of the
    tiles with the high scores that are zero in half of the dims: the other tiles' count there"""
    c = _call([64 * 14 + 9], rows, decode, seed=13, scale=0.3)
    p = c.parts()
    u = np.where(np.arange(HD) % 3 == 0, 1.0, -1.0).astype(np.float32)
    c.q += 2 * u - (c.q @ u)[..., None] * u / HD
    rng = np.random.default_rng(3)
    for i in range(c.table.shape[1] - 3):
        tile = i // 4
        up = {"high": tile < 3, "low": tile >= 11, "by turns": tile % 3 == 0}[first]
        x = rng.standard_normal((c.nova.nkv, KB, HD)).astype(np.float32) * 0.1
        if up:
            x += u * np.float32(size * np.sqrt(HD) / (2 * HD))
            p[2][c.table[0, i], :, :, ::2] = 0
        p[0][c.table[0, i]], p[1][c.table[0, i]] = quantise(x)
    c.set_parts(p)
    c.upload()
    c.run()
    c.check()


@pytest.mark.parametrize("rows,decode", FORMS)
def test_zero_and_nan_blocks_in_some_tiles(rows, decode):
    """blocks of zeros among others, a NaN row that is hidden from half of the rows, huge values after it"""
    c = _call([600 + rows], rows, decode, seed=14, scale=0.5)
    p = c.parts()
    p[3][c.table[0, 5], :, 3, 1], p[2][c.table[0, 5], :, 3, 32:64] = 0, 0
    p[3][c.table[0, 9:11]], p[2][c.table[0, 9:11]] = 0, 0
    p[3][c.table[0, 20], :, 2] = 200
    hidden = 600 + rows // 2
    if rows > 1:
        p[3][c.table[0, hidden // KB], 1, hidden % KB] = NAN
    c.set_parts(p)
    got = c.run()
    k, v = values(c.pool.rec, c.table[0], 600 + rows)
    ref, tol = attention(c.q[:rows], k, v, int(c.past[0]) + (0 if decode else 1), c.nova.group)
    if rows > 1:
        bad = np.isnan(got).reshape(rows, c.nova.nkv, -1)
        assert bad[rows // 2:, 1].all() and not bad[:, 0].any() and not bad[:rows // 2].any()
        got = np.where(np.isnan(got), ref, got)
    assert_within(got, ref, tol, "zeros")
