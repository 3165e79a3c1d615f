"""Attention over 8-bit pages against the formula in float64 over the values the
codes stand for, with the bound derived in q8ref.attention."""
import numpy as np
import pytest

from q8ref import HD, KB, Q8Pool, assert_within, attention, quantise, pack, unpack, values

pytestmark = pytest.mark.gpu
LAYER = 3
MODELS = ["qwen25_1p5b", "qwen25_7b", "qwen25_14b"]


def _nova(model):
    import nova_amd
    return nova_amd.load(model)


class Decode:
    """A batch of sessions with `n_keys` keys each, ready to be attended."""

    def __init__(self, model, n_keys, seed, scale=1.5, poison=True):
        self.nova = nova = _nova(model)
        self.n_keys = n_keys = np.asarray(n_keys, np.int32)
        self.pool = pool = Q8Pool(nova, int(((n_keys + KB - 1) // KB).sum()) + 2, LAYER, seed)
        self.table = pool.tables((n_keys + KB - 1) // KB)
        if poison:
            pool.poison_behind(self.table, n_keys)
        self.q = (pool.rng.standard_normal((len(n_keys), nova.nh, HD)) * scale).astype(np.float32)
        self.dt, self.dn, self.dq = (nova.upload(x) for x in (self.table, n_keys, self.q))
        self.o = nova.upload(np.full(self.q.shape, 3, np.float32))
        self.ws = nova.alloc(nova.attn_decode_q8_workspace_bytes(len(n_keys)))

    def launch(self, stream=None):
        self.nova.launch_attn_decode_q8_batch(self.dq.ptr, self.pool.dev.ptr, self.dt.ptr, self.table.shape[1],
                                              self.dn.ptr, len(self.n_keys), LAYER, self.pool.nb, self.o.ptr,
                                              self.ws.ptr, stream)

    def result(self):
        return self.o.numpy(self.q.shape, np.float32)

    def check(self, what):
        got, worst = self.result(), 0.0
        for i, n in enumerate(self.n_keys):
            k, v = values(self.pool.rec, self.table[i], int(n))
            ref, tol = attention(self.q[i:i + 1], k, v, int(n), self.nova.group)
            worst = max(worst, assert_within(got[i:i + 1], ref, tol, f"{what}, session {i} of {n} keys"))
        return worst


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
    print(f"[case] q8 decode {model} {name}", flush=True)
    d = Decode(model, n_keys, seed=len(name))
    d.launch()
    d.nova.dev_sync()
    print(f"  {d.check(f'{model} {name}'):.3f} of the bound")


@pytest.mark.parametrize("scale", [1e-6, 1.0, 30.0, 1e4])
def test_decode_query_sizes(scale):
    """from scores that are all alike to one key that takes everything"""
    d = Decode("qwen25_7b", [1, 100, 900], seed=5, scale=scale)
    d.launch()
    d.nova.dev_sync()
    d.check(f"scale {scale}")


def test_decode_zero_queries_and_rows():
    """a query of zeros weighs all keys alike; keys and values of zeros (scale 0)
    count in the sum; a batch of zeros only"""
    d = Decode("qwen25_7b", [200, 130, 40], seed=6)
    kc, ks, vc, vs = (np.array(x) for x in unpack(d.pool.rec))
    zero = np.zeros((d.pool.nb, d.nova.nkv, KB), bool)
    zero[d.table[0, :5]] = True                              # the first 80 keys of session 0
    zero[d.table[1, 2], :, 3:9] = True
    zero[d.table[2, :3]] = True                              # all of session 2
    kc[zero], ks[zero], vc[zero], vs[zero] = 0, 0, 0, 0
    d.pool.rec = pack(kc, ks, vc, vs)
    d.pool.push()
    d.q[1] = 0
    d.nova.dev_upload(d.dq.ptr, d.q.ctypes.data, d.q.nbytes)
    d.launch()
    d.nova.dev_sync()
    d.check("zeros")
    assert not d.result()[2].any()


@pytest.mark.parametrize("spread", [1e-3, 1e3])
def test_decode_value_scales_far_apart(spread):
    """values whose scales differ by far between tokens, the small ones with the
    large weights among them"""
    d = Decode("qwen25_1p5b", [333, 40], seed=7, poison=False)
    kc, ks, vc, vs = (np.array(x) for x in unpack(d.pool.rec))
    vs[:, :, ::3] *= spread
    vs[:, :, 1::5] *= spread * spread
    d.pool.rec = pack(kc, ks, vc, vs)
    d.pool.push()
    d.launch()
    d.nova.dev_sync()
    d.check(f"spread {spread}")


def test_decode_non_finite_rows():
    """A key or value row stored from an infinity or NaN makes every head of its
    kv head that sees it NaN, and no other."""
    d = Decode("qwen25_7b", [100, 100, 100], seed=8)
    kc, ks, vc, vs = (np.array(x) for x in unpack(d.pool.rec))
    ks[d.table[0, 2], 1, 4] = np.nan                         # key 36 of session 0, kv head 1
    vs[d.table[1, 6], 3, 3] = np.nan                         # the last key of session 1, kv head 3
    d.pool.rec = pack(kc, ks, vc, vs)
    d.pool.push()
    d.launch()
    d.nova.dev_sync()
    bad = np.isnan(d.result()).reshape(3, d.nova.nkv, -1)
    assert bad[0, 1].all() and bad[1, 3].all()
    bad[0, 1] = bad[1, 3] = False
    assert not bad.any()


def test_decode_is_the_same_every_time():
    d = Decode("qwen25_7b", [3000, 17, 900], seed=9)
    d.launch()
    d.nova.dev_sync()
    first = d.result()
    for _ in range(3):
        d.launch()
        d.nova.dev_sync()
        assert np.array_equal(first, d.result())


class Chunk:
    def __init__(self, model, past, count, seed, scale=1.5, max_q=None, behind=2, offsets=True):
        self.nova = nova = _nova(model)
        self.past, self.count = np.asarray(past, np.int32), np.asarray(count)
        keys = np.where(self.count > 0, self.past + self.count, 0)
        self.off = np.concatenate([[0], np.cumsum(self.count)]).astype(np.int32)
        self.n_rows = int(self.off[-1]) + behind
        self.max_q = int(self.count.max()) if max_q is None else max_q
        self.pool = pool = Q8Pool(nova, int(((keys + KB - 1) // KB).sum()) + 2, LAYER, seed)
        self.table = pool.tables((keys + KB - 1) // KB)
        pool.poison_behind(self.table, keys)
        self.q = (pool.rng.standard_normal((self.n_rows, nova.nh, HD)) * scale).astype(np.float32)
        self.dt, self.dp, self.doff, self.dq = (nova.upload(x) for x in (self.table, self.past, self.off, self.q))
        self.doff_ptr = self.doff.ptr if offsets else None
        self.o = nova.upload(np.full(self.q.shape, 3, np.float32))
        self.ws = nova.alloc(nova.attn_chunk_q8_workspace_bytes(len(past), self.n_rows, self.max_q))

    def launch(self, stream=None):
        self.nova.launch_attn_chunk_q8_batch(self.dq.ptr, self.pool.dev.ptr, self.dt.ptr, self.table.shape[1],
                                             self.dp.ptr, self.doff_ptr, len(self.past), self.n_rows, self.max_q, LAYER,
                                             self.pool.nb, self.o.ptr, self.ws.ptr, stream)

    def result(self):
        return self.o.numpy(self.q.shape, np.float32)

    def check(self, what):
        got, worst = self.result(), 0.0
        for i, n in enumerate(self.count):
            a, b = int(self.off[i]), int(self.off[i + 1])
            if n == 0:
                continue
            k, v = values(self.pool.rec, self.table[i], int(self.past[i] + n))
            ref, tol = attention(self.q[a:b], k, v, int(self.past[i]) + 1, self.nova.group)
            worst = max(worst, assert_within(got[a:b], ref, tol, f"{what}, session {i}: {n} rows behind {self.past[i]}"))
        assert (got[self.off[-1]:] == 3).all(), f"{what}: rows behind the last sequence were written"
        return worst


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
    print(f"[case] q8 chunk {model} {name}", flush=True)
    c = Chunk(model, past, count, seed=len(name))
    c.launch()
    c.nova.dev_sync()
    print(f"  {c.check(f'{model} {name}'):.3f} of the bound")


def test_chunk_wide_batch():
    """enough rows to fill the chip"""
    c = Chunk("qwen25_7b", [0, 900, 333, 64, 1023, 500], [512, 300, 511, 256, 400, 513], seed=21)
    c.launch()
    c.nova.dev_sync()
    print(f"  {c.check('wide'):.3f} of the bound")


@pytest.mark.parametrize("scale", [1e-6, 30.0, 1e4])
def test_chunk_query_sizes(scale):
    c = Chunk("qwen25_7b", [50, 200], [40, 3], seed=22, scale=scale)
    c.launch()
    c.nova.dev_sync()
    c.check(f"scale {scale}")


@pytest.mark.parametrize("n", [1, 6, 50])
def test_chunk_without_offsets(n):
    c = Chunk("qwen25_14b", [0, 77, 15], [n] * 3, seed=23, behind=0, offsets=False)
    c.launch()
    c.nova.dev_sync()
    c.check("uniform")


def test_chunk_larger_max_q():
    """max_q is a bound: a larger one gives the same rows within the tolerance"""
    c = Chunk("qwen25_7b", [40, 900], [3, 5], seed=24, max_q=10, behind=2)
    c.launch()
    c.nova.dev_sync()
    c.check("max_q")


def test_chunk_non_finite_key_is_seen_by_later_rows_only():
    c = Chunk("qwen25_7b", [30], [90], seed=25, behind=0)
    kc, ks, vc, vs = (np.array(x) for x in unpack(c.pool.rec))
    ks[c.table[0, 4], 2, 6] = np.nan                         # key 70, kv head 2: rows from 40 on see it
    vs[c.table[0, 5], 0, 0] = np.nan                         # value 80, kv head 0: rows from 50 on
    c.pool.rec = pack(kc, ks, vc, vs)
    c.pool.push()
    c.launch()
    c.nova.dev_sync()
    bad = np.isnan(c.result()).reshape(90, c.nova.nkv, -1)
    assert bad[40:, 2].all() and bad[50:, 0].all()
    bad[40:, 2] = bad[50:, 0] = False
    assert not bad.any()


def test_chunk_of_one_row_is_the_decode():
    """the two entry points agree on the same call within the bound"""
    n_keys = [64, 1, 777]
    d = Decode("qwen25_7b", n_keys, seed=26)
    d.launch()
    past = d.nova.upload(d.n_keys - 1)
    o = d.nova.alloc(d.q.nbytes)
    ws = d.nova.alloc(d.nova.attn_chunk_q8_workspace_bytes(3, 3, 1))
    d.nova.launch_attn_chunk_q8_batch(d.dq.ptr, d.pool.dev.ptr, d.dt.ptr, d.table.shape[1], past.ptr, None, 3, 3, 1, LAYER,
                                      d.pool.nb, o.ptr, ws.ptr, None)
    d.nova.dev_sync()
    d.check("decode")
    d.o = o
    d.check("chunk")


@pytest.mark.parametrize("make", [
    lambda: Decode("qwen25_7b", [2000, 40, 700], seed=31), lambda: Chunk("qwen25_7b", [900, 100], [5, 8], seed=32),
    lambda: Chunk("qwen25_7b", [300, 0], [120, 200], seed=33)], ids=["decode", "drafts", "chunk"])
def test_graph_replays(make):
    """A captured call replayed with eager work and other inputs between the
    replays: every replay gives the bits of the eager call."""
    c = make()
    n = c.nova
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
        assert np.array_equal(want[:c.off[-1]] if hasattr(c, "off") else want,
                              c.result()[:c.off[-1]] if hasattr(c, "off") else c.result())
        c.launch(s)                                          # eager work on the same workspace
        n.dev_stream_sync(s)
    # new inputs in the same buffers
    q2 = (c.q[::-1] * 0.5).copy()
    n.dev_upload(c.dq.ptr, q2.ctypes.data, q2.nbytes)
    n.dev_graph_launch(graph, s)
    n.dev_stream_sync(s)
    c.q = q2
    got = c.result()
    if hasattr(c, "off"):
        got[c.off[-1]:] = 3                                  # cleared above, not part of the call
        n.dev_upload(c.o.ptr, got.ctypes.data, got.nbytes)
    c.check("replay on new inputs")
    n.dev_graph_destroy(graph)
    n.dev_stream_destroy(s)


def test_two_calls_at_once():
    """calls on two streams with a workspace each"""
    a = Decode("qwen25_7b", [4000, 300, 9], seed=41)
    b = Chunk("qwen25_7b", [2000, 5], [8, 3], seed=42)
    s1, s2 = a.nova.dev_stream_create(), a.nova.dev_stream_create()
    for _ in range(5):
        a.launch(s1)
        b.launch(s2)
    a.nova.dev_sync()
    a.check("decode beside a chunk")
    b.check("chunk beside a decode")
    a.nova.dev_stream_destroy(s1)
    a.nova.dev_stream_destroy(s2)


def test_sessions_on_8_bit_pages():
    """The operators as a program uses them: the session manager over 8-bit pages;
    a prompt through RoPE + append and chunk attention, a fork that shares its
    prefix, copy-on-write, drafted tokens for both, then single tokens."""
    nova = _nova("qwen25_7b")
    rng = np.random.default_rng(50)
    h = nova.nova_paged_new_q8(3, 160)
    assert nova.nova_paged_pool_k(h) is None and nova.nova_paged_pool_v(h) is None
    pool, stream, nb = nova.nova_paged_pool_q8(h), nova.nova_paged_stream(h), nova.nova_paged_nb(h)
    a, b = nova.nova_paged_create_session(h, 1), nova.nova_paged_create_session(h, 1)
    stride = nova.nova_kvpool_nblocks(nova.nova_paged_pool(h))
    rec0 = nova.download(pool, (nova.n_layers, nb, nova.nkv, 4224), np.uint8)
    own = nova.download(nova.nova_paged_tables(h), (3, stride), np.int32)
    assert not rec0[:, own[[a, b]].ravel()].any()            # creation cleared both sessions' pages
    cs, sn = nova.alloc(160 * 64 * 4), nova.alloc(160 * 64 * 4)
    nova.launch_rope_table_rows(cs.ptr, sn.ptr, 160, stream)
    hist = {a: [], b: []}                                    # rotated k and v of every token of a session
    table_dev = nova.nova_paged_tables(h)

    def step(past, count, name):
        """RoPE + append + attention for sessions a and b (rows of the table array)"""
        n = sum(count)
        off = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
        q = rng.standard_normal((n, nova.nh, HD)).astype(np.float32)
        k = rng.standard_normal((n, nova.nkv, HD)).astype(np.float32)
        v = rng.standard_normal((n, nova.nkv, HD)).astype(np.float32)
        dp, doff, dq, dk, dv = (nova.upload(x) for x in (np.array(past, np.int32), off, q, k, v))
        o = nova.alloc(q.nbytes)
        nova.launch_rope_kv_q8_store_batch(dq.ptr, dk.ptr, dv.ptr, cs.ptr, sn.ptr, pool, table_dev, stride, dp.ptr,
                                           doff.ptr, 2, n, LAYER, nb, stream)
        if max(count) == 1 and min(count) == 1:
            keys = nova.upload((np.array(past) + 1).astype(np.int32))
            ws = nova.alloc(nova.attn_decode_q8_workspace_bytes(2))
            nova.launch_attn_decode_q8_batch(dq.ptr, pool, table_dev, stride, keys.ptr, 2, LAYER, nb, o.ptr, ws.ptr, stream)
        else:
            ws = nova.alloc(nova.attn_chunk_q8_workspace_bytes(2, n, max(count)))
            nova.launch_attn_chunk_q8_batch(dq.ptr, pool, table_dev, stride, dp.ptr, doff.ptr, 2, n, max(count), LAYER, nb,
                                            o.ptr, ws.ptr, stream)
        nova.dev_stream_sync(stream)
        rq = dq.numpy(q.shape, np.float32)                   # rotated in place
        # the rotated k, in float32 with every product rounded, as the launch defines it
        c = nova.download(cs, (160, 64), np.float32)
        s = nova.download(sn, (160, 64), np.float32)
        got = o.numpy(q.shape, np.float32)
        for i, sess in enumerate((a, b)):
            for r in range(off[i], off[i + 1]):
                pos = past[i] + r - off[i]
                x0, x1 = k[r, :, :64], k[r, :, 64:]
                rk = np.concatenate([x0 * c[pos] - x1 * s[pos], x0 * s[pos] + x1 * c[pos]], -1)
                hist[sess].append((rk, v[r]))
            if count[i]:
                ks, vs = (np.stack([t[j] for t in hist[sess]]) for j in (0, 1))
                kk, vv = (cc.astype(np.float64) * ss[..., None] for cc, ss in map(quantise, (ks, vs)))
                ref, tol = attention(rq[off[i]:off[i + 1]], kk, vv, past[i] + 1, nova.group)
                assert_within(got[off[i]:off[i + 1]], ref, tol, f"{name}, session {i}")

    step([0, 0], [40, 0], "prompt")
    nova.nova_paged_attach_prefix(h, b, a, 40)
    hist[b] = list(hist[a])
    before = nova.download(pool, (nova.n_layers, nb, nova.nkv, 4224), np.uint8)
    shared = nova.download(table_dev, (3, stride), np.int32)[a, 2]
    # b writes behind the shared tokens 32 .. 39 first: its page is copied
    nova.nova_paged_session_cow(h, b, 40, 5, stream)
    nova.nova_paged_session_cow(h, a, 40, 3, stream)
    nova.dev_stream_sync(stream)
    after = nova.download(table_dev, (3, stride), np.int32)
    assert after[b, 2] != shared and after[a, 2] == shared
    assert np.array_equal(nova.download(pool, before.shape, np.uint8)[:, after[b, 2]], before[:, shared])
    step([40, 40], [3, 5], "drafts")
    step([43, 45], [1, 1], "token")
    step([44, 46], [60, 2], "chunk and draft")
    step([104, 48], [1, 1], "token")
    nova.nova_paged_delete(h)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_non_finite_query_stays_in_its_row_and_head(bad):
    d = Decode("qwen25_7b", [70, 900], seed=61)
    c = Chunk("qwen25_7b", [30, 500], [70, 3], seed=62, behind=0)
    for x, row, head in ((d, 1, 9), (c, 40, 27)):
        x.q[row, head, 77] = bad
        x.nova.dev_upload(x.dq.ptr, x.q.ctypes.data, x.q.nbytes)
        x.launch()
        x.nova.dev_sync()
        wrong = ~np.isfinite(x.result())
        assert wrong[row, head].all()
        wrong[row, head] = False
        assert not wrong.any()


def test_attention_beyond_32_bit_offsets():
    """the last layer and the last pages of a pool of 5 GB: append, decode, chunk"""
    nova = _nova("qwen25_7b")
    nb, layer, n = 11000, 27, 40
    rng = np.random.default_rng(63)
    dev = nova.alloc((layer + 1) * nb * nova.kv_q8_page_bytes())
    k, v = (rng.standard_normal((n, nova.nkv, HD)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((n, nova.nh, HD)).astype(np.float32)
    table, zero, keys = np.array([[nb - 1, 3, nb - 2]], np.int32), np.zeros(1, np.int32), np.array([n], np.int32)
    dt, dz, dn, dk, dv, dq = (nova.upload(x) for x in (table, zero, keys, k, v, q))
    nova.launch_kv_q8_store_batch(dev.ptr, dt.ptr, 3, dz.ptr, None, 1, n, layer, nb, dk.ptr, dv.ptr, None)
    o, o1 = nova.alloc(q.nbytes), nova.alloc(q[:1].nbytes)
    ws = nova.alloc(nova.attn_chunk_q8_workspace_bytes(1, n, n))
    nova.launch_attn_chunk_q8_batch(dq.ptr, dev.ptr, dt.ptr, 3, dz.ptr, None, 1, n, n, layer, nb, o.ptr, ws.ptr, None)
    ws1 = nova.alloc(nova.attn_decode_q8_workspace_bytes(1))
    nova.launch_attn_decode_q8_batch(dq.ptr, dev.ptr, dt.ptr, 3, dn.ptr, 1, layer, nb, o1.ptr, ws1.ptr, None)
    nova.dev_sync()
    kk, vv = (c.astype(np.float64) * s[..., None] for c, s in map(quantise, (k, v)))
    ref, tol = attention(q, kk, vv, 1, nova.group)
    assert_within(o.numpy(q.shape, np.float32), ref, tol, "chunk")
    ref, tol = attention(q[:1], kk, vv, n, nova.group)
    assert_within(o1.numpy(q[:1].shape, np.float32), ref, tol, "decode")


@pytest.mark.parametrize("n_keys", [[33, 500, 1], [1], [767, 768]])
def test_short_tables(n_keys):
    """tables of up to 48 pages take one launch without a join"""
    d = Decode("qwen25_7b", n_keys, seed=64)
    assert d.table.shape[1] <= 51
    d.table = np.ascontiguousarray(d.table[:, :48])
    d.dt = d.nova.upload(d.table)
    d.launch()
    d.nova.dev_sync()
    d.check("short")


def test_keys_behind_the_table_are_left_out():
    """a session said to hold more keys than its table has entries for"""
    d = Decode("qwen25_1p5b", [64, 40], seed=65)
    d.table = np.ascontiguousarray(d.table[:, :3])           # 48 tokens each
    d.dt = d.nova.upload(d.table)
    d.n_keys = np.array([48, 40], np.int32)                  # what is left of [64, 40]
    d.launch()
    d.nova.dev_sync()
    d.check("cut")


def test_rows_behind_max_q_are_left_unwritten():
    c = Chunk("qwen25_7b", [100, 20], [9, 4], seed=66, max_q=5, behind=0)
    c.launch()
    c.nova.dev_sync()
    got = c.result()
    assert (got[5:9] == 3).all()
    for i, (a, n) in enumerate(((0, 5), (9, 4))):
        # the session's keys end with its last row that counts
        k, v = values(c.pool.rec, c.table[i], int(c.past[i]) + n)
        ref, tol = attention(c.q[a:a + n], k, v, int(c.past[i]) + 1, c.nova.group)
        assert_within(got[a:a + n], ref, tol, f"session {i}")


def test_workspace_is_enough():
    """nothing is written behind the workspace's size, whatever it held before"""
    for x in (Decode("qwen25_1p5b", [5000, 3, 900], seed=67), Chunk("qwen25_14b", [3000, 0], [6, 3], seed=68),
              Chunk("qwen25_7b", [2000, 0], [50, 200], seed=69)):
        n = x.nova
        size = x.ws.nbytes
        guard = n.upload(np.full(size + 65536, 0xff, np.uint8))              # NaN bits
        x.ws = guard
        x.launch()
        n.dev_sync()
        x.check("poisoned workspace")
        assert (n.download(guard, (65536,), np.uint8, size) == 0xff).all()


@pytest.mark.parametrize("model,past,count", [
    ("qwen25_7b", [30000], [8]),                             # one group in as many pieces as there are stretches
    ("qwen25_1p5b", [20000], [9]),
    ("qwen25_14b", [9000, 9000, 70], [12, 7, 9]),
    ("qwen25_7b", [12000] + [40] * 12, [5] + [6] * 12),      # one long, many short
    ("qwen25_7b", [5000, 2500, 1200, 600, 300], [30, 9, 20, 6, 40]),
], ids=["one", "one small", "two of three", "one of many", "halves"])
def test_groups_in_many_pieces(model, past, count):
    """the joining launch gives a group's columns one to eight teams, by its pieces"""
    c = Chunk(model, past, count, seed=60 + len(past))
    c.launch()
    c.nova.dev_sync()
    print(f"  {c.check(f'{model} pieces'):.3f} of the bound")


@pytest.mark.parametrize("model", MODELS)
def test_many_tiny_sessions(model):
    """more groups than tiles: a workgroup has few of them, or none"""
    rng = np.random.default_rng(61)
    count = [10] + rng.integers(0, 11, 299).tolist()
    c = Chunk(model, rng.integers(0, 4, 300).tolist(), count, seed=62)
    c.launch()
    c.nova.dev_sync()
    print(f"  {c.check(f'{model} tiny'):.3f} of the bound")
