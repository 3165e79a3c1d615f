"""Attention over 8-bit pages whose rows have far apart scales: a row's result depends
on the keys it sees, each by its weight, whatever stands beside them."""
import numpy as np
import pytest

from q8ref import HD, KB, Q8Pool, attention_by_row, pack, unpack, values

pytestmark = pytest.mark.gpu
LAYER = 2
MODEL = "qwen25_1p5b"


class Call:
    """A chunk of `count` rows per session behind `past` keys (decode: the last key's
    query), over pages whose codes and scales a test has changed."""

    def __init__(self, past, count, seed, scale=0.5, decode=False):
        import nova_amd
        self.nova = nova = nova_amd.load(MODEL)
        self.decode = decode
        self.past, self.count = np.asarray(past, np.int32), np.asarray(count)
        self.keys = self.past + self.count
        self.off = np.concatenate([[0], np.cumsum(self.count)]).astype(np.int32)
        self.n = int(self.off[-1])
        pages = (self.keys + KB - 1) // KB
        self.pool = Q8Pool(nova, int(pages.sum()) + 1, LAYER, seed)
        self.table = self.pool.tables(pages)
        self.parts = [np.array(x) for x in unpack(self.pool.rec)]     # K codes, K scales, V codes, V scales
        self.q = (self.pool.rng.standard_normal((self.n, nova.nh, HD)) * scale).astype(np.float32)

    def at(self, sess, key):
        """index of a key's scales and codes: [page, all heads, token]"""
        return self.table[sess, key // KB], slice(None), key % KB

    def towards(self, sess, key, score):
        """all of the session's queries share a direction u, and this key is a multiple
        of it, so that its score is about `score` for each of them"""
        u = np.where(np.arange(HD) % 3 == 0, 1.0, -1.0)
        a, b = self.off[sess], self.off[sess + 1]
        self.q[a:b] += np.float32(2) * u.astype(np.float32) - (self.q[a:b] @ u.astype(np.float32))[..., None] * u.astype(np.float32) / HD
        self.parts[0][self.at(sess, key)] = np.where(score < 0, -127, 127) * u
        self.parts[1][self.at(sess, key)] = abs(score) * np.sqrt(HD) / (2 * HD * 127)

    def run(self):
        n, p = self.nova, self.pool
        p.rec = pack(*self.parts)
        p.push()
        lens = self.keys if self.decode else self.past
        dt, dn, doff, dq = (n.upload(np.ascontiguousarray(x)) for x in (self.table, lens.astype(np.int32), self.off, self.q))
        o = n.upload(np.full(self.q.shape, 3, np.float32))
        if self.decode:
            ws = n.alloc(n.attn_decode_q8_workspace_bytes(len(lens)))
            n.launch_attn_decode_q8_batch(dq.ptr, p.dev.ptr, dt.ptr, self.table.shape[1], dn.ptr, len(lens), LAYER, p.nb, o.ptr,
                                          ws.ptr, None)
        else:
            most = int(self.count.max())
            ws = n.alloc(n.attn_chunk_q8_workspace_bytes(len(lens), self.n, most))
            n.launch_attn_chunk_q8_batch(dq.ptr, p.dev.ptr, dt.ptr, self.table.shape[1], dn.ptr, doff.ptr, len(lens), self.n,
                                         most, LAYER, p.nb, o.ptr, ws.ptr, None)
        n.dev_sync()
        return o.numpy(self.q.shape, np.float32)

    def check(self):
        got = self.run()
        assert np.isfinite(got).all()
        worst = 0.0
        for i in range(len(self.past)):
            a, b = self.off[i], self.off[i + 1]
            m = int(self.keys[i])
            k, v = values(self.pool.rec, self.table[i], m)
            pos = np.arange(m)
            vs = self.parts[3][self.table[i][pos >> 4], :, pos & 15]
            ref, tol = attention_by_row(self.q[a:b], k, v, vs, int(self.past[i]) + 1, self.nova.group)
            ratio = np.abs(got[a:b].astype(np.float64) - ref) / np.maximum(tol, 1e-300)
            worst = max(worst, ratio.max())
            r = np.unravel_index(ratio.argmax(), ratio.shape)
            assert ratio.max() <= 1, f"session {i}, row, head, dim {r}: {got[a:b][r]} instead of {ref[r]}, {ratio.max():.3g} of the bound"
        print(f"  {worst:.3f} of the bound")


# rows of a session: 1 and 4 take the kernels of few columns, 70 that of many
FORMS = [(1, True), (1, False), (4, False), (70, False)]


@pytest.mark.parametrize("power", [14, 20, 26, 34, 40, 100])
@pytest.mark.parametrize("rows", [4, 70])
def test_later_tokens_do_not_touch_earlier_rows(rows, power):
    """a token whose value scale is 2^power times the others', hidden from the rows before it"""
    c = Call([30, 200], [rows, rows], seed=1)
    for sess in (0, 1):
        c.parts[3][c.at(sess, int(c.past[sess]) + rows // 2)] *= np.float32(2.0 ** power)
    c.check()


@pytest.mark.parametrize("power", [10, 20, 40, 100])
@pytest.mark.parametrize("rows,decode", FORMS)
def test_large_value_of_small_weight(rows, decode, power):
    """a key that all rows see, its value 2^power times the others', its weight 2^-144"""
    c = Call([900 - rows, 130], [rows, rows], seed=2, decode=decode)
    for sess, key in ((0, 333), (1, 3)):
        c.towards(sess, key, -100.0)
        c.parts[3][c.at(sess, key)] *= np.float32(2.0 ** power)
    c.check()


@pytest.mark.parametrize("score", [8.0, 40.0])
@pytest.mark.parametrize("size", [0.0, 2.0 ** -60, 2.0 ** -20])
@pytest.mark.parametrize("rows,decode", FORMS)
def test_small_value_of_large_weight(rows, decode, size, score):
    """a key that takes nearly all of the weight, its value zero or small: the others' count"""
    c = Call([900 - rows, 130], [rows, rows], seed=3, decode=decode)
    for sess, key in ((0, 333), (1, 3)):
        c.towards(sess, key, score)
        c.parts[3][c.at(sess, key)] *= np.float32(size)
    c.check()


@pytest.mark.parametrize("keys", [40, 3000])
@pytest.mark.parametrize("rows,decode", FORMS)
@pytest.mark.parametrize("top", [1e-34, 1e20, 1e33, 1e37])
def test_values_near_the_ends_of_fp32(rows, decode, keys, top):
    """all values of a size, under weights that are nearly equal"""
    c = Call([max(keys - rows, 0)], [rows], seed=4, scale=0.01, decode=decode)
    c.parts[3] *= np.float32(top / c.parts[3].max() / 127)
    c.check()


@pytest.mark.parametrize("key", [7, 2000])
@pytest.mark.parametrize("rows,decode", FORMS)
def test_one_value_near_the_end_of_fp32(rows, decode, key):
    """one row of 1e37 among ordinary ones, in the first tile or later"""
    c = Call([3000], [rows], seed=4, decode=decode)
    c.parts[3][c.at(0, key)] *= np.float32(1e37 / 127 / c.parts[3][c.at(0, key)].max())
    c.check()


@pytest.mark.parametrize("rows,decode", FORMS)
def test_subnormal_scales(rows, decode):
    """the quantiser makes none, but a page may hold them"""
    c = Call([700], [rows], seed=10, scale=0.01, decode=decode)
    c.parts[3] *= np.float32(1e-38 / c.parts[3].max() / 127)
    c.check()


@pytest.mark.parametrize("power", [-100, -60, 60])
@pytest.mark.parametrize("past,rows,decode", [(899, 1, True), (896, 4, False), (830, 70, False)])
def test_value_sizes_change_between_tiles(past, rows, decode, power):
    """the first two tiles' values 2^power times the others'"""
    c = Call([past], [rows], seed=8, decode=decode)
    c.parts[3][c.table[0, :8]] *= np.float32(2.0 ** power)
    c.check()


@pytest.mark.parametrize("rows", [4, 70])
def test_rows_that_see_small_values_only(rows):
    """beside rows that see others 2^60 times as large in the same tile"""
    c = Call([0], [rows], seed=9)
    for key in range(rows // 2):
        c.parts[3][c.at(0, key)] *= np.float32(2.0 ** -60)
    c.check()


@pytest.mark.parametrize("power", [-90, 100])
@pytest.mark.parametrize("rows,decode", FORMS)
def test_large_keys_and_small_queries(rows, decode, power):
    """keys 2^power times, queries 2^-power times as large: the same scores"""
    c = Call([700], [rows], seed=5, decode=decode)
    c.parts[1] *= np.float32(2.0 ** power)
    c.q *= np.float32(2.0 ** -power)
    c.check()


@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("keys", [1, 90, 2000])
@pytest.mark.parametrize("rows,decode", FORMS)
def test_scores_of_any_size(rows, decode, keys, sign):
    """Scores of 1e33 and more, all of one sign, key j's (1 + j / 64) times the first
    one's: the largest takes everything, and a row's result is its value."""
    c = Call([keys - 1], [rows], seed=6, decode=decode)
    n = c.past[0] + rows
    u = np.where(np.arange(HD) % 3 == 0, 1, -1)
    for j in range(n):
        c.parts[0][c.at(0, j)] = 100 * u
        c.parts[1][c.at(0, j)] = 1e14 * (1 + j / 64)
    c.q[:] = sign * 1e15 * u
    got = c.run()
    _, v = values(c.pool.rec, c.table[0], int(n))
    for r in range(rows):
        want = np.repeat(v[0 if sign < 0 else c.past[0] + r], c.nova.group, 0)
        # weight times scale: two fp16 terms, 2^-21, and three fp32 operations
        assert (np.abs(got[r] - want) <= 2.0 ** -20 * np.abs(want)).all(), (r, got[r][0][:4], want[0][:4])


@pytest.mark.parametrize("times", [30.0, 1e3, 1e6])
@pytest.mark.parametrize("rows,decode", FORMS)
def test_query_with_a_loud_channel(rows, decode, times):
    """The query is held to 2^-24 of its largest component, also where K has only zeros
    beside that one: the bound's term of max|q| sum|k|."""
    c = Call([700], [rows], seed=7, decode=decode)
    c.q[..., 77] *= np.float32(times)
    c.parts[0][..., 77] = 0
    c.check()
