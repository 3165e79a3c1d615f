"""The operators as a server uses them.  Step after step: the plan gives the sessions their pages
and rows, the rows' angles follow, and per layer the rows turn, are appended to 4-bit pages
and attend; eager, or captured once and replayed.  Then the session manager over 4-bit pages."""
import ctypes as C

import numpy as np
import pytest

from planref import Planner, pages
from q4ref import HD, KB, REC, assert_within, attention, decode, quantise
from test_q4_store_gpu import _nova, _turn

pytestmark = pytest.mark.gpu
LAYERS = (0, 1, 2)


def _freqs(nova, rot, scaling=0, factor=1.0):
    import nova_amd
    out, magnitude = np.zeros(rot // 2, np.float32), C.c_double()
    cfg = nova_amd.RopeCfg(rot, scaling, 1e6, factor, 0, 1, 32)
    assert nova.nova_rope_freqs(C.byref(cfg), out.ctypes.data_as(C.POINTER(C.c_float)), C.byref(magnitude)) == rot // 2
    return out, magnitude.value


class Server:
    """`n` sessions over a pool of nb pages; every step has room for max_rows rows, of which the plan
    fills what the sessions get."""

    def __init__(self, model, n, stride, nb, max_rows, max_q, rot=HD, beside=0, scaling=None, seed=0):
        self.nova = nova = _nova(model)
        self.rng = np.random.default_rng(seed)
        self.n, self.nb, self.max_rows, self.max_q, self.rot, self.beside = n, nb, max_rows, max_q, rot, beside
        free = self.rng.permutation(nb).astype(np.int32)
        self.plan = Planner(nova, np.full((n, stride), -3, np.int32), np.zeros(n, np.int32), free, nb, max_rows)
        freq, self.magnitude = _freqs(nova, rot, **(scaling or {}))
        self.freq = nova.upload(freq)
        self.cs, self.sn = (nova.alloc(max_rows * rot // 2 * 4) for _ in range(2))
        self.pool = nova.upload(np.full(len(LAYERS) * nb * nova.nkv * REC, 255, np.uint8))      # NaN in every slot
        self.q = [nova.alloc(max_rows * nova.nh * HD * 4) for _ in LAYERS]
        self.kv = [[nova.alloc(max_rows * nova.nkv * HD * 4) for _ in range(2)] for _ in LAYERS]
        self.o = [nova.alloc(max_rows * nova.nh * HD * 4) for _ in LAYERS]
        self.ws = nova.alloc(nova.attn_chunk_q4_workspace_bytes(n, max_rows, max_q))
        self.ws1 = nova.alloc(nova.attn_decode_q4_workspace_bytes(n))
        self.stream = nova.dev_stream_create()
        self.graphs = {}
        self.past_k = [[np.zeros((0, nova.nkv, HD), np.float32) for _ in range(n)] for _ in LAYERS]
        self.past_v = [[np.zeros((0, nova.nkv, HD), np.float32) for _ in range(n)] for _ in LAYERS]

    def close(self):
        for g in self.graphs.values():
            self.nova.dev_graph_destroy(g)
        self.nova.dev_stream_destroy(self.stream)

    def launch(self, single):
        """the step on the device; `single`: every session has one new token, row i is session i's"""
        n, p, s = self.nova, self.plan, self.stream
        p.launch(s)
        n.launch_rope_angles(p.pos.ptr, self.max_rows, self.freq.ptr, self.rot, self.magnitude, self.cs.ptr, self.sn.ptr, s)
        for i, layer in enumerate(LAYERS):
            q, (k, v), o = self.q[i].ptr, self.kv[i], self.o[i].ptr
            n.launch_rope_rows_kv_q4_store_batch(q, k.ptr, v.ptr, self.cs.ptr, self.sn.ptr, self.rot, self.beside, self.pool.ptr,
                                                 p.dt.ptr, p.stride, p.past.ptr, p.off.ptr, self.n, self.max_rows, layer,
                                                 self.nb, q, s)
            if single:
                n.launch_attn_decode_q4_batch(q, self.pool.ptr, p.dt.ptr, p.stride, p.dh.ptr, self.n, layer, self.nb, o,
                                              self.ws1.ptr, s)
            else:
                n.launch_attn_chunk_q4_batch(q, self.pool.ptr, p.dt.ptr, p.stride, p.past.ptr, p.off.ptr, self.n,
                                             self.max_rows, self.max_q, layer, self.nb, o, self.ws.ptr, s)

    def step(self, keep, new, single=False, graph=False, what=""):
        nova, p, rng = self.nova, self.plan, self.rng
        nq, nk = (self.max_rows, nova.nh, HD), (self.max_rows, nova.nkv, HD)
        host = [[(rng.standard_normal(x) * m).astype(np.float32) for x, m in ((nq, 1.5), (nk, 1), (nk, 1))] for _ in LAYERS]
        rest = np.full(nq, 3, np.float32)
        if keep is None:
            keep = p.have                                    # one captured graph serves both
        p.set(keep, new)

        def inputs():
            for i in range(len(LAYERS)):
                for dev, x in zip([self.q[i], *self.kv[i], self.o[i]], host[i] + [rest]):
                    nova.dev_upload(dev.ptr, x.ctypes.data, x.nbytes)
        inputs()
        if graph and single not in self.graphs:
            nova.dev_graph_begin(self.stream)
            self.launch(single)
            self.graphs[single] = nova.dev_graph_end(self.stream)
        if graph:
            nova.dev_graph_launch(self.graphs[single], self.stream)
        else:
            self.launch(single)
        nova.dev_stream_sync(self.stream)
        _, _, left, past, keys, off, pos, _ = p.check()
        rows = int(off[-1])
        cs, sn = (x.numpy((self.max_rows, self.rot // 2), np.float32) for x in (self.cs, self.sn))
        worst = 0.0
        for i in range(len(LAYERS)):
            q, k, v = host[i]
            tq, tk = (_turn(x[:rows], cs[:rows], sn[:rows], self.rot, self.beside) for x in (q, k))
            got_q, got = self.q[i].numpy(nq, np.float32), self.o[i].numpy(nq, np.float32)
            assert np.array_equal(got_q[:rows], tq) and np.array_equal(got_q[rows:], q[rows:]), what
            for j in range(self.n):
                a, b = off[j], off[j + 1]
                for hist, x in ((self.past_k, tk), (self.past_v, v)):
                    hist[i][j] = np.concatenate([hist[i][j][:past[j]], x[a:b]])
                    assert len(hist[i][j]) == keys[j]
                if a == b:
                    continue
                kk, vv = (decode(*quantise(h[i][j])) for h in (self.past_k, self.past_v))
                ref, tol = attention(tq[a:b], kk, vv, int(past[j]) + 1, nova.group)
                worst = max(worst, assert_within(got[a:b], ref, tol, f"{what}, layer {i}, session {j}"))
            assert single or (got[rows:] == 3).all()         # rows that nobody got
        print(f"  {what}: {rows} rows, {left} pages left, {worst:.3f} of the bound", flush=True)
        return rows

    def read_back(self):
        """every token of every session, all pages of it wherever they lie"""
        nova, p = self.nova, self.plan
        off = np.concatenate([[0], np.cumsum(p.have)]).astype(np.int32)
        total = int(off[-1])
        zero, doff = nova.upload(np.zeros(self.n, np.int32)), nova.upload(off)
        k, v = (nova.alloc(max(total, 1) * nova.nkv * HD * 4) for _ in range(2))
        for i, layer in enumerate(LAYERS):
            nova.launch_kv_q4_load_batch(self.pool.ptr, p.dt.ptr, p.stride, zero.ptr, doff.ptr, self.n, total, layer, self.nb,
                                         k.ptr, v.ptr, self.stream)
            nova.dev_stream_sync(self.stream)
            for dev, hist in ((k, self.past_k), (v, self.past_v)):
                want = np.concatenate([decode(*quantise(h)) for h in hist[i]])
                assert np.array_equal(dev.numpy((total, nova.nkv, HD), np.float32), want)


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "replayed"])
@pytest.mark.parametrize("model,rot,beside,scaling", [
    ("qwen25_1p5b", 64, 1, dict(scaling=1, factor=4.0)), ("qwen25_7b", 128, 0, None), ("qwen25_14b", 96, 0, dict(scaling=2, factor=2.0))])
def test_steps(model, rot, beside, scaling, graph):
    """prompts, single tokens, drafts of which some are taken back, sessions that end and others
    that take their pages, a step that does not fit"""
    s = Server(model, 5, 20, 60, 160, 80, rot, beside, scaling, seed=rot)
    print(f"[case] step {model} rot={rot} graph={graph}", flush=True)
    assert s.step(None, [70, 1, 0, 33, 5], graph=graph, what="prompts") == 109
    for t in range(2):
        s.step(None, [1, 1, 1, 1, 1], single=False, graph=graph, what="tokens")
    assert s.step(None, [4, 3, 8, 2, 6], graph=graph, what="drafts") == 23
    have = s.plan.have
    s.step(have - [2, 3, 0, 1, 6], [4, 1, 1, 5, 1], graph=graph, what="drafts taken back")
    s.step([0, have[1], 0, 17, have[4]], [0, 2, 40, 16, 0], graph=graph, what="one ends, one starts again")
    s.step(None, [80, 80, 1, 1, 1], graph=graph, what="full step")
    rows = s.step(None, [80, 79, 80, 1, 0], graph=graph, what="too much")       # the third finds no room, nor do those after it
    assert rows == 159
    s.read_back()
    s.close()


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "replayed"])
def test_single_tokens(graph):
    """row i is session i's: the decode"""
    s = Server("qwen25_7b", 6, 12, 40, 6, 6, seed=9)
    print(f"[case] single tokens graph={graph}", flush=True)
    for t in range(18):                                      # over a page's end
        s.step(None, [1] * 6, single=True, graph=graph, what=f"token {t}")
    keep = s.plan.have - [0, 18, 3, 17, 0, 1]
    s.step(keep, [1] * 6, single=True, graph=graph, what="some start again")
    s.read_back()
    s.close()


def test_many_sessions():
    """past what one launch of the plan holds, a batch read 64 at a time"""
    n = 300
    s = Server("qwen25_1p5b", n, 30, 900, 700, 40, seed=4)
    rng = np.random.default_rng(3)
    print("[case] many sessions", flush=True)
    new = rng.integers(0, 3, n)
    new[[0, 130, 299]] = 40
    s.step(None, new, graph=True, what="start")
    s.step(None, rng.integers(0, 3, n), graph=True, what="on")
    s.step(np.where(rng.random(n) < 0.3, 0, s.plan.have), rng.integers(0, 3, n), graph=True, what="some end")
    s.read_back()
    s.close()


def test_sessions_on_4_bit_pages():
    """The session manager over 4-bit pages; a prompt, a fork that shares its prefix,
    copy-on-write, drafted tokens for both, single tokens."""
    nova = _nova("qwen25_7b")
    rng = np.random.default_rng(50)
    h = nova.nova_paged_new_q4(3, 160)
    assert nova.nova_paged_pool_k(h) is None and nova.nova_paged_pool_v(h) is None and nova.nova_paged_pool_q8(h) is None
    pool, stream, nb = nova.nova_paged_pool_q4(h), nova.nova_paged_stream(h), nova.nova_paged_nb(h)
    a, b = nova.nova_paged_create_session(h, 1), nova.nova_paged_create_session(h, 1)
    stride = nova.nova_kvpool_nblocks(nova.nova_paged_pool(h))
    shape = (nova.n_layers, nb, nova.nkv, REC)
    tables = nova.nova_paged_tables(h)
    own = nova.download(tables, (3, stride), np.int32)
    assert not nova.download(pool, shape, np.uint8)[:, own[[a, b]].ravel()].any()       # creation cleared both sessions' pages
    freq, magnitude = _freqs(nova, HD)
    dfreq, layer = nova.upload(freq), 5
    hist = {a: ([], []), b: ([], [])}

    def step(past, count, name):
        n, off = sum(count), np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
        pos = np.concatenate([p + np.arange(c) for p, c in zip(past, count)]).astype(np.int32)
        q, k, v = (rng.standard_normal((n, m, HD)).astype(np.float32) for m in (nova.nh, nova.nkv, nova.nkv))
        dp, doff, dpos, dq, dk, dv = (nova.upload(x) for x in (np.array(past, np.int32), off, pos, q, k, v))
        cs, sn = nova.alloc(n * HD * 2), nova.alloc(n * HD * 2)
        o = nova.alloc(q.nbytes)
        nova.launch_rope_angles(dpos.ptr, n, dfreq.ptr, HD, magnitude, cs.ptr, sn.ptr, stream)
        nova.launch_rope_rows_kv_q4_store_batch(dq.ptr, dk.ptr, dv.ptr, cs.ptr, sn.ptr, HD, 0, pool, tables, stride, dp.ptr,
                                                doff.ptr, 2, n, layer, nb, dq.ptr, stream)
        if list(count) == [1, 1]:
            keys = nova.upload((np.array(past) + 1).astype(np.int32))
            ws = nova.alloc(nova.attn_decode_q4_workspace_bytes(2))
            nova.launch_attn_decode_q4_batch(dq.ptr, pool, tables, stride, keys.ptr, 2, layer, nb, o.ptr, ws.ptr, stream)
        else:
            ws = nova.alloc(nova.attn_chunk_q4_workspace_bytes(2, n, max(count)))
            nova.launch_attn_chunk_q4_batch(dq.ptr, pool, tables, stride, dp.ptr, doff.ptr, 2, n, max(count), layer, nb, o.ptr,
                                            ws.ptr, stream)
        nova.dev_stream_sync(stream)
        c, s = (x.numpy((n, HD // 2), np.float32) for x in (cs, sn))
        tq, tk, got = _turn(q, c, s, HD, 0), _turn(k, c, s, HD, 0), o.numpy(q.shape, np.float32)
        for i, sess in enumerate((a, b)):
            rows = slice(off[i], off[i + 1])
            hist[sess][0].extend(tk[rows])
            hist[sess][1].extend(v[rows])
            if count[i]:
                kk, vv = (decode(*quantise(np.stack(x))) for x in hist[sess])
                ref, tol = attention(tq[rows], kk, vv, past[i] + 1, nova.group)
                assert_within(got[rows], ref, tol, f"{name}, session {i}")

    step([0, 0], [40, 0], "prompt")
    nova.nova_paged_attach_prefix(h, b, a, 40)
    hist[b] = tuple(list(x) for x in hist[a])
    before = nova.download(pool, shape, np.uint8)
    shared = nova.download(tables, (3, stride), np.int32)[a, 2]
    nova.nova_paged_session_cow(h, b, 40, 5, stream)         # b writes behind the shared tokens 32 .. 39 first: its page is copied
    nova.nova_paged_session_cow(h, a, 40, 3, stream)
    nova.dev_stream_sync(stream)
    after = nova.download(tables, (3, stride), np.int32)
    assert after[b, 2] != shared and after[a, 2] == shared
    assert np.array_equal(nova.download(pool, shape, np.uint8)[:, after[b, 2]], before[:, shared])
    step([40, 40], [3, 5], "drafts")
    step([43, 45], [1, 1], "token")
    step([44, 46], [60, 2], "chunk and draft")
    step([104, 48], [1, 1], "token")
    # a batch of them, and what an ended session leaves is cleared for the next
    nova.nova_paged_destroy_session(h, b)
    ids = (C.c_int * 1)()
    assert nova.nova_paged_create_sessions(h, 1, 1, ids) == 1
    own = nova.download(tables, (3, stride), np.int32)[ids[0]]
    assert not nova.download(pool, shape, np.uint8)[:, own].any()
    nova.nova_paged_delete(h)
