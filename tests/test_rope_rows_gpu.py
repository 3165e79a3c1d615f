"""Rows turned at positions of their own: angles against 64 bits, the rotation against the
formula in fp32 with every product rounded, in every layout."""
import numpy as np
import pytest

from test_q4_store_gpu import FORMS, MODELS, _angles, _nova, _turn

pytestmark = pytest.mark.gpu
HD = 128


@pytest.mark.parametrize("rot,rows", [(128, 1), (128, 300), (64, 37), (2, 5), (98, 700)])
@pytest.mark.parametrize("magnitude", [1.0, 0.1 * np.log(4) + 1])
def test_angles(rot, rows, magnitude):
    """Positions up to 2^28: the angle is exact in a double, its cos and sin are off by an ulp of a double
    or two, so the fp32 numbers differ from the 64-bit ones by half an ulp and next to nothing."""
    nova = _nova("qwen25_7b")
    rng = np.random.default_rng(rot + rows)
    pos = np.concatenate([[0], rng.integers(0, 1 << 20, rows)])[:rows].astype(np.int32)
    pos[-1] = (1 << 28) + 12345
    freq = (1e6 ** (-np.arange(0, rot, 2) / rot)).astype(np.float32)
    dp, df = nova.upload(pos), nova.upload(freq)
    c, s = (nova.upload(np.full((rows + 1, rot // 2), 7, np.float32)) for _ in range(2))
    nova.launch_rope_angles(dp.ptr, rows, df.ptr, rot, magnitude, c.ptr, s.ptr, None)
    nova.dev_sync()
    angle = pos[:, None].astype(np.float64) * freq.astype(np.float64)
    for got, want in ((c, np.cos(angle)), (s, np.sin(angle))):
        got, want = got.numpy((rows + 1, rot // 2), np.float32), want * magnitude
        assert (got[rows:] == 7).all()
        assert (np.abs(got[:rows] - want) <= np.abs(want) * (2.0 ** -24 + 2.0 ** -40) + 2.0 ** -50).all()


def test_angles_are_the_tables():
    """for the model's own rates the rows of launch_rope_table, but for that one's fp32 angle:
    equal where that is exact"""
    nova = _nova("qwen25_7b")
    pos = np.zeros(4, np.int32)
    freq = np.ones(64, np.float32)
    dp, df = nova.upload(pos), nova.upload(freq)
    c, s, tc, ts = (nova.alloc(4096 * 64 * 4) for _ in range(4))
    nova.launch_rope_angles(dp.ptr, 4, df.ptr, 128, 1.0, c.ptr, s.ptr, None)
    nova.launch_rope_table(tc.ptr, ts.ptr, None)
    pos2 = nova.upload(np.arange(4096, dtype=np.int32))
    c2, s2 = nova.alloc(4096 * 64 * 4), nova.alloc(4096 * 64 * 4)
    nova.launch_rope_angles(pos2.ptr, 4096, df.ptr, 128, 1.0, c2.ptr, s2.ptr, None)
    nova.dev_sync()
    assert (c.numpy((4, 64), np.float32) == 1).all() and not s.numpy((4, 64), np.float32).any()
    # pair 0 turns by one radian a position in both
    assert np.array_equal(c2.numpy((4096, 64), np.float32)[:, 0], tc.numpy((4096, 64), np.float32)[:, 0])
    assert np.array_equal(s2.numpy((4096, 64), np.float32)[:, 5], ts.numpy((4096, 64), np.float32)[:, 0])


@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("rot,beside", FORMS)
@pytest.mark.parametrize("rows", [1, 19])
def test_rows(model, rot, beside, rows):
    nova = _nova(model)
    print(f"[case] rope rows {model} rot={rot} beside={beside} rows={rows}", flush=True)
    rng = np.random.default_rng(rot)
    q = rng.standard_normal((rows + 1, nova.nh, HD)).astype(np.float32)
    k = rng.standard_normal((rows + 1, nova.nkv, HD)).astype(np.float32)
    c, s = _angles(rng, rows + 1, rot)
    pos = np.arange(rows + 1, dtype=np.int32)
    pos[rows // 2] = -1 if rows > 1 else 0
    turned = pos[:rows] >= 0
    for positions in (None, pos):
        dq, dk, dc, ds, dp = (nova.upload(x) for x in (q, k, c, s, pos))
        oq, ok = (nova.upload(np.full(x.shape, 7, np.float32)) for x in (q, k))
        for to_q, to_k in ((oq, ok), (dq, dk)):
            nova.launch_rope_rows(dq.ptr, dk.ptr, dp.ptr if positions is not None else None, dc.ptr, ds.ptr, rows, rot, beside,
                                  to_q.ptr, to_k.ptr, None)
            nova.dev_sync()
            for to, x in ((to_q, q), (to_k, k)):
                got, want = to.numpy(x.shape, np.float32), _turn(x, c, s, rot, beside)
                live = turned if positions is not None else np.ones(rows, bool)
                assert np.array_equal(got[:rows][live], want[:rows][live])
                kept = np.full_like(x, 7) if to in (oq, ok) else x           # rows at -1, rows behind the last
                assert np.array_equal(got[:rows][~live], kept[:rows][~live]) and np.array_equal(got[rows:], kept[rows:])


def test_back_and_forth_in_a_graph():
    """angles and rotation captured, replayed with new positions; turning by -p undoes p"""
    nova = _nova("qwen25_7b")
    rng = np.random.default_rng(3)
    rows, rot = 40, 128
    q = rng.standard_normal((rows, nova.nh, HD)).astype(np.float32)
    k = rng.standard_normal((rows, nova.nkv, HD)).astype(np.float32)
    freq = (1e4 ** (-np.arange(0, rot, 2) / rot)).astype(np.float32)
    dq, dk, df, dp = (nova.upload(x) for x in (q, k, freq, np.zeros(rows, np.int32)))
    oq, ok = nova.alloc(q.nbytes), nova.alloc(k.nbytes)
    c, s = nova.alloc(rows * rot * 2), nova.alloc(rows * rot * 2)
    st = nova.dev_stream_create()

    def launch():
        nova.launch_rope_angles(dp.ptr, rows, df.ptr, rot, 1.0, c.ptr, s.ptr, st)
        nova.launch_rope_rows(dq.ptr, dk.ptr, dp.ptr, c.ptr, s.ptr, rows, rot, 0, oq.ptr, ok.ptr, st)

    launch()
    nova.dev_stream_sync(st)
    nova.dev_graph_begin(st)
    launch()
    graph = nova.dev_graph_end(st)
    for trip in range(3):
        pos = rng.integers(0, 1 << 18, rows).astype(np.int32)
        nova.dev_upload(dp.ptr, pos.ctypes.data, pos.nbytes)
        nova.dev_graph_launch(graph, st)
        nova.dev_stream_sync(st)
        angle = pos[:, None].astype(np.float64) * freq.astype(np.float64)
        want = _turn(q, np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32), rot, 0)
        got = oq.numpy(q.shape, np.float32)
        # cos and sin may round the other way once in a while: 2^-23 of the pair
        pair = np.abs(q[..., :64]) + np.abs(q[..., 64:])
        assert (np.abs(got - want) <= 2.0 ** -22 * np.concatenate([pair, pair], -1)).all()
        launch()                                             # eager work between the replays
        nova.dev_stream_sync(st)
        assert np.array_equal(oq.numpy(q.shape, np.float32), got)
    nova.dev_graph_destroy(graph)
    nova.dev_stream_destroy(st)
