"""4-bit pages without a GPU: the format's numpy form against itself, and the
refusals of the entry points, which abort on the host before any HIP call."""
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

from q4ref import GRID, HD, KB, NAN, REC, attention, decode, pack, quantise, unpack

ROOT = Path(__file__).resolve().parent.parent


def test_pack_places_every_byte():
    rng = np.random.default_rng(1)
    kc, vc = (rng.integers(0, 16, (2, KB, HD)).astype(np.uint8) for _ in range(2))
    ke, ve = (rng.integers(0, 256, (2, KB, 4)).astype(np.uint8) for _ in range(2))
    rec = pack(kc, ke, vc, ve)
    for t, d in ((0, 0), (5, 37), (15, 127), (8, 64), (3, 16), (9, 111)):
        assert rec[1][t * 64 + (d >> 1)] >> (4 * (d & 1)) & 15 == kc[1, t, d]
        assert rec[1][1024 + (d >> 5) * 256 + (d & 15) * 16 + t] >> (4 * (d >> 4 & 1)) & 15 == vc[1, t, d]
        assert rec[1][2048 + (t & 3) * 16 + (d >> 5) * 4 + (t >> 2)] == ke[1, t, d >> 5]
        assert rec[1][2112 + (d >> 5) * 16 + t] == ve[1, t, d >> 5]
    assert rec.shape == (2, REC)
    for a, b in zip(unpack(rec), (kc, ke, vc, ve)):
        assert np.array_equal(a, b)
    for x in unpack(np.zeros((1, REC), np.uint8)):
        assert not x.any()


def test_quantise_is_nearest():
    """no value is off by more than half a step of its size, and no smaller power would do"""
    rng = np.random.default_rng(2)
    x = (rng.standard_normal((500, HD)) * np.exp(3 * rng.standard_normal((500, 1)))).astype(np.float32)
    c, b = quantise(x)
    unit = np.repeat(np.ldexp(1.0, b.astype(int) - 127), 32, -1)
    m = np.abs(x) / unit
    step = np.where(m < 2, .5, np.where(m < 4, 1, 2))
    assert (np.abs(decode(c, b) - x) <= step / 2 * unit).all()
    top = m.reshape(-1, 4, 32).max(-1)
    assert (top <= 7).all() and (top > 3.5).all()
    tie = np.zeros(HD, np.float32)
    tie[:9] = 7, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -2.5
    assert list(decode(*quantise(tie))[:9]) == [6, 0, 1, 1, 2, 2, 4, 4, -2]
    assert list(quantise(np.full(HD, 3.5 * 2.0 ** -100, np.float32))[1]) == [0] * 4
    assert list(quantise(np.full(HD, 3.6 * 2.0 ** -100, np.float32))[1]) == [27] * 4
    assert list(quantise(np.full(HD, np.finfo(np.float32).max, np.float32))[1]) == [223] * 4
    bad = np.ones(HD, np.float32)
    bad[40] = np.inf
    assert list(quantise(bad)[1]) == [NAN] * 4
    assert (GRID[quantise(np.ones(HD, np.float32))[0] & 7] == 4).all()       # 1 = 4 * 2^-2


def test_attention_reference_sees_its_keys():
    rng = np.random.default_rng(3)
    q = rng.standard_normal((2, 2, HD)).astype(np.float32)
    k, v = rng.standard_normal((2, 3, 1, HD))
    o, _ = attention(q, k, v, 1, 2)
    assert np.allclose(o[0], v[0, 0])                     # the first row sees one key
    o, _ = attention(q[:1], k, v, 0, 2)
    assert not o.any()


def test_page_bytes():
    import nova_amd
    for m in nova_amd.MODELS:
        n = nova_amd.load(m)
        assert n.kv_q4_page_bytes() == n.nkv * REC


STORE = "n.launch_kv_q4_store_batch({pool}, 16, {stride}, 16, {off}, {n}, {rows}, {layer}, {nb}, {k}, 16, None)"
DECODE = "n.launch_attn_decode_q4_batch({q}, {pool}, 16, {stride}, 16, {n}, {layer}, {nb}, 16, {ws}, None)"
CHUNK = ("n.launch_attn_chunk_q4_batch({q}, {pool}, 16, {stride}, 16, {off}, {n}, {rows}, {max_q}, {layer}, {nb}, 16, "
         "{ws}, None)")
ROPE = ("n.launch_rope_rows_kv_q4_store_batch({q}, 16, 16, {cs}, 16, {rot}, 0, {pool}, 16, {stride}, 16, {off}, {n}, {rows}, "
        "{layer}, {nb}, {k}, None)")
LOAD = "n.launch_kv_q4_load_batch({pool}, 16, {stride}, 16, {off}, {n}, {rows}, {layer}, {nb}, {k}, 16, None)"
ANGLES = "n.launch_rope_angles({k}, {rows}, 16, {rot}, {mag}, {cs}, 16, None)"
TURN = "n.launch_rope_rows({q}, 16, None, {cs}, 16, {rows}, {rot}, 0, {k}, 16, None)"
PLAN = ("n.launch_kv_step_plan({pool}, {stride}, 16, None, 16, {n}, {rows}, {k}, 16, {nb}, 16, 16, 16, {q}, 16, 16, {ws}, "
        "None)")
GOOD = dict(pool=16, stride=4, off=16, n=2, rows=4, layer=0, nb=4, k=16, q=16, ws=16, max_q=2, cs=16, rot=128, mag=1.0)
VALUES = {"pool": (0, 24), "k": (0, 20), "q": (0, 4), "ws": (0, 8), "cs": (0, 8), "stride": (0,), "n": (0, 65536),
          "rows": (-1, (1 << 24) + 2), "layer": (-1, 28), "nb": (0,), "max_q": (-1, 5), "rot": (0, 7, 130)}
BAD = [(call, key, value) for call, keys in (
    (STORE, "pool stride n rows layer nb k"), (LOAD, "pool stride n rows layer nb k"),
    (ROPE, "q cs pool n rows nb rot k"), (DECODE, "q pool stride n layer nb ws"),
    (CHUNK, "q pool stride n rows layer nb ws max_q"), (TURN, "q cs rows rot k"), (ANGLES, "rows rot"),
    (PLAN, "stride n rows nb ws")) for key in keys.split() for value in VALUES[key]]
BAD += [(ANGLES, "k", 0), (ANGLES, "cs", 0), (ANGLES, "mag", "float('nan')"), (PLAN, "pool", 0), (PLAN, "k", 0),
        (PLAN, "q", 0), (PLAN, "nb", (1 << 27) + 1), (PLAN, "stride", (1 << 26) + 1)]


def _abort_run(code):
    return subprocess.run([sys.executable, "-c", code], capture_output=True, text=True,
                          env={"PYTHONPATH": str(ROOT / "conflux-nova_amd"), "HIP_VISIBLE_DEVICES": ""})


def _refused(call, needle="requirement failed"):
    r = _abort_run(f"import ctypes as C, nova_amd; n = nova_amd.load('qwen25_7b'); {call}")
    assert r.returncode == -6 and needle in r.stderr and "HIP" not in r.stderr, (call, r.returncode, r.stderr[-500:])


@pytest.mark.parametrize("call,key,value", BAD)
def test_bad_arguments_are_refused(call, key, value):
    _refused(call.format(**{**GOOD, key: value}))


@pytest.mark.parametrize("call", [STORE, CHUNK, ROPE])
def test_uneven_rows_need_offsets(call):
    _refused(call.format(**{**GOOD, "off": None, "rows": 5}), "row_off || n_rows % n_sess == 0")


@pytest.mark.parametrize("ops,needle", [([(1, 2, 0), (3, 2, 1)], "dst_repeats"), ([(1, 2, 0), (2, 3, 1)], "dst_is_a_source"),
                                        ([(1, 8, 0)], "dst < nb")])
def test_page_copies_that_depend_on_each_other_are_refused(ops, needle):
    arr = f"(nova_amd.CowOp * {len(ops)})(*[nova_amd.CowOp(*o) for o in {ops}])"
    _refused(f"n.launch_kv_q4_cow_apply(16, 8, 16, {arr}, {len(ops)}, None)", needle)


def test_workspace_sizes_refuse_bad_counts():
    _refused("n.attn_decode_q4_workspace_bytes(0)")
    _refused("n.attn_chunk_q4_workspace_bytes(2, 4, 5)")
    _refused("n.kv_step_plan_workspace_bytes(0)")
    import nova_amd
    n = nova_amd.load("qwen25_7b")
    assert n.attn_decode_q4_workspace_bytes(1) % 16 == 0
    assert n.attn_chunk_q4_workspace_bytes(3, 0, 0) >= 16


def test_empty_calls_launch_nothing():
    """no rows, no ops, no pages: they return before any HIP call"""
    none = {**GOOD, "rows": 0, "max_q": 0}
    call = "; ".join([c.format(**none) for c in (CHUNK, STORE, LOAD, ROPE, ANGLES, TURN)] +
                     ["n.launch_kv_q4_cow_apply(16, 4, None, None, 0, None)",
                      "n.launch_kv_q4_zero_pages(16, 4, None, 0, None)", "print('quiet')"])
    r = _abort_run(f"import nova_amd; n = nova_amd.load('qwen25_7b'); {call}")
    assert r.returncode == 0 and "quiet" in r.stdout, r.stderr[-500:]


# ---- turning rates (host only) ----

def _freqs(**cfg):
    import ctypes as C
    import nova_amd
    n = nova_amd.load("qwen25_7b")
    c = nova_amd.RopeCfg(**{**dict(rot_dim=128, scaling=0, base=1e6, factor=1.0, train_len=0, slow_turns=1, fast_turns=32), **cfg})
    out, mag = (C.c_float * 64)(), C.c_double()
    assert n.nova_rope_freqs(C.byref(c), out, C.byref(mag)) == c.rot_dim // 2
    return np.array(out[:c.rot_dim // 2], np.float32), mag.value


@pytest.mark.parametrize("rot", [2, 64, 96, 128])
def test_rope_freqs(rot):
    i = np.arange(0, rot, 2)
    plain = 1e6 ** (-i / rot)
    near = dict(rtol=2.0 ** -23, atol=0)                     # rounded to fp32 once, from a double that may be an ulp off
    f, m = _freqs(rot_dim=rot)
    assert np.allclose(f, plain, **near) and m == 1 and f[0] == 1
    f, m = _freqs(rot_dim=rot, scaling=1, factor=4.0)
    assert np.allclose(f, plain / 4, **near) and m == 1
    f, m = _freqs(rot_dim=rot, scaling=2, factor=4.0)
    # the slowest pair turns 4 times slower, the fastest as before
    assert f[0] == 1 and m == 1 and (rot == 2 or np.isclose(f[-1], plain[-1] / 4, rtol=1e-6))
    f, m = _freqs(rot_dim=rot, scaling=3, factor=4.0, train_len=32768)
    assert np.isclose(m, 0.1 * np.log(4) + 1, rtol=1e-15)
    turns = 32768 * plain / (2 * np.pi)
    assert np.allclose(f[turns >= 32], plain[turns >= 32], **near)
    assert np.allclose(f[turns <= 1], plain[turns <= 1] / 4, **near)
    between = (turns > 1) & (turns < 32)
    keep = (turns[between] - 1) / 31
    assert np.allclose(f[between], plain[between] * (keep + (1 - keep) / 4), **near)


CFG = "nova_amd.RopeCfg({rot_dim}, {scaling}, {base}, {factor}, {train_len}, {slow_turns}, {fast_turns})"


@pytest.mark.parametrize("bad", [dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=130), dict(scaling=4), dict(scaling=-1),
                                 dict(base=0.0), dict(base="float('inf')"), dict(factor=0.5), dict(factor="float('nan')"),
                                 dict(train_len=0), dict(slow_turns=40.0), dict(slow_turns=-1.0)])
def test_rope_freqs_refuse(bad):
    cfg = {**dict(rot_dim=64, scaling=3, base=1e4, factor=2.0, train_len=100, slow_turns=1.0, fast_turns=32.0), **bad}
    _refused(f"n.nova_rope_freqs(C.byref({CFG.format(**cfg)}), (C.c_float * 64)(), C.byref(C.c_double()))")
