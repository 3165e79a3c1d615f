"""8-bit pages without a GPU: the format's numpy form against itself, and the
refusals of the entry points, which abort on the host before any HIP call."""
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

from q8ref import HD, KB, REC, attention, pack, quantise, unpack

ROOT = Path(__file__).resolve().parent.parent


def test_pack_places_every_byte():
    rng = np.random.default_rng(1)
    kc, vc = (rng.integers(-127, 128, (2, KB, HD)).astype(np.int8) for _ in range(2))
    ks, vs = (rng.standard_normal((2, KB)).astype(np.float32) for _ in range(2))
    rec = pack(kc, ks, vc, vs)
    for t, d in ((0, 0), (5, 37), (15, 127), (8, 64), (3, 16)):
        assert rec[1].view(np.int8)[(t >> 2) * 512 + (d >> 4) * 64 + (t & 3) * 16 + (d & 15)] == kc[1, t, d]
        assert rec[1].view(np.int8)[2048 + d * 16 + t] == vc[1, t, d]
    assert rec.shape == (2, REC)
    for a, b in zip(unpack(rec), (kc, ks, vc, vs)):
        assert np.array_equal(a, b)
    for x in unpack(np.zeros((1, REC), np.uint8)):
        assert not x.any()


def test_quantise_is_nearest():
    """no code is further than half a step from the value, ties go to even codes"""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((50, HD)).astype(np.float32)
    c, s = quantise(x)
    assert np.abs(c).max() == 127
    assert (np.abs(x.astype(np.float64) / s[:, None].astype(np.float64) - c) <= 0.5).all()
    tie = np.full(HD, 127, np.float32)
    tie[1:5] = 0.5, 1.5, -2.5, 3.5
    assert list(quantise(tie)[0][1:5]) == [0, 2, -2, 4]


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
        assert n.kv_q8_page_bytes() == n.nkv * REC


STORE = "n.launch_kv_q8_store_batch({pool}, 16, {stride}, 16, {off}, {n}, {rows}, {layer}, {nb}, {k}, 16, None)"
DECODE = "n.launch_attn_decode_q8_batch({q}, {pool}, 16, {stride}, 16, {n}, {layer}, {nb}, 16, {ws}, None)"
CHUNK = ("n.launch_attn_chunk_q8_batch({q}, {pool}, 16, {stride}, 16, {off}, {n}, {rows}, {max_q}, {layer}, {nb}, 16, "
         "{ws}, None)")
ROPE = ("n.launch_rope_kv_q8_store_batch({q}, 16, 16, {cs}, 16, {pool}, 16, {stride}, 16, {off}, {n}, {rows}, {layer}, "
        "{nb}, None)")
LOAD = "n.launch_kv_q8_load_batch({pool}, 16, {stride}, 16, {off}, {n}, {rows}, {layer}, {nb}, {k}, 16, None)"
GOOD = dict(pool=16, stride=4, off=16, n=2, rows=4, layer=0, nb=4, k=16, q=16, ws=16, max_q=2, cs=16)
BAD = [(call, key, value) for call, keys in (
    (STORE, "pool stride n rows layer nb k"), (LOAD, "pool stride n rows layer nb k"), (ROPE, "q cs pool n rows nb"),
    (DECODE, "q pool stride n layer nb ws"), (CHUNK, "q pool stride n rows layer nb ws max_q")) for key in keys.split()
       for value in {"pool": (0, 24), "k": (0, 20), "q": (0, 4), "ws": (0, 8), "cs": (0, 8), "stride": (0,),
                     "n": (0, 65536), "rows": (-1,), "layer": (-1, 28), "nb": (0,), "max_q": (-1, 5)}[key]]


def _abort_run(code):
    return subprocess.run([sys.executable, "-c", code], capture_output=True, text=True,
                          env={"PYTHONPATH": str(ROOT / "conflux-nova_amd"), "HIP_VISIBLE_DEVICES": ""})


def _refused(call, needle="requirement failed"):
    r = _abort_run(f"import ctypes as C, nova_amd; n = nova_amd.load('qwen25_7b'); {call}")
    assert r.returncode == -6 and needle in r.stderr and "HIP" not in r.stderr, (r.returncode, r.stderr[-500:])


@pytest.mark.parametrize("call,key,value", BAD)
def test_bad_arguments_are_refused(call, key, value):
    _refused(call.format(**{**GOOD, key: value}))


@pytest.mark.parametrize("call", [STORE, CHUNK])
def test_uneven_rows_need_offsets(call):
    _refused(call.format(**{**GOOD, "off": None, "rows": 5}), "row_off || n_rows % n_sess == 0")


@pytest.mark.parametrize("ops,needle", [
    ([(1, 2, 0), (3, 2, 1)], "dst_repeats"),               # two copies into one page
    ([(1, 2, 0), (2, 3, 1)], "dst_is_a_source"),           # a chain
    ([(2, 2, 0)], "dst_is_a_source"),                      # onto itself
    ([(1, 8, 0)], "dst < nb"),
    ([(-1, 2, 0)], "src >= 0"),
    ([(1, 2, -1)], "table_index >= 0"),
    ([(0, e + 1, e) for e in range(6)] + [(7, 7, 0)], "dst_is_a_source"),
])
def test_page_copies_that_depend_on_each_other_are_refused(ops, needle):
    arr = f"(nova_amd.CowOp * {len(ops)})(*[nova_amd.CowOp(*o) for o in {ops}])"
    _refused(f"n.launch_kv_q8_cow_apply(16, 8, 16, {arr}, {len(ops)}, None)", needle)


def test_workspace_sizes_refuse_bad_counts():
    _refused("n.attn_decode_q8_workspace_bytes(0)")
    _refused("n.attn_chunk_q8_workspace_bytes(2, 4, 5)")
    import nova_amd
    n = nova_amd.load("qwen25_7b")
    assert n.attn_decode_q8_workspace_bytes(1) % 16 == 0
    assert n.attn_chunk_q8_workspace_bytes(3, 0, 0) >= 16


def test_empty_calls_launch_nothing():
    """no rows, no ops, no pages: they return before any HIP call"""
    call = "; ".join([CHUNK.format(**{**GOOD, "rows": 0, "max_q": 0}), STORE.format(**{**GOOD, "rows": 0}),
                      LOAD.format(**{**GOOD, "rows": 0}), "n.launch_kv_q8_cow_apply(16, 4, None, None, 0, None)",
                      "n.launch_kv_q8_zero_pages(16, 4, None, 0, None)", "print('quiet')"])
    r = _abort_run(f"import nova_amd; n = nova_amd.load('qwen25_7b'); {call}")
    assert r.returncode == 0 and "quiet" in r.stdout, r.stderr[-500:]
