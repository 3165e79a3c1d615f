"""Steps in which a session gets no rows: at its table's end between others that are served, or from
where the pages run out."""
import numpy as np
import pytest

from q4ref import HD, assert_within, attention, decode, quantise
from test_q4_step_gpu import Server

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "replayed"])
@pytest.mark.parametrize("stride", [3, 66, 100])
def test_single_tokens_beside_a_full_session(graph, stride):
    """The chunk call with a row a session at most, in one launch and in two.  Session 2 fills its
    table, and the rows of those after it move up; then it ends and starts again."""
    print(f"[case] refused step, stride={stride} graph={graph}", flush=True)
    most = 16 * stride
    s = Server("qwen25_7b", 5, stride, stride + 9, 4 + most, most, seed=stride)
    s.step(None, [3, 1, most - 2, 15, 7], what="prompts")
    s.max_q = 1
    for t in range(2):
        assert s.step(None, [1] * 5, graph=graph, what=f"token {t}") == 5
    for t in range(3):
        assert s.step(None, [1] * 5, graph=graph, what=f"session 2 is full {t}") == 4
        assert list(s.plan.off.numpy((6,), np.int32)) == [0, 1, 2, 2, 3, 4]
    keep = s.plan.have.copy()
    keep[2] = 0
    assert s.step(keep, [1] * 5, graph=graph, what="it starts again") == 5
    s.read_back()
    s.close()


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "replayed"])
def test_single_tokens_until_the_pages_run_out(graph):
    print(f"[case] pages run out graph={graph}", flush=True)
    s = Server("qwen25_7b", 4, 40, 5, 60, 16, seed=3)
    s.step(None, [15, 16, 2, 16], what="prompts")            # a page each, one left
    s.max_q = 1
    assert s.step(None, [1] * 4, graph=graph, what="the last page") == 3          # session 1 has it, 3 finds none
    assert s.step(None, [1] * 4, graph=graph, what="none left") == 0              # nor does 0, and nobody after it
    keep = s.plan.have.copy()
    keep[3] = 0
    assert s.step(keep, [1, 1, 1, 0], graph=graph, what="one ends") == 3
    s.read_back()
    s.close()


def test_a_decode_reads_row_i_for_session_i():
    """and writes every row: where the last session got none, the rows of the others are theirs, and its row
    is made of its query as it came, over the keys that it holds"""
    s = Server("qwen25_7b", 3, 2, 9, 57, 32, seed=8)
    assert s.step(None, [5, 20, 32], what="prompts") == 57
    nova, rng = s.nova, np.random.default_rng(1)
    q = rng.standard_normal((s.max_rows, nova.nh, HD)).astype(np.float32)
    kv = [rng.standard_normal((s.max_rows, nova.nkv, HD)).astype(np.float32) for _ in range(2)]
    for dev, x in zip([s.q[0], *s.kv[0]], [q, *kv]):
        nova.dev_upload(dev.ptr, x.ctypes.data, x.nbytes)
    s.plan.set(s.plan.have, [1, 1, 1])
    s.launch(True)
    nova.dev_stream_sync(s.stream)
    off, keys = s.plan.check()[5], s.plan.have
    assert list(off) == [0, 1, 2, 2] and list(keys) == [6, 21, 32]
    got, turned = s.o[0].numpy(q.shape, np.float32), s.q[0].numpy(q.shape, np.float32)
    assert np.array_equal(turned[2:], q[2:]) and not np.array_equal(turned[:2], q[:2])
    kk, vv = (decode(*quantise(h[0][2])) for h in (s.past_k, s.past_v))
    ref, tol = attention(q[2:3], kk, vv, 32, nova.group)
    assert_within(got[2:3], ref, tol, "the session that got none")
    s.close()
