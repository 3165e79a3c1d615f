"""The step's bookkeeping on the GPU against the plain form, every entry of every array."""
import numpy as np
import pytest

from planref import KB, Planner, pages, plan

pytestmark = pytest.mark.gpu


def _nova():
    import nova_amd
    return nova_amd.load("qwen25_7b")


def _planner(have, stride, spare, max_rows, seed=0, garbage=False):
    rng = np.random.default_rng(seed)
    have = np.asarray(have)
    held = [pages(min(max(int(h), 0), stride * KB)) for h in have]
    nb = sum(held) + spare
    perm = rng.permutation(nb).astype(np.int32)
    tables = np.full((len(have), stride), -5 if garbage else 0, np.int32)
    off = 0
    for i, p in enumerate(held):
        tables[i, :p] = perm[off:off + p]
        off += p
    free = np.full(nb, -9, np.int32)
    free[:nb - off] = perm[off:]
    return Planner(_nova(), tables, have, free, nb - off, max_rows)


def _run(p, keep, new):
    p.set(keep, new)
    p.launch()
    p.nova.dev_sync()
    return p.check()


CASES = {
    "one token each": dict(have=[0, 15, 16, 17, 511], keep=None, new=[1] * 5, stride=40, spare=8, max_rows=5),
    "first of all": dict(have=[0], keep=None, new=[1], stride=1, spare=1, max_rows=1),
    "nothing to do": dict(have=[5, 0, 64], keep=None, new=[0, 0, 0], stride=4, spare=0, max_rows=0),
    "ends and cuts": dict(have=[100, 33, 64, 0, 16], keep=[0, 17, 64, 0, 15], new=[0] * 5, stride=8, spare=3, max_rows=4),
    "cut and grow": dict(have=[100, 33, 64, 7], keep=[90, 16, 1, 7], new=[30, 1, 64, 9], stride=9, spare=2, max_rows=120),
    "no pages left": dict(have=[16, 16, 16, 3], keep=None, new=[16, 1, 1, 1], stride=8, spare=1, max_rows=100),
    "no rows left": dict(have=[0, 0, 0, 0], keep=None, new=[10, 20, 30, 1], stride=8, spare=9, max_rows=45),
    "full table": dict(have=[30, 31, 0], keep=None, new=[2, 2, 33], stride=2, spare=9, max_rows=100),
    "odd lengths": dict(have=[-4, 1000, 20, 9], keep=[3, 5000, -1, 4], new=[5, 1, -7, 2 ** 31 - 1], stride=3, spare=9, max_rows=50),
    "more rows than asked": dict(have=[3, 90], keep=None, new=[4, 8], stride=12, spare=9, max_rows=1500),
    "sixteen and three": dict(have=list(range(0, 760, 40)), keep=None, new=[3] * 19, stride=60, spare=40, max_rows=57),
}


@pytest.mark.parametrize("name", CASES)
def test_plan(name):
    c = CASES[name]
    print(f"[case] plan {name}", flush=True)
    _run(_planner(c["have"], c["stride"], c["spare"], c["max_rows"], garbage=True), c["keep"], c["new"])


@pytest.mark.parametrize("n,stride,most_new,max_rows,spare", [
    (256, 30, 3, 1024, 300), (100, 30, 9, 1025, 300), (2, 30, 400, 1024, 90), (256, 30, 7, 2048, 300), (257, 30, 7, 2049, 300),
    (1024, 12, 40, 30000, 1500), (1025, 12, 40, 1 << 15, 4000), (5000, 4, 3, 9000, 3000),
    (65535, 2, 2, 70000, 9000), (3, 3000, 30000, 60001, 5000), (1, 9000, 100000, 100000, 9000)])
def test_large_plans(n, stride, most_new, max_rows, spare):
    """one launch and two, sessions past a workgroup's threads and past what LDS holds, a stack that runs out"""
    print(f"[case] plan of {n}", flush=True)
    rng = np.random.default_rng(n)
    have = rng.integers(0, stride * KB - min(most_new, stride * 8), n)
    keep = np.where(rng.random(n) < 0.3, have * rng.random(n), have).astype(np.int64)
    p = _planner(have, stride, spare, max_rows, seed=n)
    _run(p, keep, rng.integers(0, most_new + 1, n))
    _run(p, None, rng.integers(0, 2, n))


@pytest.mark.parametrize("max_rows", [64, 4000])
def test_steps_follow_each_other(max_rows):
    """a captured call replayed over many steps of a server: lengths, tables and the stack stay on the GPU,
    updated in place; every step is the plain form's, and no page is in two places"""
    rng = np.random.default_rng(5)
    p = _planner([0] * 12, 20, 90, max_rows, seed=3)
    st = p.nova.dev_stream_create()
    p.set([0] * 12, [3] * 12)
    p.nova.dev_graph_begin(st)
    p.launch(st)
    graph = p.nova.dev_graph_end(st)
    for step in range(25):
        keep = np.where(rng.random(12) < 0.15, (p.have * rng.choice([0, 0.5, 0.95], 12)).astype(int), p.have)
        p.set(keep, rng.choice([0, 1, 1, 1, 8, 70], 12))
        p.nova.dev_graph_launch(graph, st)
        p.nova.dev_stream_sync(st)
        p.check()
        held = [int(x) for i in range(12) for x in p.tables[i, :pages(int(p.have[i]))]] + list(p.free[:p.n_free])
        assert sorted(held) == list(range(p.nb))
    p.nova.dev_graph_destroy(graph)
    p.nova.dev_stream_destroy(st)


def test_undo():
    """what a step adds and the next gives back: the same pages come out again"""
    p = _planner([30, 5, 60], 10, 20, 40, seed=7)
    before = p.tables.copy(), p.free[:p.n_free].copy()
    first = _run(p, None, [20, 9, 5])
    _run(p, [30, 5, 60], [0, 0, 0])
    assert np.array_equal(p.free[:p.n_free], before[1])
    again = _run(p, None, [20, 9, 5])
    assert np.array_equal(first[0], again[0]) and np.array_equal(first[7], again[7])


def test_bad_pages_and_a_stack_too_full():
    """page ids outside the pool come back as they are and have no slots; more pages back than the stack
    has room for: what was free stays, nothing is written behind it"""
    nova = _nova()
    tables = np.array([[900, -3, 1, 2], [3, 0, 1, 2]], np.int32)
    free = np.array([3, 7777, -2, 0], np.int32)              # all four free, though sessions hold pages too
    p = Planner(nova, tables, [20, 64], free, 2, 40)
    p.df = nova.upload(np.concatenate([free, [55, 55, 55, 55]]).astype(np.int32))
    p.set([20, 0], [12, 20])
    p.launch()
    nova.dev_sync()
    got = p.df.numpy((8,), np.int32)
    assert list(got[:2]) == [3, 7777] and (got[4:] == 55).all()
    slots, pos = p.slots.numpy((41,), np.int64), p.pos.numpy((41,), np.int32)
    assert list(pos[:12]) == list(range(20, 32)) and (slots[:12] == -1).all()      # page -3


def test_two_plans_at_once():
    a, b = _planner([5] * 40, 30, 300, 900, seed=1), _planner(list(range(300)), 30, 600, 5000, seed=2)
    a.set(None, [20] * 40)
    b.set(None, [9] * 300)
    s1, s2 = a.nova.dev_stream_create(), a.nova.dev_stream_create()
    a.launch(s1)
    b.launch(s2)
    a.nova.dev_sync()
    a.check()
    b.check()
    a.nova.dev_stream_destroy(s1)
    a.nova.dev_stream_destroy(s2)
