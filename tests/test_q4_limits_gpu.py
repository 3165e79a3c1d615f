"""Attention over 4-bit pages where one form takes over from another: by columns (query rows times heads of a kv
head: 16 to a workgroup, up to 64 in one launch, groups of 64 past it), by the table's pages and by workgroups."""
import numpy as np
import pytest

from q4ref import KB, Call

pytestmark = pytest.mark.gpu
# query heads of a kv head
GROUP = {"qwen25_1p5b": 6, "qwen25_7b": 7, "qwen25_14b": 5}


def _cut(c, stride):
    """the call with a table of `stride` pages"""
    assert c.table.shape[1] >= stride
    c.table = np.ascontiguousarray(c.table[:, :stride])
    c.upload()
    c.run()
    c.check(f"{stride} pages, up to {c.max_q} rows")


@pytest.mark.parametrize("model", GROUP)
@pytest.mark.parametrize("stride", [64, 65, 96, 97])
@pytest.mark.parametrize("cols", [32, 48, 64])
def test_columns_and_pages(model, stride, cols):
    """The most rows of that many columns and one more, few sessions and enough of them for longer tables; in each
    call some sessions of no rows, of one, and of fewer than the others."""
    most = stride * KB
    for rows in (cols // GROUP[model], cols // GROUP[model] + 1):
        print(f"[case] q4 limits {model} stride={stride} rows={rows}", flush=True)
        _cut(Call(model, [most - rows, 9, 0, 500], [rows, 1, rows, 0], seed=75), stride)
        many = -(-64 // (2 if model == "qwen25_1p5b" else 4 if model == "qwen25_7b" else 8))
        past = [most - rows] + [40 + 3 * i for i in range(many - 1)]
        _cut(Call(model, past, [rows] + [i % (rows + 1) for i in range(many - 1)], seed=76), stride)


@pytest.mark.parametrize("past", [0, 1, 15, 16, 63, 64, 700])
@pytest.mark.parametrize("rows", [5, 7, 9])
def test_blocks_of_one_session(rows, past):
    """three and four blocks of 16 columns, the last one not whole, at the ends of pages and tiles"""
    _cut(Call("qwen25_7b", [past], [rows], seed=77), -(-(past + rows) // KB))
