"""launch_kv_step_plan in plain Python, session by session, and its call."""
import numpy as np

KB = 16


def pages(n):
    return -(-n // KB)


def plan(tables, have, keep, new, max_rows, free, n_free, nb):
    """(tables, free, n_free, past, keys, row_off, pos, slots) afterwards"""
    tables, free = tables.copy(), free.copy()
    n, stride = tables.shape
    have = [min(max(int(h), 0), stride * KB) for h in have]
    keep = [min(max(int(k), 0), h) for k, h in zip(have if keep is None else keep, have)]
    back = [int(tables[i, p]) for i in range(n) for p in range(pages(keep[i]), pages(have[i]))]
    stack = [int(x) for x in free[:n_free]] + back[::-1]
    free[:len(stack)] = stack
    rows, closed = [], False
    wished = 0
    pos, slots, taken = [], [], []
    left = len(stack)
    for i in range(n):
        add = max(int(new[i]), 0)
        if keep[i] + add > stride * KB:
            add = 0
        more = pages(keep[i] + add) - pages(keep[i])
        if closed or wished + add > max_rows or more > left:
            closed, add, more = True, 0, 0
        wished += add
        for p in range(more):
            left -= 1
            tables[i, pages(keep[i]) + p] = stack[left]
        rows.append(add)
        for r in range(add):
            p = keep[i] + r
            page = int(tables[i, p // KB])
            pos.append(p)
            slots.append(page * KB + p % KB if 0 <= page < nb else -1)
    off = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    pos = np.array(pos + [-1] * (max_rows - len(pos)), np.int32)
    slots = np.array(slots + [-1] * (max_rows - len(slots)), np.int64)
    return (tables, free, left, np.array(keep, np.int32), np.array(keep, np.int32) + np.array(rows, np.int32), off, pos, slots)


class Planner:
    """Device state of a step: lengths, tables and the stack of free pages."""

    def __init__(self, nova, tables, have, free, n_free, max_rows):
        self.nova, self.tables, self.free = nova, tables.copy(), free.copy()
        self.n, self.stride = tables.shape
        self.nb, self.max_rows = len(free), max_rows
        self.have, self.n_free = np.asarray(have, np.int32), int(n_free)
        self.dt, self.df, self.dh = nova.upload(self.tables), nova.upload(self.free), nova.upload(self.have)
        self.dn = nova.upload(np.array([n_free], np.int32))
        self.keep, self.new = nova.alloc(4 * self.n), nova.alloc(4 * self.n)
        self.past = nova.alloc(4 * self.n)
        self.off = nova.upload(np.full(self.n + 2, 7, np.int32))
        self.pos, self.slots = nova.upload(np.full(max_rows + 1, 7, np.int32)), nova.upload(np.full(max_rows + 1, 7, np.int64))
        self.ws = nova.alloc(nova.kv_step_plan_workspace_bytes(self.n))

    def set(self, keep, new):
        self.want_keep = None if keep is None else np.asarray(keep, np.int32)
        self.want_new = np.asarray(new, np.int32)
        if keep is not None:
            self.nova.dev_upload(self.keep.ptr, self.want_keep.ctypes.data, 4 * self.n)
        self.nova.dev_upload(self.new.ptr, self.want_new.ctypes.data, 4 * self.n)

    def launch(self, stream=None):
        """lengths and the count of free pages are updated in place"""
        self.nova.launch_kv_step_plan(self.dt.ptr, self.stride, self.dh.ptr, self.keep.ptr if self.want_keep is not None else None,
                                      self.new.ptr, self.n, self.max_rows, self.df.ptr, self.dn.ptr, self.nb, self.past.ptr,
                                      self.dh.ptr, self.off.ptr, self.pos.ptr, self.slots.ptr, self.dn.ptr, self.ws.ptr, stream)

    def check(self):
        """against the plain form, from the state before; takes over the state after"""
        want = plan(self.tables, self.have, self.want_keep, self.want_new, self.max_rows, self.free, self.n_free, self.nb)
        n = self.nova
        got = (self.dt.numpy(self.tables.shape, np.int32), self.df.numpy(self.free.shape, np.int32),
               int(self.dn.numpy((1,), np.int32)[0]), self.past.numpy((self.n,), np.int32), self.dh.numpy((self.n,), np.int32),
               self.off.numpy((self.n + 2,), np.int32), self.pos.numpy((self.max_rows + 1,), np.int32),
               self.slots.numpy((self.max_rows + 1,), np.int64))
        for g, guard in ((got[5], 1), (got[6], 1), (got[7], 1)):
            assert (g[-guard:] == 7).all()                   # nothing behind the arrays
        got = got[:5] + tuple(g[:-1] for g in got[5:])
        for name, g, w in zip(("tables", "free pages", "free count", "past", "keys", "row_off", "pos", "slots"), got, want):
            assert np.array_equal(g, w), (name, np.argwhere(np.asarray(g) != np.asarray(w))[:5])
        self.tables, self.free, self.n_free, self.have = want[0], want[1], want[2], want[4]
        return want
