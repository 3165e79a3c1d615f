"""The 4-bit page format and the operators over it in numpy, in 64 bits, from
their definitions (include/nova_kernel.h): packing, the quantiser, attention."""
from __future__ import annotations

import numpy as np

KB, HD, REC = 16, 128, 2176
GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
NAN = 255


def quantise(x):
    """(codes uint8 [..., 128], exponent bytes uint8 [..., 4]) of rows x [..., 128] fp32."""
    x = np.asarray(x, np.float32).astype(np.float64)
    y = x.reshape(x.shape[:-1] + (4, 32))
    with np.errstate(all="ignore"):
        top = np.abs(y).max(-1)                              # NaN propagates
        _, ex = np.frexp(np.where(np.isfinite(top), top, 1.0))
        e = ex - 3                                           # top in [2^(ex-1), 2^ex): 7 2^e from 7/8 2^ex down
        e = np.where(top > 7 * np.ldexp(1.0, e), e + 1, e)
        byte = np.where(top > 0, np.minimum(e + 127, 223), 0)
        byte = np.where(byte < 27, 0, byte)
        m = np.abs(np.ldexp(y, (127 - byte)[..., None]))
        up = np.searchsorted((GRID[1:] + GRID[:-1]) / 2, np.where(np.isfinite(m), m, 0), side="right")
        down = np.searchsorted((GRID[1:] + GRID[:-1]) / 2, np.where(np.isfinite(m), m, 0), side="left")
    code = np.where(up % 2 == 0, up, down) | np.where(np.signbit(y), 8, 0)
    code = np.where(byte[..., None] > 0, code, 0).reshape(x.shape)
    bad = ~np.isfinite(x).all(-1)
    code[bad] = 0
    byte[bad] = NAN
    return code.astype(np.uint8), byte.astype(np.uint8)


def decode(code, byte):
    """float64 values of codes [..., 128] and exponent bytes [..., 4]"""
    v = GRID[code & 7] * np.where(code & 8, -1.0, 1.0)
    b = byte.astype(np.int64)
    p = np.where(b == NAN, np.nan, np.where(b == 0, 0.0, np.ldexp(1.0, b - 127)))
    return v * np.repeat(p, 32, -1)


def pack(kc, ke, vc, ve):
    """records [..., 2176] uint8 of pages kc, vc [..., 16, 128], ke, ve [..., 16, 4]"""
    lead = kc.shape[:-2]
    rec = np.empty(lead + (REC,), np.uint8)
    rec[..., :1024] = (kc[..., 0::2] | (kc[..., 1::2] << 4)).reshape(lead + (1024,))
    v = vc.reshape(lead + (KB, 4, 2, 16))
    v = v[..., 0, :] | (v[..., 1, :] << 4)                   # [token][32s][dim]
    rec[..., 1024:2048] = np.moveaxis(v, -3, -1).reshape(lead + (1024,))
    e = ke.reshape(lead + (4, 4, 4))                         # [t >> 2][t & 3][32s]
    rec[..., 2048:2112] = np.moveaxis(e, -3, -1).reshape(lead + (64,))
    rec[..., 2112:] = np.swapaxes(ve, -1, -2).reshape(lead + (64,))
    return rec


def unpack(rec):
    lead = rec.shape[:-1]
    k = rec[..., :1024].reshape(lead + (KB, 64))
    kc = np.stack([k & 15, k >> 4], -1).reshape(lead + (KB, HD))
    v = np.moveaxis(rec[..., 1024:2048].reshape(lead + (4, 16, KB)), -1, -3)
    vc = np.stack([v & 15, v >> 4], -2).reshape(lead + (KB, HD))
    ke = np.moveaxis(rec[..., 2048:2112].reshape(lead + (4, 4, 4)), -1, -3).reshape(lead + (KB, 4))
    ve = np.swapaxes(rec[..., 2112:].reshape(lead + (4, KB)), -1, -2)
    return kc, ke, vc, ve


class Q4Pool:
    """Random 4-bit pages of one layer on the device and on the host.  Pages lie
    anywhere in the pool; the other layers are device memory nobody touched."""

    def __init__(self, nova, nb, layer, seed):
        self.nova, self.nb, self.layer = nova, nb, layer
        self.rng = rng = np.random.default_rng(seed)
        self.page = nova.nkv * REC
        assert nova.kv_q4_page_bytes() == self.page
        self.dev = nova.alloc((layer + 1) * nb * self.page)
        # keys with a few strong channels and uneven tokens, as projections give
        gain = np.ones(HD, np.float32)
        gain[rng.permutation(HD)[:4]] = 5
        tok = np.exp(0.25 * rng.standard_normal((nb, nova.nkv, KB, 1))).astype(np.float32)
        k = rng.standard_normal((nb, nova.nkv, KB, HD)).astype(np.float32) * gain * tok
        v = rng.standard_normal((nb, nova.nkv, KB, HD)).astype(np.float32) * tok[:, :, ::-1]
        self.rec = pack(*quantise(k), *quantise(v))
        self.push()

    def off(self):
        return self.layer * self.nb * self.page

    def push(self):
        self.nova.dev_upload(self.dev.ptr + self.off(), self.rec.ctypes.data, self.rec.nbytes)

    def pull(self):
        return self.nova.download(self.dev, self.rec.shape, np.uint8, self.off())

    def tables(self, pages, extra=3, fill=0x7ffffff0):
        """Rows over shuffled pages; entries that no key needs hold `fill`."""
        pages = np.asarray(pages)
        stride = max(int(pages.max()), 1) + extra
        out = np.full((len(pages), stride), fill, np.int32)
        perm = self.rng.permutation(self.nb).astype(np.int32)
        assert pages.sum() <= self.nb
        at = 0
        for i, p in enumerate(pages):
            out[i, :p] = perm[at:at + p]
            at += p
        return out

    def poison_behind(self, table, n_keys):
        """NaN and loud codes in every slot of the sessions' last pages that holds no key."""
        for i, n in enumerate(n_keys):
            if n % KB:
                kc, ke, vc, ve = (np.array(x) for x in unpack(self.rec[table[i, n // KB]]))
                kc[:, n % KB:], vc[:, n % KB:] = 15, 7
                ke[:, n % KB:], ve[:, n % KB:] = NAN, NAN
                ve[:, n % KB::2] = 254
                self.rec[table[i, n // KB]] = pack(kc, ke, vc, ve)
        self.push()


def values(rec, table, n):
    """K, V [n][NKV][128] float64 of a session's first n tokens"""
    pos = np.arange(n)
    kc, ke, vc, ve = unpack(rec[table[pos >> 4]])
    at = np.arange(n), slice(None), pos & 15
    return decode(kc[at], ke[at]), decode(vc[at], ve[at])


def attention(q, k, v, first, group):
    """Rows q [n][NH][128] over k, v [T][NKV][128] float64, row r seeing keys
    [0, first + r); and how far an fp32 result may be from it, per output element.

    The bound: a score is a sum of 128 products in fp32 against q that was scaled
    (2^-24 of each q_d) and is held to 2^-24 of the largest of its 32 dims; five
    instructions add the products up, each off by at most 2^-23 of the sum of their
    sizes.  All of that is below 2^-20 of sum |q_d k_d| + max|q| sum |k_d|, and so is the
    rounding of score less reference: the score's error.  A weight carries it and 2^-20 from
    exp2 and the rescaling; the weight itself goes in whole.  The sums over n keys run
    through chains of at most 3 n / 32 + 64 additions of 2^-24.  With weights off by e
    relatively, sum p_j v_j / sum p_j is off by at most 2 e sum p_j |v_j|, of the keys that the
    row sees.  Weights are fp32 numbers relative to a reference that is at most the row's
    largest score, so one below 2^-126 of the largest is no normal number and may count as 0
    (as its product with a value may, and once more where pieces are joined): each of
    n keys then adds up to 2^-125 of the largest |v|.  A weight in fp16 terms is cut below 2^-24
    where the largest of its tile (64 keys from a multiple of 64) stands at 2^2 or more, so it
    loses up to 2^-26 of that one, or, where the reference has come down by its 80 octaves,
    2^-102 of the row's largest."""
    n, nh, _ = q.shape
    out, tol = np.zeros((n, nh, HD)), np.zeros((n, nh, HD))
    if len(k) == 0:
        return out, tol
    for h in range(nh):
        kh, vh = k[:, h // group], v[:, h // group]
        x = q[:, h].astype(np.float64)
        seen = np.arange(len(kh))[None, :] < np.minimum(first + np.arange(n), len(kh))[:, None]
        kz, vz = np.nan_to_num(kh), np.nan_to_num(vh)        # (a hidden key may be NaN)
        s = x @ kz.T / np.sqrt(HD)
        size = (np.abs(x) @ np.abs(kz).T + np.abs(x).max(-1, keepdims=True) * np.abs(kz).sum(-1)) / np.sqrt(HD)
        s = np.where(seen, s, -np.inf)
        with np.errstate(invalid="ignore"):
            p = np.exp(s - s.max(-1, keepdims=True))
            p = np.where(seen, p / p.sum(-1, keepdims=True), 0)
        out[:, h] = p @ vz
        e = 2.0 ** -20 * np.where(seen, size, 0).max(-1) + 2.0 ** -20 + (3 * len(kh) / 32 + 64) * 2.0 ** -24
        most = np.where(seen, np.abs(vz).max(-1), 0).max(-1)
        tiles = np.arange(len(kh)) // 64
        tops = np.stack([p[:, tiles == t].max(-1) for t in range(tiles[-1] + 1)], -1)[:, tiles] * seen
        tol[:, h] = (2 * e[:, None] * (p @ np.abs(vz)) + 2.0 ** -26 * (tops @ np.abs(vz)) +
                     (seen.sum(-1) * (2.0 ** -125 + 2.0 ** -102) * most)[:, None])
    return out, tol


def assert_within(got, ref, tol, what):
    assert np.isfinite(got).all(), f"{what}: not finite"
    err = np.abs(got.astype(np.float64) - ref)
    worst = (err / np.maximum(tol, 1e-44)).max(initial=0)
    assert (err <= tol).all(), f"{what}: {worst:.2f} of the bound, max abs {err.max():.3e}"
    return worst


class Call:
    """An attention call over random pages: a chunk of `count` rows per session behind `past`
    keys, or (decode) one query per session over `past` keys."""

    def __init__(self, model, past, count=None, seed=0, scale=1.5, max_q=None, behind=2, offsets=True, poison=True, layer=3):
        import nova_amd
        self.nova = nova = nova_amd.load(model)
        self.layer, self.decode = layer, count is None
        self.past = np.asarray(past, np.int32)
        self.count = np.ones(len(past), int) if self.decode else np.asarray(count)
        self.keys = self.past if self.decode else np.where(self.count > 0, self.past + self.count, 0)
        self.off = np.concatenate([[0], np.cumsum(self.count)]).astype(np.int32)
        self.n_rows = int(self.off[-1]) + (0 if self.decode else behind)
        self.max_q = int(self.count.max()) if max_q is None else max_q
        pages = (self.keys + KB - 1) // KB
        self.pool = Q4Pool(nova, int(pages.sum()) + 2, layer, seed)
        self.table = self.pool.tables(pages)
        if poison:
            self.pool.poison_behind(self.table, self.keys)
        self.q = (self.pool.rng.standard_normal((self.n_rows, nova.nh, HD)) * scale).astype(np.float32)
        self.offsets = offsets
        self.upload()
        n = len(past)
        self.ws = nova.alloc(nova.attn_decode_q4_workspace_bytes(n) if self.decode else
                             nova.attn_chunk_q4_workspace_bytes(n, self.n_rows, self.max_q))

    def upload(self):
        self.dt, self.dp, self.doff, self.dq = (self.nova.upload(np.ascontiguousarray(x))
                                                for x in (self.table, self.past, self.off, self.q))
        self.o = self.nova.upload(np.full(self.q.shape, 3, np.float32))

    def parts(self):
        return [np.array(x) for x in unpack(self.pool.rec)]

    def set_parts(self, parts):
        self.pool.rec = pack(*parts)
        self.pool.push()

    def launch(self, stream=None):
        n, p = self.nova, self.pool
        if self.decode:
            n.launch_attn_decode_q4_batch(self.dq.ptr, p.dev.ptr, self.dt.ptr, self.table.shape[1], self.dp.ptr,
                                          len(self.past), self.layer, p.nb, self.o.ptr, self.ws.ptr, stream)
        else:
            n.launch_attn_chunk_q4_batch(self.dq.ptr, p.dev.ptr, self.dt.ptr, self.table.shape[1], self.dp.ptr,
                                         self.doff.ptr if self.offsets else None, len(self.past), self.n_rows, self.max_q,
                                         self.layer, p.nb, self.o.ptr, self.ws.ptr, stream)

    def result(self):
        return self.o.numpy(self.q.shape, np.float32)

    def run(self):
        self.launch()
        self.nova.dev_sync()
        return self.result()

    def check(self, what=""):
        got, worst = self.result(), 0.0
        for i, n in enumerate(self.count):
            a, b = int(self.off[i]), int(self.off[i + 1])
            if n == 0:
                continue
            k, v = values(self.pool.rec, self.table[i], int(self.keys[i]))
            first = int(self.past[i]) + (0 if self.decode else 1)
            ref, tol = attention(self.q[a:b], k, v, first, self.nova.group)
            worst = max(worst, assert_within(got[a:b], ref, tol, f"{what}, session {i}: {n} rows behind {self.past[i]}"))
        assert (got[self.off[-1]:] == 3).all(), f"{what}: rows behind the last sequence were written"
        print(f"  {worst:.3f} of the bound", flush=True)
        return worst
