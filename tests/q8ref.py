"""The 8-bit page format and the operators over it in numpy, in 64 bits, from
their definitions (include/nova_kernel.h): packing, the quantiser, attention."""
from __future__ import annotations

import numpy as np

KB, HD, REC = 16, 128, 4224


def quantise(x):
    """(codes int8, scales fp32) of rows x [..., 128] fp32.  The quotient of two
    fp32 numbers is never so near to the middle of two codes that its float64
    rounding could land on it, so rint of it is the exact quotient's."""
    x = np.asarray(x, np.float32)
    top = np.abs(x).max(-1)                        # NaN propagates
    with np.errstate(all="ignore"):
        s = (top.astype(np.float64) / 127.0).astype(np.float32)
        s = np.minimum(s, np.float32(float.fromhex("0x1.020406p+121")))    # 127 s stays finite
        s = np.where(np.isfinite(top), np.where(s >= np.float32(2.0 ** -126), s, np.float32(0)), np.float32(np.nan))
        live = s > 0
        c = np.rint(x.astype(np.float64) / np.where(live, s, 1).astype(np.float64)[..., None])
    c = np.where(live[..., None], c, 0)
    return c.astype(np.int8), s.astype(np.float32)


def pack(kc, ks, vc, vs):
    """records [..., 4224] uint8 of pages kc, vc [..., 16, 128] int8, ks, vs [..., 16] fp32"""
    lead = kc.shape[:-2]
    rec = np.empty(lead + (REC,), np.uint8)
    k = kc.reshape(lead + (4, 4, 8, 16))
    rec[..., :2048] = np.swapaxes(k, -2, -3).reshape(lead + (2048,)).view(np.uint8)
    rec[..., 2048:4096] = np.ascontiguousarray(np.swapaxes(vc, -1, -2)).reshape(lead + (2048,)).view(np.uint8)
    rec[..., 4096:4160] = np.ascontiguousarray(ks, np.float32).view(np.uint8)
    rec[..., 4160:] = np.ascontiguousarray(vs, np.float32).view(np.uint8)
    return rec


def unpack(rec):
    lead = rec.shape[:-1]
    k = np.ascontiguousarray(rec[..., :2048]).view(np.int8).reshape(lead + (4, 8, 4, 16))
    kc = np.swapaxes(k, -2, -3).reshape(lead + (16, 128))
    v = np.ascontiguousarray(rec[..., 2048:4096]).view(np.int8).reshape(lead + (128, 16))
    ks = np.ascontiguousarray(rec[..., 4096:4160]).view(np.float32)
    vs = np.ascontiguousarray(rec[..., 4160:]).view(np.float32)
    return kc, ks, np.swapaxes(v, -1, -2), vs


class Q8Pool:
    """Random 8-bit pages of one layer on the device and on the host.  Pages lie
    anywhere in the pool; the other layers are device memory nobody touched."""

    def __init__(self, nova, nb, layer, seed, v_tokens=None):
        self.nova, self.nb, self.layer = nova, nb, layer
        self.rng = rng = np.random.default_rng(seed)
        self.page = nova.nkv * REC
        assert nova.kv_q8_page_bytes() == self.page
        self.dev = nova.alloc((layer + 1) * nb * self.page)
        # keys with a few strong channels and uneven tokens, as projections give
        gain = np.ones(HD, np.float32)
        gain[rng.permutation(HD)[:4]] = 5
        tok = np.exp(0.25 * rng.standard_normal((nb, nova.nkv, KB, 1))).astype(np.float32)
        self.k = rng.standard_normal((nb, nova.nkv, KB, HD)).astype(np.float32) * gain * tok
        self.v = rng.standard_normal((nb, nova.nkv, KB, HD)).astype(np.float32) * tok[:, :, ::-1]
        self.rec = pack(*quantise(self.k), *quantise(self.v))
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
        """NaN scales and loud codes in every slot of the sessions' last pages that
        holds no key."""
        for i, n in enumerate(n_keys):
            if n % KB:
                r = self.rec[table[i, n // KB]]
                kc, ks, vc, vs = (np.array(x) for x in unpack(r))
                kc[:, n % KB:], vc[:, n % KB:] = -128, 127
                ks[:, n % KB:], vs[:, n % KB:] = np.nan, np.inf
                self.rec[table[i, n // KB]] = pack(kc, ks, vc, vs)
        self.push()


def values(rec, table, n):
    """K, V [n][NKV][128] float64 of a session's first n tokens"""
    pos = np.arange(n)
    kc, ks, vc, vs = unpack(rec)
    k = kc.astype(np.float64) * ks[..., None].astype(np.float64)
    v = vc.astype(np.float64) * vs[..., None].astype(np.float64)
    return (k[table[pos >> 4], :, pos & 15], v[table[pos >> 4], :, pos & 15])


def attention(q, k, v, first, group):
    """Rows q [n][NH][128] over k, v [T][NKV][128] float64, row r seeing keys
    [0, first + r); and how far an fp32 result may be from it, per output row.

    The bound: a score is a sum of 128 products in fp32 (or of exact integer
    products against q kept to 2^-23 of its largest component), whose roundings
    add up like a random walk to at most sqrt(128) * 2^-24 < 2^-20 of
    sum |q_d k_d| + max|q| sum |k_d|: that is the score's error d.  Weights carry
    d, 2^-20 from exp2, scaling and their split, and the sums over n keys run
    through chains of at most n / 32 + 64 additions of 2^-24.  With weights off by
    e relatively, the normalised sum is off by at most 2 e max|v|."""
    n, nh, _ = q.shape
    out, tol = np.zeros((n, nh, HD)), np.zeros((n, nh, 1))
    if len(k) == 0:
        return out, tol
    for h in range(nh):
        kh, vh = k[:, h // group], v[:, h // group]
        x = q[:, h].astype(np.float64)
        s = x @ kh.T / np.sqrt(HD)
        size = (np.abs(x) @ np.abs(kh).T + np.abs(x).max(-1, keepdims=True) * np.abs(kh).sum(-1)) / np.sqrt(HD)
        seen = np.arange(len(kh))[None, :] < np.minimum(first + np.arange(n), len(kh))[:, None]
        s = np.where(seen, s, -np.inf)
        with np.errstate(invalid="ignore"):
            p = np.exp(s - s.max(-1, keepdims=True))
            o = np.where(seen.any(-1)[:, None], (p @ vh) / p.sum(-1, keepdims=True), 0)
        out[:, h] = o
        e = 2.0 ** -20 * np.where(seen, size, 0).max(-1) + 2.0 ** -20 + (len(kh) / 32 + 64) * 2.0 ** -24
        tol[:, h, 0] = 2 * e * np.abs(vh).max()
    return out, tol


def assert_within(got, ref, tol, what):
    assert np.isfinite(got).all(), f"{what}: not finite"
    err = np.abs(got.astype(np.float64) - ref)
    worst = (err / np.maximum(tol, 1e-30)).max(initial=0)
    assert (err <= tol).all(), f"{what}: {worst:.2f} of the bound, max abs {err.max():.3e}"
    return worst


def attention_by_row(q, k, v, v_scale, first, group):
    """The formula as in `attention`, and a bound that is each row's own: only keys
    that the row sees enter it, with their weights.

    e is the relative error of a weight as derived there.  An output element is
    sum p_j v_j, so weights off by e move it by at most 2 e sum p_j |v_j|, taken per
    element.  A weight times its value's scale is also rounded to a fixed step: two fp16
    terms, cut below 2^-24, where the row's largest such product stands at 2^6 or
    more, so each of n keys adds up to 2^-30 of the largest p_j times its value's
    largest component (127 scales).  v_scale: the scales [T][NKV]."""
    n, nh, _ = q.shape
    out, tol = np.zeros((n, nh, HD)), np.zeros((n, nh, HD))
    for h in range(nh):
        kh, vh, sh = k[:, h // group], v[:, h // group], v_scale[:, h // group].astype(np.float64)
        for r in range(n):
            m = min(first + r, len(kh))
            x = q[r, h].astype(np.float64)
            s = kh[:m] @ x / np.sqrt(HD)
            size = (np.abs(kh[:m]) @ np.abs(x) + np.abs(x).max() * np.abs(kh[:m]).sum(-1)) / np.sqrt(HD)
            p = np.exp(s - s.max())
            p /= p.sum()
            e = 2.0 ** -20 * size.max() + 2.0 ** -20 + (m / 32 + 64) * 2.0 ** -24
            out[r, h] = p @ vh[:m]
            tol[r, h] = 2 * e * (p @ np.abs(vh[:m])) + m * 2.0 ** -30 * 127 * (p * sh[:m]).max()
    return out, tol
