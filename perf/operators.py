"""The operators of the 8-bit paged KV cache: inputs, plain forms, calls and exact results.

The cache holds K and V as int8 codes with one fp32 scale per token and kv head.
A page (16 tokens of one layer) is a record of 4224 bytes per kv head:

    K code of token t, dim d   byte (t >> 2) * 512 + (d >> 4) * 64 + (t & 3) * 16 + (d & 15)
    V code of token t, dim d   byte 2048 + d * 16 + t
    K scale of token t         fp32 at byte 4096 + 4 t
    V scale of token t         fp32 at byte 4160 + 4 t

and the pool is [layer][page][kv head][4224].  Four kinds of case:

* ``store``   quantise the rows of every session as they are written into its
  pages, and read the same rows back (the outputs: the values the codes stand for).
* ``decode``  one query token per session over all of its keys.
* ``chunk``   a ragged chunk of new tokens per session (already in the cache) over
  its prefix and itself, causally.
* ``cow``     the page copies and block-table patches of forked sessions.

Lengths are drawn with the case's own ``mix``, so every seed does the same amount
of work; pages are scattered over the pool by a seeded shuffle.
"""
import ctypes
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

KB = 16                      # tokens per page
HD = 128
REC = 4224                   # bytes per page and kv head
# query heads, kv heads, layers
MODELS = {"qwen25_1p5b": (12, 2, 28), "qwen25_7b": (28, 4, 28), "qwen25_14b": (40, 8, 48)}
LAYER, LAYERS = 1, 2         # the attention and store cases run on the second layer of two


def listed():
    return [
        # a decode step's appends: one token of each of 16 sessions
        dict(name="store_7b_step", kind="store", model="qwen25_7b", sessions=16, q_lo=1, q_hi=1, past_lo=511,
             past_hi=8191, mix=2024),
        # the appends of the chunked prefill benchmark: 8 sessions x 512 tokens
        dict(name="store_7b_chunk", kind="store", model="qwen25_7b", sessions=8, q_lo=512, q_hi=512, past_lo=0,
             past_hi=4096, mix=2024),
        # one user, the small model, a chat of 1025 tokens: latency and launches
        dict(name="decode_1p5b_single", kind="decode", model="qwen25_1p5b", sessions=1, ctx_lo=1025, ctx_hi=1025, mix=1),
        # many short chats at once
        dict(name="decode_7b_short_chats", kind="decode", model="qwen25_7b", sessions=24, ctx_lo=17, ctx_hi=600, mix=7),
        # the benchmark's own step: a ragged batch of 16 sessions
        dict(name="decode_7b_ragged16", kind="decode", model="qwen25_7b", sessions=16, ctx_lo=512, ctx_hi=8192,
             mix=2024),
        # long documents on the large model
        dict(name="decode_14b_long", kind="decode", model="qwen25_14b", sessions=8, ctx_lo=32768, ctx_hi=32768, mix=1),
        # drafted tokens to be checked: 1 to 8 rows per session behind the same contexts
        dict(name="chunk_7b_drafts", kind="chunk", model="qwen25_7b", sessions=16, q_lo=1, q_hi=8, past_lo=512,
             past_hi=8192, mix=2024),
        # prompts of unequal lengths on the small model, some of them follow-ups
        dict(name="chunk_1p5b_mixed", kind="chunk", model="qwen25_1p5b", sessions=12, q_lo=1, q_hi=300, past_lo=0,
             past_hi=700, mix=5),
        # a follow-up question behind a long document on the large model
        dict(name="chunk_14b_followup", kind="chunk", model="qwen25_14b", sessions=1, q_lo=300, q_hi=300,
             past_lo=12001, past_hi=12001, mix=1),
        # the benchmark's chunked prefill: 8 sessions x 512 tokens over ragged prefixes
        dict(name="chunk_7b_batch", kind="chunk", model="qwen25_7b", sessions=8, q_lo=512, q_hi=512, past_lo=0,
             past_hi=4096, mix=2024),
        # one forked session of the small model writes its first token
        dict(name="cow_1p5b_one", kind="cow", model="qwen25_1p5b", children=1, donors=1),
        # 64 sessions forked from 4 prompts write their first token
        dict(name="cow_7b_fork", kind="cow", model="qwen25_7b", children=64, donors=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges: any model, sizes spread over their logarithm."""
    model = rng.choice(sorted(MODELS))
    nh, nkv, _ = MODELS[model]
    kind = rng.choice(["store"] * 2 + ["decode"] * 4 + ["chunk"] * 4 + ["cow"])
    mix = rng.randrange(1 << 20)
    if kind == "cow":
        children = _log(rng, 1, 64)
        # a 14B page is four times a 7B one over all layers
        children = max(1, children // (4 if model == "qwen25_14b" else 1))
        return dict(kind="cow", model=model, children=children, donors=rng.randint(1, children), mix=mix)
    sessions = _log(rng, 1, 32)
    if kind == "decode":
        hi = _log(rng, 1, 32768)
        lo = rng.randint(max(1, hi // 16), hi)
        while sessions > 1 and sessions * hi * nkv * 264 > 5.0e8:
            sessions -= 1
        return dict(kind="decode", model=model, sessions=sessions, ctx_lo=lo, ctx_hi=hi, mix=mix)
    q_hi = _log(rng, 1, 1024)
    q_lo = rng.choice([q_hi, rng.randint(1, q_hi), 1])
    hi = _log(rng, 1, 16384)
    lo = rng.choice([0, rng.randint(0, hi), hi])
    if kind == "store":
        while sessions > 1 and sessions * q_hi * nkv > 8 * 512 * 4:
            sessions -= 1
        return dict(kind="store", model=model, sessions=sessions, q_lo=q_lo, q_hi=min(q_hi, 8 * 512 * 4 // nkv),
                    past_lo=lo, past_hi=hi, mix=mix)
    while sessions > 1 and sessions * q_hi * nh * (hi + q_hi) > 2.2e8:
        sessions -= 1
    while q_hi > 1 and sessions * q_hi * nh * (hi + q_hi) > 2.2e8:
        q_hi //= 2
    return dict(kind="chunk", model=model, sessions=sessions, q_lo=min(q_lo, q_hi), q_hi=q_hi, past_lo=lo, past_hi=hi,
                mix=mix)


# ------------------------------------------------------------------ inputs

class _State:
    """What a serving program holds before the call."""


def _lengths(n, lo, hi, mix):
    return np.random.default_rng(mix).integers(lo, hi + 1, n).astype(np.int64)


def _shape(case):
    """(keys before the call, rows of the call) per session."""
    n = case["sessions"]
    if case["kind"] == "decode":
        return _lengths(n, case["ctx_lo"], case["ctx_hi"], case["mix"]), np.ones(n, np.int64)
    return (_lengths(n, case["past_lo"], case["past_hi"], case["mix"]),
            _lengths(n, case["q_lo"], case["q_hi"], case["mix"] + 1))


def _dev(array):
    return torch.from_numpy(np.ascontiguousarray(array)).cuda()


def _normal(g, shape, scale=1.0):
    return torch.empty(shape, device="cuda").normal_(0.0, scale, generator=g)


def _rows(g, shape):
    """K rows as they come out of a projection: a few channels are several times the others, and tokens differ."""
    gain = torch.ones(shape[-1], device="cuda")
    gain[torch.randperm(shape[-1], generator=g, device="cuda")[:4]] = 5.0
    tok = torch.exp(_normal(g, shape[:-1] + (1,), 0.25))
    return _normal(g, shape) * gain * tok


def _fill(pool, g, nkv):
    """Random pages for one layer's records [nb][NKV][REC], as an append would have left them."""
    nb = pool.shape[0]
    x = _rows(g, (nb, nkv, KB, HD))
    d = (x.abs().amax(-1) / 127.0)
    c = torch.round(x / d[..., None]).to(torch.int8)
    pool[..., :2048] = c.view(nb, nkv, 4, 4, 8, 16).transpose(3, 4).reshape(nb, nkv, 2048).view(torch.uint8)
    pool[..., 4096:4160] = d.contiguous().view(torch.uint8)
    x = _normal(g, (nb, nkv, KB, HD)) * torch.exp(_normal(g, (nb, nkv, KB, 1), 0.25))
    d = (x.abs().amax(-1) / 127.0)
    c = torch.round(x / d[..., None]).to(torch.int8)
    pool[..., 2048:4096] = c.transpose(2, 3).reshape(nb, nkv, 2048).view(torch.uint8)
    pool[..., 4160:] = d.contiguous().view(torch.uint8)


def prepare(case, seed):
    s = _State()
    s.case = case
    nh, nkv, n_layers = MODELS[case["model"]]
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    if case["kind"] == "cow":
        n = case["children"]
        order = np.random.default_rng(seed).permutation(case["donors"] + n).astype(np.int32)
        s.nb = len(order)
        s.pool = torch.zeros((n_layers, s.nb, nkv, REC), dtype=torch.uint8, device="cuda")
        for layer in range(n_layers):
            _fill(s.pool[layer], g, nkv)
        # the session manager's decisions: copy page src to dst, then table entry index = dst
        s.ops = np.zeros(n, np.dtype([("src", "<i4"), ("dst", "<i4"), ("index", "<i8")]))
        s.ops["src"] = order[np.arange(n) % case["donors"]]
        s.ops["dst"] = order[case["donors"]:]
        s.ops["index"] = np.arange(n) * 3 + 1
        s.table = torch.zeros(3 * n, dtype=torch.int32, device="cuda")
        return s
    past, rows = _shape(case)
    keys = past if case["kind"] == "decode" else past + rows
    pages = (keys + KB - 1) // KB
    s.nb, s.stride = int(pages.sum()) + 8, int(pages.max())
    perm = np.random.default_rng(seed).permutation(s.nb).astype(np.int32)
    table = np.zeros((len(pages), s.stride), np.int32)
    for i, p in enumerate(pages):
        off = int(pages[:i].sum())
        table[i, :p] = perm[off:off + p]
    s.table = _dev(table)
    s.n = len(pages)
    s.n_rows, s.max_q = int(rows.sum()), int(rows.max())
    s.past = _dev(past.astype(np.int32))                    # decode: the keys of each session
    s.row_off = _dev(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32))
    s.pool = torch.zeros((LAYERS, s.nb, nkv, REC), dtype=torch.uint8, device="cuda")
    if case["kind"] == "store":
        s.k, s.v = _rows(g, (s.n_rows, nkv, HD)), _normal(g, (s.n_rows, nkv, HD))
        s.k_out, s.v_out = torch.empty_like(s.k), torch.empty_like(s.v)
    else:
        _fill(s.pool[LAYER], g, nkv)
        # post-RoPE queries are not unit scale: scores spread over several units
        s.q = _normal(g, (s.n_rows, nh, HD), 1.5)
        s.o = torch.empty_like(s.q)
    return s


# ------------------------------------------------------------------ passes

def run(s):
    if own:
        return _own(s)
    return {"store": _plain_store, "decode": _plain_attention, "chunk": _plain_attention, "cow": _plain_cow}[
        s.case["kind"]](s)


_WORKSPACE = {}


def _workspace(nbytes):
    """One workspace for the calls of each stream, as long as it is large enough: calls on two streams may overlap.
    A larger one takes its place in the stream's own order (it is allocated on that stream)."""
    stream = torch.cuda.current_stream()
    key = stream.device_index, stream.cuda_stream
    if key not in _WORKSPACE or _WORKSPACE[key].numel() < nbytes:
        _WORKSPACE[key] = torch.empty(nbytes, dtype=torch.uint8, device=stream.device)
    return _WORKSPACE[key].data_ptr()


_LIBRARY = {}


def _library(model):
    """The package and a model's library, loaded once per program."""
    if model not in _LIBRARY:
        path = str(Path(__file__).resolve().parent.parent / "conflux-nova_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import nova_amd
        _LIBRARY[model] = nova_amd, nova_amd.load(model)
    return _LIBRARY[model]


def _own(s):
    nova_amd, nova = _library(s.case["model"])
    st = torch.cuda.current_stream().cuda_stream
    kind = s.case["kind"]
    if kind == "cow":
        nova.launch_kv_q8_cow_apply(s.pool.data_ptr(), s.nb, s.table.data_ptr(),
                                    ctypes.cast(s.ops.ctypes.data, ctypes.POINTER(nova_amd.CowOp)), len(s.ops), st)
        return s.pool, s.table
    pool, table, past = s.pool.data_ptr(), s.table.data_ptr(), s.past.data_ptr()
    if kind == "store":
        off = s.row_off.data_ptr()
        nova.launch_kv_q8_store_batch(pool, table, s.stride, past, off, s.n, s.n_rows, LAYER, s.nb, s.k.data_ptr(),
                                      s.v.data_ptr(), st)
        nova.launch_kv_q8_load_batch(pool, table, s.stride, past, off, s.n, s.n_rows, LAYER, s.nb, s.k_out.data_ptr(),
                                     s.v_out.data_ptr(), st)
        return s.k_out, s.v_out
    if kind == "decode":
        ws = _workspace(nova.attn_decode_q8_workspace_bytes(s.n))
        nova.launch_attn_decode_q8_batch(s.q.data_ptr(), pool, table, s.stride, past, s.n, LAYER, s.nb, s.o.data_ptr(),
                                         ws, st)
    else:
        ws = _workspace(nova.attn_chunk_q8_workspace_bytes(s.n, s.n_rows, s.max_q))
        nova.launch_attn_chunk_q8_batch(s.q.data_ptr(), pool, table, s.stride, past, s.row_off.data_ptr(), s.n,
                                        s.n_rows, s.max_q, LAYER, s.nb, s.o.data_ptr(), ws, st)
    return s.o


def _row_places(s):
    """(page, slot) of every row of the call."""
    row = torch.arange(s.n_rows, device="cuda")
    sess = torch.searchsorted(s.row_off[1:].long(), row, right=True)
    pos = s.past.long()[sess] + row - s.row_off.long()[sess]
    return s.table[sess, pos // KB].long(), pos % KB


def _plain_store(s):
    layer = s.pool[LAYER]
    page, slot = _row_places(s)
    nkv = layer.shape[1]
    d = torch.arange(HD, device="cuda")
    head = torch.arange(nkv, device="cuda")[None, :, None]
    k_at = (slot // 4)[:, None] * 512 + (d // 16) * 64 + (slot % 4)[:, None] * 16 + d % 16
    v_at = 2048 + d * 16 + slot[:, None]
    out = []
    for x, at, scale_at in ((s.k, k_at, 4096), (s.v, v_at, 4160)):
        a = x.abs().amax(-1)
        scale = (a.double() / 127.0).float()
        scale = torch.where(scale < 2.0 ** -126, torch.zeros_like(scale), scale)
        code = torch.round(x.double() / scale.double()[..., None])
        code = torch.where(scale[..., None] > 0, code, torch.zeros_like(code)).to(torch.int8)
        layer[page[:, None, None], head, at[:, None, :]] = code.view(torch.uint8)
        four = scale_at + 4 * slot[:, None] + torch.arange(4, device="cuda")
        layer[page[:, None, None], head, four[:, None, :]] = scale.view(torch.uint8).view(scale.shape + (4,))
        # read back from the pages
        got = layer[page[:, None, None], head, at[:, None, :]].view(torch.int8).float()
        got_scale = layer[page[:, None, None], head, four[:, None, :]].view(torch.float32)
        out.append(got * got_scale)
    return tuple(out)


def _plain_attention(s):
    nh, nkv, _ = MODELS[s.case["model"]]
    group = nh // nkv
    n, t = s.n, s.stride * KB
    rec = s.pool[LAYER][s.table.long()]                                    # [n][pages][NKV][REC]
    rec = rec.transpose(1, 2)                                              # [n][NKV][pages][REC]
    k = rec[..., :2048].view(torch.int8).view(n, nkv, s.stride, 4, 8, 4, 16).transpose(4, 5).reshape(n, nkv, t, HD)
    k = k.float() * rec[..., 4096:4160].contiguous().view(torch.float32).reshape(n, nkv, t, 1)
    v = rec[..., 2048:4096].view(torch.int8).view(n, nkv, s.stride, HD, KB).transpose(3, 4).reshape(n, nkv, t, HD)
    v = v.float() * rec[..., 4160:].contiguous().view(torch.float32).reshape(n, nkv, t, 1)
    # the rows of each session, padded to the longest chunk
    row = torch.arange(s.n_rows, device="cuda")
    sess = torch.searchsorted(s.row_off[1:].long(), row, right=True)
    at = row - s.row_off.long()[sess]
    q = torch.zeros((n, s.max_q, nh, HD), device="cuda")
    q[sess, at] = s.q
    q = q.view(n, s.max_q, nkv, group, HD).transpose(1, 2).reshape(n, nkv, s.max_q * group, HD)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(HD))
    seen = s.past.long()[:, None] + (torch.arange(s.max_q, device="cuda") + 1 if s.case["kind"] == "chunk" else 0)
    seen = seen.expand(n, s.max_q)
    hidden = torch.arange(t, device="cuda") >= seen[:, :, None]            # [n][max_q][t]
    score = score.view(n, nkv, s.max_q, group, t).masked_fill_(hidden[:, None, :, None, :], -math.inf)
    score -= score.amax(-1, keepdim=True)
    score.exp_()
    score /= score.sum(-1, keepdim=True)
    o = torch.matmul(score.view(n, nkv, s.max_q * group, t), v)
    o = o.view(n, nkv, s.max_q, group, HD).transpose(1, 2).reshape(n, s.max_q, nh, HD)
    return o[sess, at]


def _plain_cow(s):
    src, dst, at = (_dev(s.ops[f].astype(np.int64)) for f in ("src", "dst", "index"))
    s.pool[:, dst] = s.pool[:, src]
    s.table[at] = dst.to(torch.int32)
    return s.pool, s.table


# ------------------------------------------------------------------ work and exact results

def work(case):
    nh, nkv, n_layers = MODELS[case["model"]]
    if case["kind"] == "cow":
        # a page copied is read and written once; donors shared by children are read once
        pages = case["children"] + min(case["donors"], case["children"])
        return {"bytes": pages * n_layers * nkv * REC, "flops": 0}
    past, rows = _shape(case)
    n_rows = int(rows.sum())
    if case["kind"] == "store":
        # fp32 rows in, codes and scales written, the values out again
        return {"bytes": 2 * n_rows * nkv * (4 * HD + 2 * (HD + 4) + 4 * HD), "flops": 0}
    if case["kind"] == "decode":
        keys, pairs = int(past.sum()), int(past.sum())
    else:
        keys = int((past + rows).sum())
        pairs = int((rows * past + rows * (rows + 1) // 2).sum())
    return {"bytes": keys * nkv * 2 * (HD + 4) + 2 * n_rows * nh * HD * 4, "flops": 4.0 * HD * nh * pairs}


def exact(case, seed):
    """From the definitions, in 64 bits, byte by byte through the page format."""
    if case["kind"] == "cow":
        return None
    s = prepare(case, seed)
    if case["kind"] == "store":
        out = []
        for x in (s.k.double(), s.v.double()):
            top = x.abs().max(dim=2).values
            step = (top / 127).to(torch.float32).to(torch.float64)         # the scale is kept in fp32
            code = torch.where(step[:, :, None] >= 2.0 ** -126, (x / step[:, :, None]).round(), x * 0)
            out.append(code * step[:, :, None])
        return tuple(out)
    nh, nkv, _ = MODELS[case["model"]]
    group = nh // nkv
    past, rows = _shape(case)
    d = torch.arange(HD, device="cuda")
    o = torch.zeros((s.n_rows, nh, HD), dtype=torch.float64, device="cuda")
    flat = s.pool[LAYER].reshape(-1)
    first = 0
    for i in range(s.n):
        n_q = int(rows[i])
        n_keys = int(past[i]) + (n_q if case["kind"] == "chunk" else 0)
        tok = torch.arange(n_keys, device="cuda")
        page, slot = s.table[i].long()[tok // KB], tok % KB
        for h in range(nkv):
            base = (page * nkv + h) * REC
            k_at = base[:, None] + ((slot >> 2) * 512 + (slot & 3) * 16)[:, None] + (d >> 4) * 64 + (d & 15)
            k = flat[k_at].view(torch.int8).double()
            v = flat[base[:, None] + 2048 + slot[:, None] + d * 16].view(torch.int8).double()
            four = torch.arange(4, device="cuda")
            ks = flat[(base + 4096 + 4 * slot)[:, None] + four].view(torch.float32).double()
            vs = flat[(base + 4160 + 4 * slot)[:, None] + four].view(torch.float32).double()
            q = s.q[first:first + n_q, h * group:(h + 1) * group].reshape(n_q * group, HD).double()
            score = (q @ (k * ks).T) / math.sqrt(HD)
            if case["kind"] == "chunk":
                limit = past[i] + torch.arange(n_q, device="cuda").repeat_interleave(group)
                score[tok[None, :] > limit[:, None]] = -math.inf
            p = torch.softmax(score, dim=1)
            o[first:first + n_q, h * group:(h + 1) * group] = (p @ (v * vs)).view(n_q, group, HD)
        first += n_q
    return o
