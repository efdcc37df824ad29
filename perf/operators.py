"""Performance cases of the paged K/V cache's operators: the rows of new tokens put into pages, and the gated GQA
attention of one new token or of chunks of new tokens over paged rows, at the attention shapes of the 4B-class
configuration (16 q heads on 4 kv heads of 256, 64 rotated dims) and, in drawn cases, other head counts the tests hold.

Kinds of case:
  append   K (rotated, normed) and V rows of new tokens of n sequences into their pages
  decode   one new token of each of n sequences over its paged rows
  prefill  chunks of new tokens of n sequences over their paged rows

Sequence i holds `rows` cached rows (fewer, unequally many, where `ragged`) and brings `tokens` new ones (likewise); its
pages of `page` rows lie in a random order in the pool, whose free pages and unwritten rows hold other conversations'
stale values.  `half` is a cache of 16-bit floats, else of 32-bit ones; a row is rounded to it once.

Streams: the library works on its context's own stream, which does not wait for torch's nor torch's for it.  prepare()
waits for the card before it takes memory that an earlier state's calls may still read, and after it has made the
inputs; run() enqueues, as a serving loop does, whose calls follow each other on that stream, and whoever takes its
outputs elsewhere synchronises first.

Where `own` is false, run() computes the same with elementary torch operations: 32 bits, with 64 for the rotation and
the norm (whose K rows are rounded to 16 bits).  Where it is true it calls the library's front end, on buffers of the
same shape and contents.
"""
import ctypes
import math
import os
import sys

import numpy as np
import torch

own = False

EPS = 1e-6
HD, ROPE_DIM, ROPE_BASE = 256, 64, 1e7


def listed():
    a = {"nh": 16, "nkv": 4}
    return [
        # The smallest call: one token's rows of a conversation, as after a drafter's step.
        {"name": "append_1", "kind": "append", "half": True, "n": 1, "rows": 4000, "tokens": 1, "ragged": False, "page": 64, **a},
        # A 2048-token prompt in the last attention layer, where all but the last token need their rows only.
        {"name": "append_2048", "kind": "append", "half": True, "n": 1, "rows": 0, "tokens": 2048, "ragged": False, "page": 64, **a},
        # Prompts of six users at once, full precision, small pages.
        {"name": "append_6_f32", "kind": "append", "half": False, "n": 6, "rows": 1000, "tokens": 1300, "ragged": True, "page": 16, **a},
        # One conversation of 8K tokens.
        {"name": "decode_8k", "kind": "decode", "half": True, "n": 1, "rows": 8191, "tokens": 1, "ragged": False, "page": 64, **a},
        # A full batch of ordinary conversations of unequal lengths, small pages.
        {"name": "decode_64", "kind": "decode", "half": True, "n": 64, "rows": 4000, "tokens": 1, "ragged": True, "page": 16, **a},
        # Eight long conversations in the full-precision cache.
        {"name": "decode_8x32k_f32", "kind": "decode", "half": False, "n": 8, "rows": 32639, "tokens": 1, "ragged": True, "page": 256, **a},
        # The first tokens of three short conversations: latency.
        {"name": "decode_short_f32", "kind": "decode", "half": False, "n": 3, "rows": 77, "tokens": 1, "ragged": True, "page": 16, **a},
        # A 2048-token prompt from an empty cache.
        {"name": "prefill_2048", "kind": "prefill", "half": True, "n": 1, "rows": 0, "tokens": 2048, "ragged": False, "page": 64, **a},
        # A chunk of a long prompt over 16K rows.
        {"name": "prefill_512_16k", "kind": "prefill", "half": True, "n": 1, "rows": 16000, "tokens": 512, "ragged": False, "page": 64, **a},
        # A mixed batch of a server: a prompt's chunk beside short turns of other conversations, odd sizes.
        {"name": "prefill_mixed", "kind": "prefill", "half": True, "n": 6, "rows": 5000, "tokens": 307, "ragged": True, "page": 16, **a},
        # The next user turn of a conversation, full precision.
        {"name": "prefill_133_8k_f32", "kind": "prefill", "half": False, "n": 1, "rows": 8000, "tokens": 133, "ragged": False, "page": 16, **a},
        # A medium prompt, full precision.
        {"name": "prefill_1000_f32", "kind": "prefill", "half": False, "n": 1, "rows": 0, "tokens": 1000, "ragged": False, "page": 64, **a},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    """One more case: sizes spread over their logarithm, no dearer than the largest listed one of its kind."""
    kind = rng.choice(["append", "decode", "decode", "prefill", "prefill"])
    nh, nkv = rng.choice([(16, 4), (16, 4), (16, 4), (8, 4), (16, 2), (4, 4)])
    c = {"kind": kind, "half": rng.random() < 0.6, "ragged": rng.random() < 0.5, "page": rng.choice([16, 16, 32, 64, 128, 256]),
         "nh": nh, "nkv": nkv}
    if kind == "append":
        n = _log_int(rng, 1, 16)
        return {**c, "n": n, "rows": rng.randint(0, 3000), "tokens": _log_int(rng, 1, 2048 // n)}
    if kind == "decode":
        n = _log_int(rng, 1, 64)
        return {**c, "n": n, "rows": _log_int(rng, 1, min(32639, 200000 // n)), "tokens": 1}
    n = _log_int(rng, 1, 8)
    rows = 0 if rng.random() < 0.4 else _log_int(rng, 16, 16000 // n)
    top = 2048 // n            # n T (rows + T / 2) within that of a 2048-token prompt
    while top > 2 and n * top * (rows + top / 2) > 2048 * 1024:
        top -= 1
    return {**c, "n": n, "rows": rows, "tokens": _log_int(rng, 1, top)}


def _lens(case):
    """Cached rows of each sequence: equal, or falling to about a third of the first."""
    n, rows = case["n"], case["rows"]
    return [rows - (2 * i * rows) // (3 * n) if case["ragged"] else rows for i in range(n)]


def _counts(case):
    """New tokens of each sequence: equal, or falling with the square of the place, one at least."""
    n, t = case["n"], case["tokens"]
    return [max(1, t * (n - i) ** 2 // n ** 2) if case["ragged"] else t for i in range(n)]


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(0x51356000 + seed)
    return g


def _normal(g, *shape, mean=0.0, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std + mean


def _freqs():
    """The rotation's frequencies 1 / base^(i / 32), each operation in 32 bits."""
    m = ctypes.CDLL("libm.so.6")
    m.powf.restype, m.powf.argtypes = ctypes.c_float, [ctypes.c_float, ctypes.c_float]
    half = ROPE_DIM // 2
    return np.array([np.float32(1) / np.float32(m.powf(ROPE_BASE, np.float32(i) / np.float32(half))) for i in range(half)],
                    np.float32)


def _layout(case, seed):
    """(lens, counts, pages a sequence needs at most, pages of the pool, the table [n][pages] on the host)."""
    lens, counts = _lens(case), _counts(case)
    per = max(-(-(a + b) // case["page"]) for a, b in zip(lens, counts))
    pool = case["n"] * per + 7
    order = np.random.RandomState(seed % (1 << 31)).permutation(pool)[:case["n"] * per]
    return lens, counts, per, pool, order.reshape(case["n"], per).astype(np.int32)


def _inputs(case, seed):
    g = _gen(seed)
    lens, counts, per, pool, table = _layout(case, seed)
    rows = sum(counts)
    x = {"k": _normal(g, rows, case["nkv"] * HD), "v": _normal(g, rows, case["nkv"] * HD),
         "q_norm": _normal(g, HD, mean=1.0, std=0.02), "k_norm": _normal(g, HD, mean=1.0, std=0.02)}
    if case["kind"] != "append":
        x["q_gate"] = _normal(g, rows, 2 * case["nh"] * HD)
    return x, lens, counts, per, pool, table


def _fill(g, pages):
    """The pool's contents: normal values, in pieces (the conversations' cached rows and stale ones alike)."""
    flat = pages.view(-1)
    step = 1 << 26
    for at in range(0, flat.numel(), step):
        part = flat[at:at + step]
        part.copy_(torch.randn(part.numel(), generator=g, device="cuda", dtype=torch.float32))


class _Foreign:
    """Memory of the library's cache as torch takes it; it lives as long as its owner."""

    def __init__(self, owner, ptr, shape, half):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": tuple(shape), "strides": None, "typestr": "<f2" if half else "<f4",
                                         "data": (ptr, False), "version": 2}


class _Owner:
    """A context and its paged cache, closed once neither the state nor a view of their memory is left."""

    def __init__(self, case, x, lens, counts, per, pool, table):
        here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3.5sharp_amd")
        if here not in sys.path:
            sys.path.insert(0, here)
        import q35mix
        self.ctx = q35mix.Context(q35mix.qwen35_config(num_layers=1, num_heads=case["nh"], num_kv_heads=case["nkv"],
                                                       is_recurrent=[0]), n_seqs=1, kv_capacity=16)
        self.ctx.set_attn_weights(0, {k: x[k].cpu().numpy() for k in ("q_norm", "k_norm")})
        self.cache = q35mix.PagedCache(self.ctx, n_seqs=case["n"], max_rows=per * case["page"], n_pages=pool,
                                       page_rows=case["page"], kv_type=q35mix.KV_F16 if case["half"] else q35mix.KV_F32)
        for i in range(case["n"]):
            self.cache.map(i, 0, table[i])
        self.cache.advance(list(range(case["n"])), lens)
        self.kinds = (q35mix.STATE_KEYS, q35mix.STATE_VALUES)

    def pages(self, shape, half):
        return [torch.as_tensor(_Foreign(self, self.cache.device_ptr(0, kind)[0], shape, half), device="cuda")
                for kind in self.kinds]

    def __del__(self):
        if hasattr(self, "cache"):
            self.cache.close()
        if hasattr(self, "ctx"):
            self.ctx.close()


class _Buf:
    """A torch tensor as the front end takes device buffers (.ptr)."""

    def __init__(self, t):
        assert t.is_contiguous()
        self.t, self.ptr, self.nbytes = t, t.data_ptr(), t.numel() * t.element_size()


def prepare(case, seed):
    if own:
        torch.cuda.synchronize()
    x, lens, counts, per, pool, table = _inputs(case, seed)
    n, nkv, half = case["n"], case["nkv"], case["half"]
    shape = (pool, nkv, case["page"], HD)
    s = {"case": case, "x": x}
    if own:
        # the library's cache: its pages are its own memory, the tables are set and checked once
        s["owner"] = _Owner(case, x, lens, counts, per, pool, table)
        s["pages"] = s["owner"].pages(shape, half)
    else:
        s["pages"] = [torch.empty(shape, device="cuda", dtype=torch.float16 if half else torch.float32) for _ in range(2)]
    for which, p in enumerate(s["pages"]):
        _fill(_gen(seed * 131 + which + 1), p)
    rows = sum(counts)
    if case["kind"] != "append":
        s["out"] = torch.zeros(rows, case["nh"] * HD, device="cuda", dtype=torch.float32)
    if own:
        s["cache"], s["seqs"], s["counts"] = s["owner"].cache, list(range(n)), counts
        s["args"] = [_Buf(x[k]) for k in (("k", "v") if case["kind"] == "append" else ("q_gate", "k", "v"))]
        if case["kind"] != "append":
            s["args"].append(_Buf(s["out"]))
        torch.cuda.synchronize()
        return s
    # Plan of the plain form: each new row's sequence, place in its chunk and position.
    seq = np.repeat(np.arange(n), counts)
    at = np.concatenate([np.arange(c) for c in counts])
    pos = at + np.array(lens)[seq]
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int64)).cuda()  # noqa: E731
    s.update(seq=dev(seq), at=dev(at), pos=dev(pos), table=dev(table), lens=dev(np.array(lens)), most=max(counts),
             ends=dev(np.array(lens) + np.array(counts)), freq=torch.from_numpy(_freqs()).cuda())
    return s


# ------------------------------------------------------------------ the plain form

def _rope_norm(r, w, pos, freq):
    """r [rows][heads][256] at positions pos: the rotation of dims (d, d + 32), d < 32, then the (1 + w) norm, in 64 bits."""
    angle = (pos.float()[:, None] * freq)[:, None].double()
    c, s = torch.cos(angle), torch.sin(angle)
    r = r.double()
    h = ROPE_DIM // 2
    a, b = r[..., :h], r[..., h:ROPE_DIM]
    r = torch.cat([a * c - b * s, a * s + b * c, r[..., ROPE_DIM:]], -1)
    return r / torch.sqrt((r * r).mean(-1, keepdim=True) + EPS) * (1 + w.double())


def _plain_append(s):
    case, x = s["case"], s["x"]
    rows, nkv = s["pos"].numel(), case["nkv"]
    page, row = s["table"][s["seq"], s["pos"] // case["page"]], s["pos"] % case["page"]
    kp, vp = s["pages"]
    kp[page, :, row] = _rope_norm(x["k"].view(rows, nkv, HD), x["k_norm"], s["pos"], s["freq"]).to(kp.dtype)
    vp[page, :, row] = x["v"].view(rows, nkv, HD).to(vp.dtype)


def _plain_attend(s):
    """Every sequence padded to the longest: [n][kv head][group x new rows][cached rows]."""
    case, x = s["case"], s["x"]
    n, nh, nkv, T = case["n"], case["nh"], case["nkv"], s["most"]
    G, rows = nh // nkv, s["pos"].numel()
    qg = x["q_gate"].view(rows, nh, 2, HD)
    q = torch.zeros(n, T, nh, HD, device="cuda", dtype=torch.float32)
    q[s["seq"], s["at"]] = _rope_norm(qg[:, :, 0], x["q_norm"], s["pos"], s["freq"]).float()
    q = q.view(n, T, nkv, G, HD).permute(0, 2, 3, 1, 4).reshape(n, nkv, G * T, HD)
    K, V = (p[s["table"]].transpose(1, 2).reshape(n, nkv, -1, HD).float() for p in s["pages"])
    L = K.shape[2]
    cols = torch.arange(L, device="cuda")
    V = V.masked_fill((cols >= s["ends"][:, None])[:, None, :, None], 0.0)
    scores = (torch.matmul(q, K.transpose(2, 3).contiguous()) / math.sqrt(HD)).view(n, nkv, G, T, L)
    hidden = cols > (s["lens"][:, None] + torch.arange(T, device="cuda"))[:, :, None]          # [n][T][L]
    scores = scores.masked_fill(hidden[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = torch.matmul((p / p.sum(-1, keepdim=True)).view(n, nkv, G * T, L), V)
    o = o.view(n, nkv, G, T, HD).permute(0, 3, 1, 2, 4).reshape(n, T, nh, HD)[s["seq"], s["at"]]
    s["out"].copy_((o / (1 + torch.exp(-qg[:, :, 1]))).view(rows, nh * HD))


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        if kind == "append":
            s["cache"].append(0, s["seqs"], s["counts"], *s["args"])
        elif kind == "decode":
            s["cache"].attn_decode(0, s["seqs"], *s["args"])
        else:
            s["cache"].attn_prefill(0, s["seqs"], s["counts"], *s["args"])
    else:
        _plain_append(s)
        if kind != "append":
            _plain_attend(s)
    got = {"keys": s["pages"][0], "values": s["pages"][1]}
    if kind != "append":
        got["out"] = s["out"]
    return got


# ------------------------------------------------------------------ work

def work(case):
    """Bytes: cached rows and inputs read once, new rows and outputs written once.  Flops: Q K^T and P V over the rows a
    token sees; of an append, the rotation and the norm (about six operations a K value)."""
    nh, nkv = case["nh"], case["nkv"]
    lens, counts = _lens(case), _counts(case)
    width = 2 if case["half"] else 4
    rows = sum(counts)
    b = rows * nkv * HD * 2 * (4 + width)
    if case["kind"] == "append":
        return {"bytes": b, "flops": 6 * rows * nkv * HD}
    b += sum(lens) * nkv * HD * 2 * width + 12 * rows * nh * HD
    pairs = sum(c * a + c * (c + 1) // 2 for a, c in zip(lens, counts))
    return {"bytes": b, "flops": 4 * HD * nh * pairs}


# ------------------------------------------------------------------ 64-bit results

def _turned64(r, w, first):
    """Rows r [tokens][heads][256] of one sequence from position `first` on: rotated by complex products, then normed."""
    T = r.shape[0]
    pos = np.arange(first, first + T).astype(np.float32)
    ang = torch.from_numpy((pos[:, None] * _freqs()).astype(np.float64)).cuda()                # products rounded to 32 bits
    z = torch.complex(r[..., :32].double(), r[..., 32:64].double()) * torch.polar(torch.ones_like(ang), ang)[:, None]
    y = torch.cat([z.real, z.imag, r[..., 64:].double()], -1)
    return y * torch.rsqrt(y.square().sum(-1, keepdim=True) / HD + EPS) * (w.double() + 1)


def exact(case, seed):
    x, lens, counts, per, pool, table = _inputs(case, seed)
    n, nh, nkv, R = case["n"], case["nh"], case["nkv"], case["page"]
    G = nh // nkv
    store = torch.float16 if case["half"] else torch.float32
    pages = []
    for which in range(2):
        p = torch.empty(pool, nkv, R, HD, device="cuda", dtype=store)
        _fill(_gen(seed * 131 + which + 1), p)
        pages.append(p)
    outs, at = [], 0
    new = []
    for i, (a, c) in enumerate(zip(lens, counts)):
        tok = slice(at, at + c)
        at += c
        k = _turned64(x["k"][tok].view(c, nkv, HD), x["k_norm"], a)
        v = x["v"][tok].double().view(c, nkv, HD)
        new.append((k, v))
        if case["half"]:
            k, v = k.half().double(), v.half().double()       # what the cache holds
        if case["kind"] == "append":
            continue
        t = torch.from_numpy(table[i].astype(np.int64)).cuda()
        qg = x["q_gate"][tok].view(c, nh, 2, HD)
        q = _turned64(qg[:, :, 0], x["q_norm"], a)
        seen = torch.arange(a + c, device="cuda")[None] <= (a + torch.arange(c, device="cuda"))[:, None]
        o = torch.empty(c, nh, HD, device="cuda", dtype=torch.float64)
        for h in range(nkv):
            K = torch.cat([pages[0][t, h].reshape(-1, HD)[:a].double(), k[:, h]])
            V = torch.cat([pages[1][t, h].reshape(-1, HD)[:a].double(), v[:, h]])
            for j in range(G * h, G * h + G):
                s = torch.mm(q[:, j], K.t()).div_(math.sqrt(HD)).masked_fill_(~seen, -math.inf)
                o[:, j] = torch.mm(torch.softmax(s, -1), V)
        outs.append((o * torch.sigmoid(qg[:, :, 1].double())).view(c, nh * HD))
    wide = [p.double() for p in pages]
    for i, (a, c) in enumerate(zip(lens, counts)):
        pos = np.arange(a, a + c)
        pg, rw = (torch.from_numpy(v.astype(np.int64)).cuda() for v in (table[i][pos // R], pos % R))
        for which in range(2):
            wide[which][pg, :, rw] = new[i][which]
    got = {"keys": wide[0], "values": wide[1]}
    if outs:
        got["out"] = torch.cat(outs)
    return got
