"""Performance cases of a paged K/V cache held in 4 bits and of its page tables made on the GPU, at the attention shapes
of the 4B-class configuration (16 q heads on 4 kv heads of 256, 64 rotated dims) and, in drawn cases, other head counts
the tests hold.

Kinds of case:
  append   K (rotated, normed) and V rows of new tokens of n sequences into their pages, in 4 bits
  decode   the gated attention of one new token of each of n sequences over its 4-bit rows
  prefill  the gated attention of chunks of new tokens of n sequences over their 4-bit rows
  plan     page tables and the new tokens' slots of n requests from their lengths and a list of free pages

A row of a kv head is held as 8 blocks of 32 values: codes 0, 1/2, 1, 3/2, 2, 3, 4, 6 with a sign, times a power of two
that a block shares, the smallest one 2^s with the block's largest value at most 7 2^s, s from -23 to 13; a value is
rounded to the nearest code, ties to the even one, at most 6.  K rows are rounded to 32 bits first.  The first three kinds
return the new rows as the values that the cache holds of them.

Sequence i holds `rows` cached rows (fewer, unequally many, where `ragged`) and brings `tokens` new ones (likewise); its
pages of `page` rows lie in a random order in the pool, whose free pages and unwritten rows hold other conversations'
stale values.  A plan keeps the pages of the cached rows and takes the others from the free list in the requests' order,
each request all of its pages or none; `short` is how many requests the free list falls short of.

Streams: the library works on its context's own stream, which does not wait for torch's nor torch's for it.  prepare()
waits for the card before it takes memory that an earlier state's calls may still read, and after it has made the
inputs; run() enqueues, as a serving loop does, whose calls follow each other on that stream, and whoever takes its
outputs elsewhere synchronises first.

Where `own` is false, run() computes the same with elementary torch operations: 32 bits, with 64 for the rotation and
the norm (whose K rows are rounded to 4 bits).  Where it is true it calls the library's front end, on buffers of the
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
BLOCK = 32                          # values that share a power of two
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    a = {"nh": 16, "nkv": 4}
    return [
        # The smallest call: one token's rows of a conversation, as after a drafter's step.
        {"name": "append_1", "kind": "append", "n": 1, "rows": 4000, "tokens": 1, "ragged": False, "page": 64, **a},
        # A 2048-token prompt in the last attention layer, where all but the last token need their rows only.
        {"name": "append_2048", "kind": "append", "n": 1, "rows": 0, "tokens": 2048, "ragged": False, "page": 64, **a},
        # Prompts of six users at once, small pages.
        {"name": "append_6", "kind": "append", "n": 6, "rows": 1000, "tokens": 1300, "ragged": True, "page": 16, **a},
        # One conversation of 8K tokens.
        {"name": "decode_8k", "kind": "decode", "n": 1, "rows": 8191, "tokens": 1, "ragged": False, "page": 64, **a},
        # A full batch of ordinary conversations of unequal lengths, small pages.
        {"name": "decode_64", "kind": "decode", "n": 64, "rows": 4000, "tokens": 1, "ragged": True, "page": 16, **a},
        # Eight long conversations: what four bits are for.
        {"name": "decode_8x32k", "kind": "decode", "n": 8, "rows": 32639, "tokens": 1, "ragged": True, "page": 256, **a},
        # The first tokens of three short conversations: latency.
        {"name": "decode_short", "kind": "decode", "n": 3, "rows": 77, "tokens": 1, "ragged": True, "page": 16, **a},
        # A 2048-token prompt from an empty cache.
        {"name": "prefill_2048", "kind": "prefill", "n": 1, "rows": 0, "tokens": 2048, "ragged": False, "page": 64, **a},
        # A chunk of a long prompt over 16K rows.
        {"name": "prefill_512_16k", "kind": "prefill", "n": 1, "rows": 16000, "tokens": 512, "ragged": False, "page": 64, **a},
        # A mixed batch of a server: a prompt's chunk beside short turns of other conversations, odd sizes.
        {"name": "prefill_mixed", "kind": "prefill", "n": 6, "rows": 5000, "tokens": 307, "ragged": True, "page": 16, **a},
        # A decode step of a full batch: some requests begin a page, three find none.
        {"name": "plan_step", "kind": "plan", "n": 64, "rows": 4000, "tokens": 1, "ragged": True, "page": 16, "short": 3, **a},
        # Prompts of many users behind their shared prefixes and earlier turns, long tables.
        {"name": "plan_prompts", "kind": "plan", "n": 128, "rows": 9000, "tokens": 2048, "ragged": True, "page": 64, "short": 0, **a},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    """One more case: sizes spread over their logarithm, no dearer than the largest listed one of its kind."""
    kind = rng.choice(["append", "decode", "decode", "prefill", "prefill", "plan"])
    nh, nkv = rng.choice([(16, 4), (16, 4), (16, 4), (8, 4), (16, 2), (4, 4), (16, 1)])
    c = {"kind": kind, "ragged": rng.random() < 0.5, "page": rng.choice([16, 16, 32, 64, 128, 256]), "nh": nh, "nkv": nkv}
    if kind == "append":
        n = _log_int(rng, 1, 16)
        return {**c, "n": n, "rows": rng.randint(0, 3000), "tokens": _log_int(rng, 1, 2048 // n)}
    if kind == "decode":
        n = _log_int(rng, 1, 64)
        return {**c, "n": n, "rows": _log_int(rng, 1, min(32639, 200000 // n)), "tokens": 1}
    if kind == "plan":
        n = _log_int(rng, 1, 128)
        return {**c, "n": n, "rows": _log_int(rng, 1, 9000), "tokens": _log_int(rng, 1, 2048), "short": rng.choice([0, 0, min(n, 2)])}
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
    g.manual_seed(0x51344000 + seed)
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
    order = np.random.RandomState(seed % (1 << 31)).permutation(pool)
    return lens, counts, per, pool, order[:case["n"] * per].reshape(case["n"], per).astype(np.int32)


def _inputs(case, seed):
    g = _gen(seed)
    lens, counts, per, pool, table = _layout(case, seed)
    rows = sum(counts)
    x = {"k": _normal(g, rows, case["nkv"] * HD), "v": _normal(g, rows, case["nkv"] * HD),
         "q_norm": _normal(g, HD, mean=1.0, std=0.02), "k_norm": _normal(g, HD, mean=1.0, std=0.02)}
    if case["kind"] != "append":
        x["q_gate"] = _normal(g, rows, 2 * case["nh"] * HD)
    return x, lens, counts, per, pool, table


def _requests(case, seed):
    """A plan's inputs on the host: lengths, tokens, the table before (pages of the cached rows, -1 behind them), the free
    pages in a random order, all or as few as `short` says."""
    lens, counts, per, pool, pages = _layout(case, seed)
    R = case["page"]
    have = np.array([-(-a // R) for a in lens])
    need = np.array([-(-(a + b) // R) for a, b in zip(lens, counts)]) - have
    table = np.where(np.arange(per)[None] < have[:, None], pages, -1).astype(np.int32)
    free = np.setdiff1d(np.arange(pool, dtype=np.int32), table[table >= 0])
    free = np.random.RandomState((seed * 7 + 1) % (1 << 31)).permutation(free).astype(np.int32)
    asking = np.nonzero(need)[0]
    if case["short"] and len(asking) > case["short"]:
        free = free[:int(need.cumsum()[asking[-case["short"]]]) - 1]
    return np.array(lens, np.int32), np.array(counts, np.int32), per, pool, table, free


def _power(s):
    """2^s of whole numbers s in the range of 32-bit floats."""
    return ((s.int() + 127) << 23).view(torch.float32)


def _pack(x):
    """x [..., 256] in 32 bits as the cache holds it: codes [..., 128], two a byte, the even dim's in the lower half, and
    the blocks' powers of two [..., 8], as s + 127."""
    b = x.view(*x.shape[:-1], HD // BLOCK, BLOCK)
    top = b.abs().amax(-1)
    m, e = torch.frexp(top)                                  # top = m 2^e, 1/2 <= m < 1
    s = torch.where(m <= 0.875, e - 3, e - 2).masked_fill(top == 0, -23).clamp(-23, 13)
    y = b.abs() * _power(-s)[..., None]
    per = 2.0 - (y >= 2).float() - 0.5 * (y >= 4)            # codes a unit: 2 up to 2, 1 up to 4, then 1/2
    y = torch.clamp(torch.round(y * per) / per, max=6.0)     # (ties go to the even multiple, which is the even code)
    code = torch.where(y <= 2, 2 * y, torch.where(y <= 4, y + 2, 7.0)).to(torch.uint8) + 8 * torch.signbit(b).to(torch.uint8)
    code = code.view(*x.shape[:-1], HD // 2, 2)
    return code[..., 0] + 16 * code[..., 1], (s + 127).to(torch.uint8)


def _values(codes, scales):
    """The values of codes [..., 128] and scales [..., 8], in 32 bits."""
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device="cuda", dtype=torch.float32)
    low, high = level[(codes & 15).int()], level[(codes >> 4).int()]
    x = torch.stack([low, high], -1).view(*codes.shape[:-1], HD // BLOCK, BLOCK)
    return (x * _power(scales.int() - 127)[..., None]).view(*codes.shape[:-1], HD)


def _fill(g, codes, scales):
    """The pool's contents: normal values, in pieces (the conversations' cached rows and stale ones alike)."""
    codes, scales = codes.view(-1, HD // 2), scales.view(-1, HD // BLOCK)
    step = 1 << 18
    for at in range(0, codes.shape[0], step):
        n = min(step, codes.shape[0] - at)
        codes[at:at + n], scales[at:at + n] = _pack(torch.randn(n, HD, generator=g, device="cuda", dtype=torch.float32))


def _pool(case, seed, which, pool):
    shape = (pool, case["nkv"], case["page"])
    codes = torch.empty(*shape, HD // 2, device="cuda", dtype=torch.uint8)
    scales = torch.empty(*shape, HD // BLOCK, device="cuda", dtype=torch.uint8)
    _fill(_gen(seed * 131 + which + 1), codes, scales)
    return codes, scales


class _Foreign:
    """Memory of the library's cache as torch takes it; it lives as long as its owner."""

    def __init__(self, owner, ptr, shape, typestr):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": tuple(shape), "strides": None, "typestr": typestr, "data": (ptr, False),
                                         "version": 2}


class _Owner:
    """A paged cache, and the layer of its context that has the state's weights.  A program has one context, of several layers,
    whose calls follow each other on one stream, and makes a cache once for conversations that come and go: a state takes
    one that neither an earlier state nor a view of its memory has any more."""
    program = None

    def __init__(self, case, per, pool, x=None):
        here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3.5sharp_amd")
        if here not in sys.path:
            sys.path.insert(0, here)
        import q35mix
        self.kinds = (q35mix.STATE_KEYS, q35mix.STATE_VALUES)
        key = (case["nh"], case["nkv"], case["n"], per, pool, case["page"], x is None)
        if _Owner.program is None or _Owner.program.key != key or not _Owner.program.places:
            _Owner.program = _Program(q35mix, key, 1 if x is None else 5)
        self.of = _Owner.program
        self.ctx, self.place = self.of.ctx, self.of.places.pop(0)
        self.layer = 0 if x is None else self.place
        if self.place not in self.of.caches:
            self.of.caches[self.place] = q35mix.PagedCache(self.ctx, n_seqs=case["n"], max_rows=per * case["page"], n_pages=pool,
                                                           page_rows=case["page"], kv_type=q35mix.KV_MXFP4)
        self.cache = self.of.caches[self.place]
        if x is not None:
            self.ctx.set_attn_weights(self.layer, {k: x[k].cpu().numpy() for k in ("q_norm", "k_norm")})

    def hold(self, lens, table):
        """The conversations' pages and lengths, in place of the ones before."""
        for i, (rows, pages) in enumerate(zip(lens, table)):
            if self.cache.length(i) > rows:
                self.cache.truncate(i, rows)
            self.cache.map(i, 0, pages)
        self.cache.advance(list(range(len(lens))), [rows - self.cache.length(i) for i, rows in enumerate(lens)])

    def put(self, which, codes, scales):
        """One pool's contents in the library's layout: of each (page, kv head) the rows' codes, then their scales, K's by
        row and V's by 16 rows, block by block."""
        pool, nkv, page = codes.shape[:3]
        to = torch.as_tensor(_Foreign(self, self.cache.device_ptr(self.layer, self.kinds[which])[0], (pool, nkv, page * 136), "|u1"),
                             device="cuda")
        to[..., :page * 128] = codes.view(pool, nkv, -1)
        if which:
            scales = scales.view(pool, nkv, page // 16, 16, 8).transpose(3, 4)
        to[..., page * 128:] = scales.reshape(pool, nkv, -1)

    def tables(self):
        table, lens, pages = self.cache.tables()
        n = self.cache.n_seqs
        return [torch.as_tensor(_Foreign(self, at, shape, "<i4"), device="cuda") for at, shape in ((table, (n, pages)), (lens, (n,)))]

    def __del__(self):
        if hasattr(self, "cache"):
            self.of.places.insert(0, self.place)


class _Program:
    """A context and its caches, for five states at once, closed when none has them and another shape is asked for."""

    def __init__(self, q35mix, key, layers):
        self.key, self.places, self.caches = key, list(range(5)), {}
        self.ctx = q35mix.Context(q35mix.qwen35_config(num_layers=layers, num_heads=key[0], num_kv_heads=key[1],
                                                       is_recurrent=[0] * layers), n_seqs=1, kv_capacity=16)

    def __del__(self):
        if hasattr(self, "ctx") and not sys.is_finalizing():
            for cache in self.caches.values():
                cache.close()
            self.ctx.close()


class _Buf:
    """A torch tensor as the front end takes device buffers (.ptr)."""

    def __init__(self, t):
        assert t.is_contiguous()
        self.t, self.ptr, self.nbytes = t, t.data_ptr(), t.numel() * t.element_size()


def _prepare_plan(case, seed):
    lens, counts, per, pool, table, free = _requests(case, seed)
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    x = {"rows": dev(lens), "tokens": dev(counts), "free": dev(free)}
    s = {"case": case, "x": x, "pool": pool, "slots": torch.empty(int(counts.sum()), device="cuda", dtype=torch.int64),
         "taken": torch.empty(case["n"], device="cuda", dtype=torch.int32)}
    if own:
        # the library's cache: its table holds the pages of the cached rows, which a plan does not touch (one head)
        s["owner"] = _Owner({**case, "nh": 1, "nkv": 1}, per, pool)
        s["cache"] = s["owner"].cache
        s["table"], s["lens"] = s["owner"].tables()
        s["args"] = [_Buf(t) for t in (x["rows"], x["tokens"], x["free"], s["slots"], s["taken"])]
    else:
        s["table"] = torch.empty(case["n"], per, device="cuda", dtype=torch.int32)
        s["lens"] = torch.empty(case["n"], device="cuda", dtype=torch.int32)
    s["table"].copy_(dev(table))
    torch.cuda.synchronize()
    return s


def prepare(case, seed):
    if own:
        torch.cuda.synchronize()
    if case["kind"] == "plan":
        return _prepare_plan(case, seed)
    x, lens, counts, per, pool, table = _inputs(case, seed)
    n, nkv, rows = case["n"], case["nkv"], sum(counts)
    s = {"case": case, "x": x, "keys": torch.empty(rows, nkv * HD, device="cuda", dtype=torch.float32),
         "values": torch.empty(rows, nkv * HD, device="cuda", dtype=torch.float32)}
    if case["kind"] != "append":
        s["out"] = torch.zeros(rows, case["nh"] * HD, device="cuda", dtype=torch.float32)
    pools = [_pool(case, seed, which, pool) for which in range(2)]
    if own:
        # the library's cache: its pages are its own memory, its tables are set and checked as conversations come
        s["owner"] = _Owner(case, per, pool, x)
        s["cache"], s["layer"], s["seqs"], s["lens"], s["counts"] = s["owner"].cache, s["owner"].layer, list(range(n)), lens, counts
        s["owner"].hold(lens, table)
        for which in range(2):
            s["owner"].put(which, *pools[which])
        s["args"] = [_Buf(x[k]) for k in (("k", "v") if case["kind"] == "append" else ("q_gate", "k", "v"))]
        if case["kind"] != "append":
            s["args"].append(_Buf(s["out"]))
        s["held"] = [_Buf(s["keys"]), _Buf(s["values"])]
        torch.cuda.synchronize()
        return s
    s["pools"] = pools
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
    (kc, ke), (vc, ve) = s["pools"]
    k = _pack(_rope_norm(x["k"].view(rows, nkv, HD), x["k_norm"], s["pos"], s["freq"]).float())
    v = _pack(x["v"].view(rows, nkv, HD))
    kc[page, :, row], ke[page, :, row] = k
    vc[page, :, row], ve[page, :, row] = v
    s["keys"].copy_(_values(*k).view(rows, nkv * HD))
    s["values"].copy_(_values(*v).view(rows, nkv * HD))


def _plain_attend(s):
    """Every sequence padded to the longest: [n][kv head][group x new rows][cached rows]."""
    case, x = s["case"], s["x"]
    n, nh, nkv, T = case["n"], case["nh"], case["nkv"], s["most"]
    G, rows = nh // nkv, s["pos"].numel()
    qg = x["q_gate"].view(rows, nh, 2, HD)
    q = torch.zeros(n, T, nh, HD, device="cuda", dtype=torch.float32)
    q[s["seq"], s["at"]] = _rope_norm(qg[:, :, 0], x["q_norm"], s["pos"], s["freq"]).float()
    q = q.view(n, T, nkv, G, HD).permute(0, 2, 3, 1, 4).reshape(n, nkv, G * T, HD)
    K, V = (_values(*(t[s["table"]].transpose(1, 2).reshape(n, nkv, -1, t.shape[-1]) for t in pool)) for pool in s["pools"])
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


def _plain_plan(s):
    x, R, table = s["x"], s["case"]["page"], s["table"]
    rows, tokens, free = x["rows"].long(), x["tokens"].long(), x["free"]
    have = (rows + R - 1) // R
    need = (rows + tokens + R - 1) // R - have
    upto = need.cumsum(0)
    served = (need == 0) | (upto <= free.numel())
    col = torch.arange(table.shape[1], device="cuda")
    new = (col >= have[:, None]) & (col < (have + need)[:, None]) & served[:, None]
    place = ((upto - need - have)[:, None] + col).clamp(0, free.numel() - 1)
    table.copy_(torch.where(col < have[:, None], table, torch.where(new, free[place], -1)))
    s["lens"].copy_(rows)
    s["taken"].copy_(torch.where(served, need, -1))
    ends = tokens.cumsum(0)
    slot = torch.arange(s["slots"].numel(), device="cuda")
    i = torch.searchsorted(ends, slot, right=True)
    pos = rows[i] + slot - (ends - tokens)[i]
    page = table[i, pos // R].long()
    s["slots"].copy_(torch.where(page < 0, -1, page * R + pos % R))


def run(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "plan":
        if own:
            s["cache"].plan(case["n"], *s["args"])
        else:
            _plain_plan(s)
        return {k: s[k] for k in ("table", "lens", "slots", "taken")}
    if own:
        if kind == "append":
            s["cache"].append(s["layer"], s["seqs"], s["counts"], *s["args"])
        elif kind == "decode":
            s["cache"].attn_decode(s["layer"], s["seqs"], *s["args"])
        else:
            s["cache"].attn_prefill(s["layer"], s["seqs"], s["counts"], *s["args"])
        s["cache"].rows(s["layer"], s["seqs"], s["lens"], s["counts"], *s["held"])
    else:
        _plain_append(s)
        if kind != "append":
            _plain_attend(s)
    return {k: s[k] for k in ("keys", "values", "out") if k in s}


# ------------------------------------------------------------------ work

def work(case):
    """Bytes: cached rows (136 of each kv head, K and V) and inputs read once, new rows, the values they stand for and outputs
    written once.  Flops: Q K^T and P V over the rows a token sees; of an append, the rotation and the norm (about six
    operations a K value).  A plan: lengths and taken pages in and out, the table's kept entries read and the others
    written, the slots; an operation an entry and slot."""
    nh, nkv = case["nh"], case["nkv"]
    lens, counts = _lens(case), _counts(case)
    n, rows = case["n"], sum(counts)
    if case["kind"] == "plan":
        per = max(-(-(a + b) // case["page"]) for a, b in zip(lens, counts))
        return {"bytes": 16 * n + 4 * n * per + 8 * rows, "flops": n * per + rows}
    b = rows * nkv * 2 * (HD * 4 + 136 + HD * 4)
    if case["kind"] == "append":
        return {"bytes": b, "flops": 6 * rows * nkv * HD}
    b += sum(lens) * nkv * 2 * 136 + 12 * rows * nh * HD
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


def _held64(r):
    """What the cache holds of rows r [..., 256]: each value's block exponent is ceil(log2(largest / 7)), and its code the
    number of borders between neighbours that it passes, a border itself going to the even code."""
    b = r.double().reshape(-1, BLOCK)
    unit = torch.exp2(torch.ceil(torch.log2(b.abs().max(-1, keepdim=True).values / 7)).clamp(-23, 13))
    y = b.abs() / unit
    code = torch.zeros_like(y, dtype=torch.int64)
    for i in range(7):
        border = (LEVELS[i] + LEVELS[i + 1]) / 2
        code += y >= border if i % 2 else y > border
    y = torch.tensor(LEVELS, device="cuda", dtype=torch.float64)[code]
    return (torch.copysign(y, b) * unit).reshape(r.shape)


def _cached64(codes, scales):
    """Rows of the pool: value by value from the code's sign, exponent and fraction bits."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(torch.int32)
    e, f = (c >> 1) & 3, (c & 1).double()
    mag = torch.where(e == 0, f / 2, (1 + f / 2) * torch.exp2((e - 1).double()))
    unit = torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, -1)
    return torch.where(c >= 8, -mag, mag) * unit


def exact(case, seed):
    if case["kind"] == "plan":
        return None                                       # whole numbers
    x, lens, counts, per, pool, table = _inputs(case, seed)
    n, nh, nkv = case["n"], case["nh"], case["nkv"]
    G = nh // nkv
    pools = [_pool(case, seed, which, pool) for which in range(2)]
    outs, at, new = [], 0, [[], []]
    for i, (a, c) in enumerate(zip(lens, counts)):
        tok = slice(at, at + c)
        at += c
        k = _held64(_turned64(x["k"][tok].view(c, nkv, HD), x["k_norm"], a).float())
        v = _held64(x["v"][tok].view(c, nkv, HD))
        new[0].append(k.view(c, nkv * HD))
        new[1].append(v.view(c, nkv * HD))
        if case["kind"] == "append":
            continue
        t = torch.from_numpy(table[i].astype(np.int64)).cuda()
        qg = x["q_gate"][tok].view(c, nh, 2, HD)
        q = _turned64(qg[:, :, 0], x["q_norm"], a)
        seen = torch.arange(a + c, device="cuda")[None] <= (a + torch.arange(c, device="cuda"))[:, None]
        o = torch.empty(c, nh, HD, device="cuda", dtype=torch.float64)
        for h in range(nkv):
            K, V = (torch.cat([_cached64(*(p[t, h].flatten(0, 1)[:a] for p in pools[w])), r[:, h]]) for w, r in ((0, k), (1, v)))
            for j in range(G * h, G * h + G):
                s = torch.mm(q[:, j], K.t()).div_(math.sqrt(HD)).masked_fill_(~seen, -math.inf)
                o[:, j] = torch.mm(torch.softmax(s, -1), V)
        outs.append((o * torch.sigmoid(qg[:, :, 1].double())).view(c, nh * HD))
    got = {"keys": torch.cat(new[0]), "values": torch.cat(new[1])}
    if outs:
        got["out"] = torch.cat(outs)
    return got
