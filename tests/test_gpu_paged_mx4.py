"""Paged K/V cache in 4 bits on the GPU: rows appended and read back, attention of one new token and of chunks of new
tokens, against a plain restatement in 64 bits (numpy).

Tolerances.  Rows: the kernels form a K row in 64 bits, round it to fp32 and then to its codes, as the restatement does:
codes and scales must be equal (see test_gpu_paged.py).  Outputs: the cache's values take part exactly.  q is held to
2^-20 of the largest value of its 32 dims at least, with random signs: the largest of 32 normal values being about 2.2
of their deviation, a score's relative deviation is 2.2 2^-20 / sqrt(3) = 1.2e-6 of its size in the norms' product, which
for these rows is up to 1.44 |q| |k| / 16 / 16 = 2 in units of log2, 2.4e-6.  The fp32 sums are those of the other caches:
9e-6 (test_gpu_paged.py).  2e-5 of the largest output covers two deviations of both together.
"""
import ctypes

import numpy as np
import pytest

import mx4_rows
import q35mix
import synth
from q35mix import KV_F16, KV_F32, KV_MXFP4, STATE_KEYS, STATE_VALUES
from test_gpu_paged import HD, Paged, close_to, refused, rope_norm, say

pytestmark = pytest.mark.gpu


class Mx4(Paged):
    """Pages as codes and scales; where nothing was written the scale is NaN."""

    def __init__(self, **kw):
        self.codes = None
        super().__init__(KV_MXFP4, **kw)

    def push(self):
        if self.codes is None:
            shape = (self.n_pages, self.nkv, self.R)
            self.codes = [np.full((*shape, 128), 0x5a, np.uint8) for _ in range(2)]
            self.scales = [np.full((*shape, 8), 255, np.uint8) for _ in range(2)]
            self.pages = None
        for which, kind in enumerate((STATE_KEYS, STATE_VALUES)):
            ptr, n = self.c.device_ptr(self.layer, kind)
            a = mx4_rows.to_pool(which, self.codes[which], self.scales[which])
            assert n == a.nbytes
            q35mix.check(q35mix.lib().q35m_copy_h2d(self.ctx.handle, ptr, a.ctypes.data, n))

    def pull(self):
        got = []
        for which, kind in enumerate((STATE_KEYS, STATE_VALUES)):
            ptr, n = self.c.device_ptr(self.layer, kind)
            a = np.empty((self.n_pages, self.nkv, 136 * self.R), np.uint8)
            q35mix.check(q35mix.lib().q35m_copy_d2h(self.ctx.handle, a.ctypes.data, ptr, n))
            got.append(mx4_rows.from_pool(which, a, self.R))
        return got

    def set_row(self, which, s, r, x):
        """Row r of sequence s becomes x [kv heads][256] in 4 bits."""
        at = self.table[s][r // self.R], slice(None), r % self.R
        self.codes[which][at], self.scales[which][at] = mx4_rows.encode(np.asarray(x, np.float32))

    def seed_rows(self, lens, salt=0, scale=1.0):
        for s, n in enumerate(lens):
            for which in range(2):
                x = synth.normal(7000 + 31 * salt + 2 * s + which, n * self.nkv * HD).reshape(n, self.nkv, HD) * scale
                t = np.arange(n)
                at = self.table[s][t // self.R], slice(None), t % self.R
                self.codes[which][at], self.scales[which][at] = mx4_rows.encode(x.astype(np.float32))
        self.push()
        self.c.advance(list(range(len(lens))), list(lens))
        for s, n in enumerate(lens):
            self.len[s] = n

    def rows_of(self, s, n, which):
        t = np.arange(n)
        at = self.table[s][t // self.R], slice(None), t % self.R
        return mx4_rows.decode(self.codes[which][at], self.scales[which][at])

    def put(self, seqs, tokens, x):
        at = 0
        for s, t in zip(seqs, tokens):
            k = rope_norm(x["k"][at:at + t].reshape(t, self.nkv, HD), self.w["k_norm"], self.len[s] + np.arange(t))
            v = x["v"][at:at + t].reshape(t, self.nkv, HD)
            at += t
            if t:
                r = self.len[s] + np.arange(t)
                to = self.table[s][r // self.R], slice(None), r % self.R
                for which, y in enumerate((k, v)):
                    self.codes[which][to], self.scales[which][to] = mx4_rows.encode(y.astype(np.float32))

    def check_pages(self):
        for which, (codes, scales) in enumerate(self.pull()):
            bad = scales != self.scales[which]
            assert not bad.any(), (which, int(bad.sum()), np.argwhere(bad)[:4])
            nan = np.repeat(scales == 255, 16, -1) & (self.codes[which] == 0)       # a NaN block's codes are 0
            bad = (codes != self.codes[which]) & ~nan
            assert not bad.any(), (which, int(bad.sum()), np.argwhere(bad)[:4])


# ------------------------------------------------------------------ rows

@pytest.mark.parametrize("lens,tokens,page", [([0], [1], 16), ([15, 0, 33], [2, 0, 40], 16), ([100, 3], [1, 129], 64),
                                              ([0, 7, 1, 64], [300, 0, 1, 0], 32), ([1000], [24], 1024)])
@pytest.mark.parametrize("nh,nkv", [(16, 4), (4, 4), (16, 1)])
def test_append_and_rows(lens, tokens, page, nh, nkv):
    n = len(lens)
    with Mx4(nh=nh, nkv=nkv, n_seqs=n, max_rows=1024, page_rows=page, salt=n) as p:
        p.seed_rows(lens, salt=n)
        x = p.inputs(sum(tokens), salt=20 + n)
        k, v = p.dev(x, "k", "v")
        p.c.append(0, list(range(n)), tokens, k, v)
        p.put(range(n), tokens, x)
        p.check_pages()
        assert [p.c.length(s) for s in range(n)] == lens              # not moved
        total = [a + b for a, b in zip(lens, tokens)]
        rows = sum(total) - sum(a // 2 for a in total)
        kd, vd = (p.ctx.array((rows + 1, nkv * HD), np.full((rows + 1, nkv * HD), 7, np.float32)) for _ in range(2))
        p.c.rows(0, list(range(n)), [a // 2 for a in total], [a - a // 2 for a in total], kd, vd)
        for which, d in enumerate((kd, vd)):
            want = np.concatenate([p.rows_of(s, a, which)[a // 2:] for s, a in enumerate(total)]).reshape(rows, -1)
            got = d.download()
            assert np.array_equal(got[:rows].view(np.uint32), want.view(np.uint32))
            assert (got[rows] == 7).all()


def test_values_at_the_format_s_edges():
    """V rows, which are held as they come: ties of every pair of codes, largest values at and beside 7 2^s, the range's
    ends, zeros of both signs, blocks that are not finite."""
    T = 40
    with Mx4(max_rows=64) as p:
        x = p.inputs(T, salt=3)
        v = x["v"].reshape(T, 4, 8, 32)
        ties = np.array([0, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5, -6, -7, -0.0], np.float32)
        near = np.concatenate([np.nextafter(ties, np.float32(100)), np.nextafter(ties, np.float32(-100))])
        for j, s in enumerate(range(-26, 16)):
            if j < T:
                v[j, 0, 0, :20] = ties * np.float32(2.0 ** s)
                v[j, 0, 1, :20] = near[:20] * np.float32(2.0 ** s)
                v[j, 0, 2, :20] = near[20:] * np.float32(2.0 ** s)
        for j, top in enumerate((7.0, np.nextafter(np.float32(7), np.float32(8)), np.nextafter(np.float32(7), np.float32(6)), 3.5, 4.0, 1.75)):
            v[j, 1, 0] = np.linspace(-1, 1, 32).astype(np.float32) * np.float32(top)
        v[0, 2, 0], v[0, 2, 1], v[0, 2, 2] = 0.0, -0.0, np.float32(1e-45)
        v[1, 2, 0, 3], v[1, 2, 1, 4], v[1, 2, 2, 5] = np.inf, -np.inf, np.nan
        v[2, 2, 0], v[2, 2, 1, 7], v[2, 2, 2, 9] = np.float32(3e38), np.float32(-3e38), np.float32(57344)
        v[3, 2, 0], v[3, 2, 1] = np.float32(2.0 ** -24), np.float32(2.0 ** -25)
        k, vd = p.dev(x, "k", "v")
        p.c.append(0, [0], [T], k, vd)
        p.put([0], [T], x)
        p.check_pages()
        kd, out = p.ctx.array((T, 1024)), p.ctx.array((T, 1024))
        p.c.rows(0, [0], [0], [T], kd, out)
        got, want = out.download().reshape(T, 4, HD), p.rows_of(0, T, 1)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)])
        assert (np.abs(want[2, 2, :32]) == 6 * 2.0 ** 13).all() and np.isnan(want[1, 2, :96]).all()


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
def test_rows_of_the_wider_caches(kv_type):
    with Paged(kv_type, n_seqs=2, max_rows=64, page_rows=16) as p:
        p.seed_rows([40, 17], salt=1)
        k, v = p.ctx.array((30, 1024)), p.ctx.array((30, 1024))
        p.c.rows(0, [1, 0], [3, 24], [14, 16], k, v)
        for which, d in enumerate((k, v)):
            want = np.concatenate([p.rows_of(1, 17, which)[3:], p.rows_of(0, 40, which)[24:]]).astype(np.float32).reshape(30, -1)
            assert np.array_equal(d.download(), want)


# ------------------------------------------------------------------ one new token

def decode(p, seqs, lens, salt):
    x = p.inputs(len(seqs), salt=salt)
    out = p.ctx.array((len(seqs) + 1, p.nh * HD), np.full((len(seqs) + 1, p.nh * HD), 5, np.float32))
    p.c.attn_decode(0, list(seqs), *p.dev(x, "q_gate", "k", "v"), out)
    p.put(seqs, [1] * len(seqs), x)
    want, got = p.attend(seqs, [1] * len(seqs), x), out.download()
    p.check_pages()
    assert (got[-1] == 5).all()
    return close_to(got[:-1], want)


@pytest.mark.parametrize("lens", [[0], [1], [14, 15, 16], [31, 32, 33, 0], [126, 127, 128, 129], [510, 511, 512, 513],
                                  [1023, 5], [700, 0, 1, 300, 64]])
@pytest.mark.parametrize("page", [16, 64, 1024])
def test_decode_lengths(lens, page):
    with Mx4(n_seqs=len(lens), max_rows=1024, page_rows=page, salt=len(lens)) as p:
        p.seed_rows(lens, salt=2)
        say(decode(p, range(len(lens)), lens, 9))


@pytest.mark.parametrize("nh,nkv", [(4, 4), (8, 4), (16, 4), (8, 1), (16, 2), (16, 1), (24, 1), (32, 1), (32, 2)])
def test_decode_heads(nh, nkv):
    lens = [300, 0, 77, 640]
    with Mx4(nh=nh, nkv=nkv, n_seqs=4, max_rows=700, page_rows=32, salt=nh + nkv) as p:
        p.seed_rows(lens, salt=nh)
        say(decode(p, [2, 0, 3, 1], lens, nh))


def test_decode_full_batch():
    lens = [(37 * i * i) % 900 for i in range(64)]
    with Mx4(nh=4, nkv=1, n_seqs=64, max_rows=1024, page_rows=16) as p:
        p.seed_rows(lens, salt=4)
        say(decode(p, range(64), lens, 5))


# ------------------------------------------------------------------ chunks

def prefill(p, seqs, tokens, salt, some=None):
    rows = sum(tokens)
    x = p.inputs(rows, salt=salt)
    out = p.ctx.array((rows + 1, p.nh * HD), np.full((rows + 1, p.nh * HD), 5, np.float32))
    p.c.attn_prefill(0, list(seqs), list(tokens), *p.dev(x, "q_gate", "k", "v"), out)
    p.put(seqs, tokens, x)
    want, got = p.attend(seqs, tokens, x, some=some), out.download()
    p.check_pages()
    assert (got[-1] == 5).all()
    return close_to(got[:-1], want)


@pytest.mark.parametrize("lens,tokens", [([0], [1]), ([0], [16]), ([0], [17]), ([63], [1]), ([64], [2]), ([5], [130]),
                                         ([250, 3], [6, 70]), ([0, 100, 33, 7], [40, 0, 1, 90]), ([600], [65]), ([0], [200])])
@pytest.mark.parametrize("page", [16, 128])
def test_prefill_lengths(lens, tokens, page):
    with Mx4(n_seqs=len(lens), max_rows=1024, page_rows=page, salt=len(lens)) as p:
        p.seed_rows(lens, salt=6)
        say(prefill(p, range(len(lens)), tokens, 11))


@pytest.mark.parametrize("nh,nkv", [(4, 4), (8, 4), (16, 4), (8, 1), (16, 2), (16, 1), (24, 1), (32, 1)])
def test_prefill_heads(nh, nkv):
    with Mx4(nh=nh, nkv=nkv, n_seqs=3, max_rows=700, page_rows=32, salt=nh) as p:
        p.seed_rows([300, 0, 77], salt=nh)
        say(prefill(p, [2, 0, 1], [35, 21, 48], nh + 1))


@pytest.mark.parametrize("nh,nkv,rows,tokens", [(16, 4, 0, 1000), (16, 2, 2900, 100)])
def test_prefill_long(nh, nkv, rows, tokens):
    with Mx4(nh=nh, nkv=nkv, max_rows=4000, page_rows=64) as p:
        p.seed_rows([rows], salt=8)
        say(prefill(p, [0], [tokens], 12, some=list(range(0, tokens, 97)) + [tokens - 1]))


def test_a_conversation():
    """Prompts, tokens, a prompt's rows alone, more tokens, over a prefix that two sequences share."""
    with Mx4(n_seqs=2, max_rows=256, page_rows=16) as p:
        prefill(p, [0], [48], 1)
        p.step([48, 0])
        p.c.map(1, 0, p.table[0][:3])
        p.table[1][:3] = p.table[0][:3]
        p.c.advance([1], [48])
        p.len[1] = 48
        for turn in range(3):
            prefill(p, [0, 1], [5 + turn, 20 - turn], 2 + turn)
            p.step([5 + turn, 20 - turn])
            for _ in range(3):
                decode(p, [1, 0], p.len, 30 + turn)
                p.step([1, 1])
            x = p.inputs(7, salt=50 + turn)
            p.c.append(0, [0], [7], *p.dev(x, "k", "v"))
            p.put([0], [7], x)
            p.step([7, 0])
        p.check_pages()


# ------------------------------------------------------------------ what is not finite

def test_blocks_that_are_not_finite_reach_only_the_tokens_that_see_them():
    """V of some tokens in a chunk has infinities and NaN: their blocks are NaN in the outputs of later tokens, and every other
    value is as without them."""
    T, bad = 70, {11: (0, 37), 40: (1, 200), 69: (2, 3)}        # token: (kv head, dim)
    with Mx4(n_seqs=1, max_rows=512, page_rows=16) as p:
        p.seed_rows([130], salt=5)
        x = p.inputs(T, salt=6)
        v = x["v"].reshape(T, 4, HD)
        for (t, (h, d)), worst in zip(bad.items(), (np.inf, -np.inf, np.nan)):
            v[t, h, d] = worst
        out = p.ctx.array((T, p.nh * HD))
        p.c.attn_prefill(0, [0], [T], *p.dev(x, "q_gate", "k", "v"), out)
        p.put([0], [T], x)
        p.check_pages()
        got = out.download().reshape(T, 16, HD)
        nan = np.zeros_like(got, bool)
        for t, (h, d) in bad.items():
            nan[t:, 4 * h:4 * h + 4, d // 32 * 32:d // 32 * 32 + 32] = True
        assert np.array_equal(np.isnan(got), nan)
        for s in p.scales:
            s[s == 255] = 127                                   # (what the others' results are made of stays)
        want = p.attend([0], [T], x).reshape(T, 16, HD)
        close_to(got, np.where(nan, np.nan, want))
        # the next token sees all three
        p.step([T])
        p.put([0], [0], x)
        y = p.inputs(1, salt=7)
        p.c.attn_decode(0, [0], *p.dev(y, "q_gate", "k", "v"), out)
        got = out.download()[0].reshape(16, HD)
        assert np.array_equal(np.isnan(got), nan[-1])


def test_rows_that_are_not_a_sequence_s_own_are_not_seen():
    """Stale rows of a page behind the length are NaN blocks (the fixture's), in K and in V; every test above runs beside
    them, and here beside a long sequence's too."""
    with Mx4(n_seqs=2, max_rows=512, page_rows=256) as p:
        p.seed_rows([257, 400], salt=9)
        decode(p, [0, 1], p.len, 3)
        p.step([1, 1])
        prefill(p, [0, 1], [3, 66], 4)


# ------------------------------------------------------------------ captured calls

def capture(p, calls):
    hip = q35mix.hip()
    stream, graph, ex = ctypes.c_void_p(p.ctx.stream), ctypes.c_void_p(), ctypes.c_void_p()
    p.ctx.sync()
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    try:
        calls()
    finally:
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, ctypes.c_size_t(0)) == 0

    def launch():
        assert hip.hipGraphLaunch(ex, stream) == 0
        p.ctx.sync()

    def end():
        p.ctx.sync()
        assert hip.hipGraphExecDestroy(ex) == 0 and hip.hipGraphDestroy(graph) == 0
    return launch, end


def test_captured_calls_follow_lengths():
    with Mx4(n_seqs=2, max_rows=700, page_rows=16) as p:
        p.seed_rows([500, 3], salt=1)
        x, y = p.inputs(2, salt=2), p.inputs(9, salt=3)
        out, outp = p.ctx.array((2, p.nh * HD)), p.ctx.array((9, p.nh * HD))
        d, e = p.dev(x, "q_gate", "k", "v"), p.dev(y, "q_gate", "k", "v")
        p.c.attn_decode(0, [0, 1], *d, out)                     # (whatever the first calls load is loaded)
        launch, end = capture(p, lambda: (p.c.attn_decode(0, [0, 1], *d, out), p.c.attn_prefill(0, [1, 0], [4, 5], *e, outp)))
        for step in range(9):                                   # (over unit and page ends)
            launch()
            p.put([0, 1], [1, 1], x)
            close_to(out.download(), p.attend([0, 1], [1, 1], x))
            p.put([1, 0], [4, 5], y)
            close_to(outp.download(), p.attend([1, 0], [4, 5], y))
            p.check_pages()
            p.step([5, 4])
        end()


# ------------------------------------------------------------------ refusals

def test_refusals():
    cfg = q35mix.qwen35_config(num_layers=2, is_recurrent=[1, 0])
    with q35mix.Context(cfg, n_seqs=1, kv_capacity=16) as ctx:
        with q35mix.PagedCache(ctx, n_seqs=2, max_rows=100, n_pages=8, page_rows=16, kv_type=KV_MXFP4) as c:
            k = ctx.array((8, 1024))
            assert c.device_ptr(1, STATE_KEYS)[1] == 8 * 4 * 16 * 136
            refused(q35mix.ERR_CAPACITY, lambda: c.rows(1, [0], [0], [1], k, k), "mapped")
            c.map(0, 0, range(3))
            c.rows(1, [0], [40], [8], k, k)
            c.rows(1, [0], [100], [0], k, k)
            refused(q35mix.ERR_CAPACITY, lambda: c.rows(1, [0], [41], [8], k, k), "mapped")
            refused(q35mix.ERR_CAPACITY, lambda: c.rows(1, [0], [99], [2], k, k), "exceed")
            refused(q35mix.ERR_CAPACITY, lambda: c.rows(1, [0], [2 ** 31 - 1], [2 ** 24], k, k), "exceed")
            refused(q35mix.ERR_INVALID, lambda: c.rows(1, [0], [-1], [1], k, k), "row")
            refused(q35mix.ERR_INVALID, lambda: c.rows(1, [0], [1], [-1], k, k), "row")
            refused(q35mix.ERR_INVALID, lambda: c.rows(0, [0], [0], [1], k, k), "DeltaNet")
            refused(q35mix.ERR_INVALID, lambda: c.rows(1, [0, 0], [0, 0], [1, 1], k, k), "repeated")
            refused(q35mix.ERR_UNSUPPORTED, lambda: c.rows(1, [0], [0], [2 ** 24 + 1], k, k), "rows")
            null = type("Null", (), {"ptr": None})()
            refused(q35mix.ERR_INVALID, lambda: c.rows(1, [0], [0], [1], null, k), "null")
            refused(q35mix.ERR_INVALID, lambda: c.rows(1, [0], [0], [1], k, q35mix.DeviceView(k, 1, (1, 1024))), "aligned")
            ctx.sync()
