"""Paged K/V cache on the GPU: rows appended, attention of one new token and of
chunks of new tokens, against a plain restatement in 64 bits (numpy).

Tolerances.  Cache rows: the kernels form a K row in 64 bits and round it to
fp32, then to the cache's type; the restatement does the same, and two 64-bit
results a few 1e-16 apart round alike (they would have to straddle a rounding
border of relative spacing 2^-24: once in 1e8 values), so rows must be equal.
Outputs: everything after the cache is fp32.  A score (in units of log2, below
32 in size for these rows) is a sum of 256 products; each addition rounds by at
most 2^-25 * 32 = 9.5e-7, with random signs 16 * 9.5e-7 / sqrt(3) = 9e-6 over
the sum, which is the relative error of a weight; the output is a mean under
those weights.  2e-5 of the largest output covers two such deviations.
"""
import ctypes

import numpy as np
import pytest

import q35mix
import synth
from q35mix import KV_F16, KV_F32, STATE_KEYS, STATE_VALUES

pytestmark = pytest.mark.gpu

HD, HALF = 256, 32
TOL = 2e-5


def say(msg):
    print(msg, flush=True)


_libm = ctypes.CDLL("libm.so.6")
_libm.powf.restype, _libm.powf.argtypes = ctypes.c_float, [ctypes.c_float, ctypes.c_float]
FREQ = np.array([np.float32(1) / np.float32(_libm.powf(1e7, np.float32(i) / np.float32(HALF))) for i in range(HALF)],
                np.float32)
EPS = float(np.float32(1e-6))


def rope_norm(x, w, pos):
    """x [rows][heads][256] at positions pos [rows], in 64 bits."""
    ang = (np.asarray(pos, np.float32)[:, None] * FREQ).astype(np.float64)[:, None]
    c, s = np.cos(ang), np.sin(ang)
    y = x.astype(np.float64).copy()
    a, b = y[..., :HALF].copy(), y[..., HALF:2 * HALF].copy()
    y[..., :HALF], y[..., HALF:2 * HALF] = a * c - b * s, a * s + b * c
    return y / np.sqrt((y ** 2).mean(-1, keepdims=True) + EPS) * (1 + w.astype(np.float64))


def cast(x, kv_type):
    with np.errstate(over="ignore"):
        return x.astype(np.float32).astype(np.float16 if kv_type == KV_F16 else np.float32)


def bits(a):
    return a.view(np.uint16 if a.dtype == np.float16 else np.uint32)


class Paged:
    """A paged cache beside its plain restatement: pages as numpy arrays."""

    def __init__(self, kv_type, nh=16, nkv=4, n_seqs=1, max_rows=256, page_rows=16, salt=0, spare=3, layers=1, layer=0):
        self.type, self.nh, self.nkv, self.R = kv_type, nh, nkv, page_rows
        rec = [0 if l == layer else 1 for l in range(layers)]
        self.ctx = q35mix.Context(q35mix.qwen35_config(num_layers=layers, num_heads=nh, num_kv_heads=nkv,
                                                       is_recurrent=rec), n_seqs=1, kv_capacity=16)
        self.layer = layer
        self.w = synth.attn_weights(HD, salt=salt)
        self.ctx.set_attn_weights(layer, self.w)
        per = -(-max_rows // page_rows)
        self.n_pages = n_seqs * per + spare
        self.c = q35mix.PagedCache(self.ctx, n_seqs=n_seqs, max_rows=max_rows, n_pages=self.n_pages,
                                   page_rows=page_rows, kv_type=kv_type)
        order = np.random.RandomState(salt + 5).permutation(self.n_pages)[:n_seqs * per]
        self.table = order.reshape(n_seqs, per)
        for s in range(n_seqs):
            self.c.map(s, 0, self.table[s])
        self.len = [0] * n_seqs
        dt = np.float16 if kv_type == KV_F16 else np.float32
        shape = (self.n_pages, nkv, page_rows, HD)
        self.pages = [np.full(shape, np.nan, dt) for _ in range(2)]      # nothing may be read that was not written
        self.push()

    def close(self):
        self.c.close()
        self.ctx.close()

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def push(self):
        for kind, p in zip((STATE_KEYS, STATE_VALUES), self.pages):
            ptr, n = self.c.device_ptr(self.layer, kind)
            assert n == p.nbytes
            q35mix.check(q35mix.lib().q35m_copy_h2d(self.ctx.handle, ptr, p.ctypes.data, n))

    def pull(self):
        got = []
        for kind, p in zip((STATE_KEYS, STATE_VALUES), self.pages):
            ptr, n = self.c.device_ptr(self.layer, kind)
            a = np.empty_like(p)
            q35mix.check(q35mix.lib().q35m_copy_d2h(self.ctx.handle, a.ctypes.data, ptr, n))
            got.append(a)
        return got

    def seed_rows(self, lens, salt=0, scale=1.0):
        """Cached rows of normal values; the rest of every page stays NaN."""
        for s, n in enumerate(lens):
            for which, p in enumerate(self.pages):
                x = synth.normal(7000 + 31 * salt + 2 * s + which, n * self.nkv * HD).reshape(n, self.nkv, HD) * scale
                for r in range(n):
                    p[self.table[s][r // self.R], :, r % self.R] = cast(x[r], self.type)
        self.push()
        self.c.advance(list(range(len(lens))), list(lens))
        for s, n in enumerate(lens):
            self.len[s] = n

    def inputs(self, rows, salt=0):
        return synth.attn_inputs(max(rows, 1), self.nh, self.nkv, HD, salt=salt)

    def rows_of(self, s, n, which):
        t = np.arange(n)
        return self.pages[which][self.table[s][t // self.R], :, t % self.R]         # [n][kv head][256]

    def put(self, seqs, tokens, x):
        """The restatement of an append: writes self.pages, returns nothing."""
        at = 0
        for s, t in zip(seqs, tokens):
            k = rope_norm(x["k"][at:at + t].reshape(t, self.nkv, HD), self.w["k_norm"], self.len[s] + np.arange(t))
            v = x["v"][at:at + t].reshape(t, self.nkv, HD)
            for j in range(t):
                r = self.len[s] + j
                self.pages[0][self.table[s][r // self.R], :, r % self.R] = cast(k[j], self.type)
                self.pages[1][self.table[s][r // self.R], :, r % self.R] = cast(v[j], self.type)
            at += t

    def attend(self, seqs, tokens, x, some=None):
        """[sum of tokens][nh * 256] in 64 bits (rows `some` of each chunk only, the others NaN)."""
        G, outs, at = self.nh // self.nkv, [], 0
        for s, t in zip(seqs, tokens):
            qg = x["q_gate"][at:at + t].reshape(t, self.nh, 2, HD)
            at += t
            n = self.len[s] + t
            q = rope_norm(qg[:, :, 0], self.w["q_norm"], self.len[s] + np.arange(t)) / 16.0
            K, V = (self.rows_of(s, n, w).astype(np.float64) for w in (0, 1))
            out = np.full((t, self.nh, HD), np.nan)
            for j in range(t) if some is None else [a for a in some if a < t]:
                m = self.len[s] + j + 1
                for h in range(self.nh):
                    sc = K[:m, h // G] @ q[j, h]
                    p = np.exp(sc - sc.max())
                    out[j, h] = (p / p.sum()) @ V[:m, h // G]
            out /= 1 + np.exp(-qg[:, :, 1].astype(np.float64))
            outs.append(out.reshape(t, self.nh * HD))
        return np.concatenate(outs) if outs else np.zeros((0, self.nh * HD))

    def dev(self, x, *names):
        return [self.ctx.array(x[k].shape, x[k]) for k in names]

    def check_pages(self):
        for got, want in zip(self.pull(), self.pages):
            nan = np.isnan(want)
            assert np.array_equal(np.isnan(got), nan)
            bad = (bits(got) != bits(want)) & ~nan
            assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4])

    def step(self, lens):
        self.c.advance(list(range(len(lens))), lens)
        for s, t in enumerate(lens):
            self.len[s] += t


def close_to(got, want, tol=TOL):
    ok = ~np.isnan(want)
    e = float(np.max(np.abs(got[ok] - want[ok])) / np.max(np.abs(want[ok])))
    assert np.isfinite(got[ok]).all()
    assert e <= tol, e
    return e


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
@pytest.mark.parametrize("lens,tokens,page", [([0], [1], 16), ([15, 0, 33], [2, 0, 40], 16), ([100, 3], [1, 129], 64),
                                              ([0, 7, 1, 64], [300, 0, 1, 0], 32), ([1000], [24], 1024)])
def test_append(kv_type, lens, tokens, page):
    n = len(lens)
    with Paged(kv_type, n_seqs=n, max_rows=1024, page_rows=page, salt=n) as p:
        p.seed_rows(lens, salt=n)
        x = p.inputs(sum(tokens), salt=20 + n)
        k, v = p.dev(x, "k", "v")
        p.c.append(0, list(range(n)), tokens, k, v)
        p.put(range(n), tokens, x)
        p.check_pages()
        assert [p.c.length(s) for s in range(n)] == lens              # not moved


def test_append_far_positions_and_other_heads():
    """Positions where the rotation's angles are large, 1 and 5 kv heads."""
    for nh, nkv in ((8, 1), (5, 5)):
        with Paged(KV_F16, nh=nh, nkv=nkv, max_rows=200_000, page_rows=256, spare=0, salt=nkv) as p:
            p.c.advance([0], [199_990])
            p.len[0] = 199_990
            x = p.inputs(10, salt=3)
            p.c.append(0, [0], [10], *p.dev(x, "k", "v"))
            p.put([0], [10], x)
            p.check_pages()


def test_append_values_at_the_edges_of_fp16():
    """Overflow to infinity, subnormals, zeros of both signs, NaN: as numpy rounds them; a zero K row stays zero."""
    with Paged(KV_F16, nh=4, nkv=1, max_rows=32) as p:
        x = p.inputs(4)
        x = {k: v.copy() for k, v in x.items()}
        x["v"][0, :10] = [65504, 65519, 65520, 1e6, -1e30, 6e-8, 2.9e-8, 1e-30, -0.0, np.nan]
        x["v"][1, 0] = -np.inf
        x["k"][2] = 0
        x["k"][3] = 1e-20
        p.c.append(0, [0], [4], *p.dev(x, "k", "v"))
        p.put([0], [4], x)
        row = p.table[0][0]
        for got, want in zip(p.pull(), p.pages):
            assert np.array_equal(got[row, 0, :4], want[row, 0, :4], equal_nan=True)
            assert np.array_equal(np.signbit(got[row, 0, 0, :9]), np.signbit(want[row, 0, 0, :9]))


# ------------------------------------------------------------------ decode

@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
@pytest.mark.parametrize("nh,nkv", [(16, 4), (4, 4), (8, 4), (16, 2), (16, 1), (24, 1), (32, 1)])
def test_decode_head_counts(kv_type, nh, nkv):
    lens = [0, 1, 15, 16, 17, 63, 64, 130]
    with Paged(kv_type, nh=nh, nkv=nkv, n_seqs=len(lens), max_rows=160, page_rows=16, salt=nh) as p:
        p.seed_rows(lens, salt=nh + nkv)
        x = p.inputs(len(lens), salt=nh)
        out = p.ctx.array((len(lens), nh * HD))
        seqs = list(range(len(lens)))
        p.c.attn_decode(0, seqs, *p.dev(x, "q_gate", "k", "v"), out)
        p.put(seqs, [1] * len(lens), x)
        want = p.attend(seqs, [1] * len(lens), x)
        e = close_to(out.download(), want)
        say(f"decode {nh}/{nkv} type {kv_type}: {e:.1e}")
        p.check_pages()


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
@pytest.mark.parametrize("lens,page", [([5], 16), ([31], 16), ([32], 32), ([33, 31], 64), ([127, 128, 129], 16), ([255, 256], 128),
                                       ([2000, 3, 700], 16), ([5000], 256), ([511, 512, 513, 0, 1], 1024)])
def test_decode_lengths(kv_type, lens, page):
    n = len(lens)
    with Paged(kv_type, n_seqs=n, max_rows=max(lens) + 1, page_rows=page, salt=n) as p:
        p.seed_rows(lens, salt=40 + n)
        seqs = list(range(n))[::-1]                                  # any order
        x = p.inputs(n, salt=50)
        out = p.ctx.array((n, p.nh * HD))
        p.c.attn_decode(0, seqs, *p.dev(x, "q_gate", "k", "v"), out)
        p.put(seqs, [1] * n, x)
        e = close_to(out.download(), p.attend(seqs, [1] * n, x))
        say(f"decode {lens} pages of {page} type {kv_type}: {e:.1e}")
        p.check_pages()


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
def test_decode_full_batch(kv_type):
    """64 sequences of 0 to 700 rows, more head groups than compute units."""
    lens = [(37 * i * i) % 701 for i in range(64)]
    with Paged(kv_type, nh=8, nkv=4, n_seqs=64, max_rows=701, page_rows=32, salt=9) as p:
        p.seed_rows(lens, salt=2)
        x = p.inputs(64, salt=51)
        out = p.ctx.array((64, p.nh * HD))
        p.c.attn_decode(0, list(range(64)), *p.dev(x, "q_gate", "k", "v"), out)
        p.put(range(64), [1] * 64, x)
        say(f"decode of 64: {close_to(out.download(), p.attend(range(64), [1] * 64, x)):.1e}")
        p.check_pages()


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
def test_decode_sharp_and_flat_weights(kv_type):
    """Scores so far apart that one row takes all, and K rows of zeros (all rows alike)."""
    for scale in (40.0, 0.0):
        with Paged(kv_type, n_seqs=2, max_rows=700, page_rows=64) as p:
            p.seed_rows([600, 333], salt=4)
            for s, n in enumerate([600, 333]):
                t = np.arange(n)
                p.pages[0][p.table[s][t // p.R], :, t % p.R] = cast(p.rows_of(s, n, 0).astype(np.float32) * scale, kv_type)
            p.push()
            x = p.inputs(2, salt=52)
            out = p.ctx.array((2, p.nh * HD))
            p.c.attn_decode(0, [0, 1], *p.dev(x, "q_gate", "k", "v"), out)
            p.put([0, 1], [1, 1], x)
            # scores of 40 times the size are rounded 40 times as far
            close_to(out.download(), p.attend([0, 1], [1, 1], x), TOL * max(scale, 1.0))


@pytest.mark.parametrize("kv_type,up", [(KV_F32, 2.0 ** 20), (KV_F16, 2.0 ** 12)])
def test_extreme_norm_weights(kv_type, up):
    """q rows far beyond fp16's range over K rows as far below one (fp16 subnormals), and large V: q's fp16 halves are
    scaled into their range."""
    with Paged(kv_type, n_seqs=1, max_rows=300, page_rows=16) as p:
        p.w = {"q_norm": np.full(HD, up, np.float32), "k_norm": np.full(HD, 1 / up - 1, np.float32)}
        p.ctx.set_attn_weights(0, p.w)
        p.seed_rows([255], salt=6, scale=1 / up)
        t = np.arange(255)
        p.pages[1][p.table[0][t // p.R], :, t % p.R] = cast(p.rows_of(0, 255, 1).astype(np.float32) * (up * 512), kv_type)
        p.push()
        x = p.inputs(2, salt=53)
        out = p.ctx.array((2, p.nh * HD))
        p.c.attn_prefill(0, [0], [2], *p.dev(x, "q_gate", "k", "v"), out)
        p.put([0], [2], x)
        want = p.attend([0], [2], x)
        close_to(out.download(), want)
        p.c.attn_decode(0, [0], *p.dev(x, "q_gate", "k", "v"), out)     # the first token again
        close_to(out.download()[:1], want[:1])
        p.check_pages()


def test_decode_pool_beyond_4_gib():
    """Pages whose offsets pass 32 bits: the last pages of a pool of over 2^32 bytes."""
    pages, R = 4200, 1024                               # x 1 head x 1024 rows x 256 x 4 B = 4.1 GiB a layer's keys
    with q35mix.Context(q35mix.qwen35_config(num_layers=1, num_heads=4, num_kv_heads=1, is_recurrent=[0]), n_seqs=1,
                        kv_capacity=16) as ctx:
        w = synth.attn_weights(HD)
        ctx.set_attn_weights(0, w)
        with q35mix.PagedCache(ctx, 2, 2048, pages, R, KV_F32) as c:
            assert c.device_ptr(0, STATE_KEYS)[1] > 1 << 32
            T = 1100
            x = synth.attn_inputs(T + 1, 4, 1, HD, salt=8)
            c.map(0, 0, [0, 1])
            c.map(1, 0, [pages - 1, pages - 2])
            dev = lambda a: ctx.array(a.shape, a)  # noqa: E731
            outs, outd = ctx.array((2 * T, 4 * HD)), ctx.array((2, 4 * HD))
            twice = {k: np.concatenate([v[:T], v[:T]]) for k, v in x.items()}
            c.attn_prefill(0, [0, 1], [T, T], dev(twice["q_gate"]), dev(twice["k"]), dev(twice["v"]), outs)
            c.advance([0, 1], [T, T])
            last = {k: np.concatenate([v[T:], v[T:]]) for k, v in x.items()}
            c.attn_decode(0, [0, 1], dev(last["q_gate"]), dev(last["k"]), dev(last["v"]), outd)
            got, one = outs.download(), outd.download()
            assert np.isfinite(got).all() and np.max(np.abs(got[:T] - got[T:])) <= TOL * np.max(np.abs(got))
            assert np.max(np.abs(one[0] - one[1])) <= TOL * np.max(np.abs(one))


# ------------------------------------------------------------------ prefill

@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
@pytest.mark.parametrize("nh,nkv", [(16, 4), (4, 4), (8, 4), (16, 2), (16, 1), (24, 1), (32, 1)])
def test_prefill_head_counts(kv_type, nh, nkv):
    lens, tokens = [0, 61, 5], [70, 33, 0]
    with Paged(kv_type, nh=nh, nkv=nkv, n_seqs=3, max_rows=128, page_rows=16, salt=nh) as p:
        p.seed_rows(lens, salt=nh)
        x = p.inputs(sum(tokens), salt=60)
        out = p.ctx.array((sum(tokens), nh * HD))
        p.c.attn_prefill(0, [0, 1, 2], tokens, *p.dev(x, "q_gate", "k", "v"), out)
        p.put([0, 1, 2], tokens, x)
        e = close_to(out.download(), p.attend([0, 1, 2], tokens, x))
        say(f"prefill {nh}/{nkv} type {kv_type}: {e:.1e}")
        p.check_pages()


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
@pytest.mark.parametrize("lens,tokens,page", [([0], [1], 16), ([0], [2], 16), ([63], [1], 64), ([64], [1], 16), ([0], [15], 16),
                                              ([0], [16], 16), ([0], [17], 16), ([1], [64], 32), ([0], [65], 64), ([31], [130], 16),
                                              ([0, 0, 9], [1, 257, 3], 16), ([700, 0, 64], [5, 0, 48], 128)])
def test_prefill_lengths(kv_type, lens, tokens, page):
    n = len(lens)
    with Paged(kv_type, n_seqs=n, max_rows=max(a + b for a, b in zip(lens, tokens)), page_rows=page, salt=n) as p:
        p.seed_rows(lens, salt=70 + n)
        x = p.inputs(sum(tokens) + 3, salt=61)                        # three rows behind the last sequence
        x["q_gate"][-3:], x["k"][-3:], x["v"][-3:] = np.nan, np.nan, np.nan
        out = p.ctx.array((sum(tokens) + 3, p.nh * HD), np.full((sum(tokens) + 3, p.nh * HD), 77.0, np.float32))
        p.c.attn_prefill(0, list(range(n)), tokens, *p.dev(x, "q_gate", "k", "v"), out)
        p.put(range(n), tokens, x)
        got = out.download()
        e = close_to(got[:-3], p.attend(range(n), tokens, x))
        assert (got[-3:] == 77.0).all()                               # left as they were
        say(f"prefill {tokens} behind {lens} pages of {page} type {kv_type}: {e:.1e}")
        p.check_pages()


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
@pytest.mark.parametrize("start,T", [(3000, 40), (0, 700), (900, 333)])
def test_prefill_longer(kv_type, start, T):
    """Tiles cut between workgroups and joined again; some rows of each."""
    with Paged(kv_type, nh=8, nkv=2, max_rows=start + T, page_rows=64) as p:
        p.seed_rows([start], salt=5)
        x = p.inputs(T, salt=62)
        out = p.ctx.array((T, p.nh * HD))
        p.c.attn_prefill(0, [0], [T], *p.dev(x, "q_gate", "k", "v"), out)
        p.put([0], [T], x)
        some = sorted({0, 1, T // 3, T // 2, T // 2 + 17, T - 2, T - 1})
        e = close_to(out.download(), p.attend([0], [T], x, some))
        say(f"prefill {T} behind {start} type {kv_type}: {e:.1e}")
        p.check_pages()


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
def test_prefill_full_batch(kv_type):
    """64 sequences of 0 to 150 rows with chunks of 0 to 4 tokens each."""
    lens, tokens = [(29 * i * i) % 151 for i in range(64)], [(7 * i) % 5 for i in range(64)]
    T = sum(tokens)
    with Paged(kv_type, nh=4, nkv=2, n_seqs=64, max_rows=155, page_rows=16, salt=11) as p:
        p.seed_rows(lens, salt=3)
        x = p.inputs(T, salt=67)
        out = p.ctx.array((T, p.nh * HD))
        p.c.attn_prefill(0, list(range(64)), tokens, *p.dev(x, "q_gate", "k", "v"), out)
        p.put(range(64), tokens, x)
        say(f"prefill of 64: {close_to(out.download(), p.attend(range(64), tokens, x)):.1e}")
        p.check_pages()


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
@pytest.mark.parametrize("start,T", [(10, 113), (10, 118), (1, 127), (10, 241), (10, 246), (0, 256), (250, 7)])
def test_prefill_tiles_past_the_rows(kv_type, start, T):
    """A last tile whose 64 query rows reach past the chunk, and past the rows up to which tiles are not cut."""
    with Paged(kv_type, n_seqs=1, max_rows=start + T, page_rows=16, salt=6) as p:
        p.seed_rows([start], salt=1)
        x = p.inputs(T, salt=73)
        out = p.ctx.array((T, p.nh * HD))
        p.c.attn_prefill(0, [0], [T], *p.dev(x, "q_gate", "k", "v"), out)
        p.put([0], [T], x)
        close_to(out.download(), p.attend([0], [T], x, sorted({0, T // 2, max(T - 17, 0), max(T - 2, 0), T - 1})))
        p.check_pages()


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
@pytest.mark.parametrize("max_rows", [117, 128])
def test_a_sequence_filled_to_its_last_row(kv_type, max_rows):
    """A chunk and then single tokens up to row max_rows - 1; the next is refused."""
    with Paged(kv_type, n_seqs=1, max_rows=max_rows, page_rows=16, spare=0) as p:
        T = max_rows - 2
        x = p.inputs(max_rows, salt=68)
        parts = [{k: v[a:b] for k, v in x.items()} for a, b in ((0, T), (T, T + 1), (T + 1, T + 2))]
        some = [0, 15, 16, 63, 64, T - 1]
        for part, n in zip(parts, (T, 1, 1)):
            out = p.ctx.array((n, p.nh * HD))
            d = p.dev(part, "q_gate", "k", "v")
            p.c.attn_prefill(0, [0], [n], *d, out) if n > 1 else p.c.attn_decode(0, [0], *d, out)
            p.put([0], [n], part)
            close_to(out.download(), p.attend([0], [n], part, some if n > 1 else None))
            p.step([n])
        p.check_pages()
        for call in (lambda: p.c.attn_decode(0, [0], *d, out), lambda: p.c.attn_prefill(0, [0], [1], *d, out)):
            refused(q35mix.ERR_CAPACITY, call)


def test_fp32_values_far_beyond_fp16():
    """V of 2^100 in one head and of 2^-90 in another (2^-14 of it is still a normal number): fp32 all the way."""
    T, n = 37, 300
    with Paged(KV_F32, nh=4, nkv=2, n_seqs=1, max_rows=n + T, page_rows=64) as p:
        p.seed_rows([n], salt=9)
        scale = np.array([2.0 ** 100, 2.0 ** -90], np.float32)
        t = np.arange(n)
        p.pages[1][p.table[0][t // p.R], :, t % p.R] = p.rows_of(0, n, 1) * scale[:, None]
        p.push()
        x = {k: v.copy() for k, v in p.inputs(T, salt=69).items()}
        x["v"] = (x["v"].reshape(T, 2, HD) * scale[:, None]).reshape(T, 2 * HD)
        out, one = p.ctx.array((T, p.nh * HD)), p.ctx.array((1, p.nh * HD))
        d = p.dev(x, "q_gate", "k", "v")
        p.c.attn_decode(0, [0], *d, one)
        p.c.attn_prefill(0, [0], [T], *d, out)
        p.put([0], [T], x)
        want, got, first = p.attend([0], [T], x), out.download(), one.download()
        for heads in (slice(0, 2 * HD), slice(2 * HD, 4 * HD)):
            close_to(got[:, heads], want[:, heads])
            close_to(first[:, heads], want[:1, heads])
        p.check_pages()


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_prefill_values_not_finite_stay_where_they_are_seen(kv_type, value):
    """A V value that is not finite reaches the tokens that see its row, in its dim and heads, and no other output."""
    T, at, dim = 40, 21, 130
    with Paged(kv_type, n_seqs=2, max_rows=128, page_rows=16) as p:
        p.seed_rows([50, 10], salt=5)
        x = {k: v.copy() for k, v in p.inputs(2 * T, salt=63).items()}
        clean = p.ctx.array((2 * T, p.nh * HD))
        p.c.attn_prefill(0, [0, 1], [T, T], *p.dev(x, "q_gate", "k", "v"), clean)
        want = clean.download()
        x["v"][at, HD + dim] = value                                  # kv head 1 of sequence 0
        out = p.ctx.array((2 * T, p.nh * HD))
        p.c.attn_prefill(0, [0, 1], [T, T], *p.dev(x, "q_gate", "k", "v"), out)
        got = out.download().reshape(2 * T, p.nh, HD)
        hit = np.zeros(got.shape, bool)
        hit[at:T, 4:8, dim] = True
        assert not np.isfinite(got[hit]).any()
        assert np.array_equal(got[~hit], want.reshape(got.shape)[~hit])


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
def test_decode_and_prefill_rows_of_other_sequences_do_not_leak(kv_type):
    """NaN in one sequence's cached V leaves the others as they were."""
    with Paged(kv_type, n_seqs=3, max_rows=200, page_rows=16) as p:
        p.seed_rows([100, 150, 60], salt=5)
        x = p.inputs(3, salt=64)
        a, b = p.ctx.array((3, p.nh * HD)), p.ctx.array((3, p.nh * HD))
        p.c.attn_decode(0, [0, 1, 2], *p.dev(x, "q_gate", "k", "v"), a)
        p.c.attn_prefill(0, [0, 1, 2], [1, 1, 1], *p.dev(x, "q_gate", "k", "v"), b)
        before = a.download(), b.download()
        p.pages = p.pull()
        p.pages[1][p.table[1][2], :, 3] = np.nan
        p.push()
        p.c.attn_decode(0, [0, 1, 2], *p.dev(x, "q_gate", "k", "v"), a)
        p.c.attn_prefill(0, [0, 1, 2], [1, 1, 1], *p.dev(x, "q_gate", "k", "v"), b)
        for was, now in zip(before, (a.download(), b.download())):
            assert np.array_equal(was[[0, 2]], now[[0, 2]]) and np.isnan(now[1]).all()


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
def test_conversations(kv_type):
    """As a server uses them: a prompt in chunks, a second sequence that shares its
    first pages, the last layer's prompt rows appended without attention, decode
    steps of the batch across page borders, a truncation; the contiguous cache's
    mixers give the same outputs."""
    R, S = 16, 3
    with Paged(kv_type, n_seqs=S, max_rows=160, page_rows=R, salt=3) as p:
        with q35mix.Context(q35mix.qwen35_config(num_layers=1, is_recurrent=[0]), n_seqs=S, kv_capacity=160) as flat:
            flat.set_attn_weights(0, p.w)

            def both(seqs, tokens, salt, alone=False):
                x = p.inputs(sum(tokens), salt=salt)
                out = p.ctx.array((sum(tokens), p.nh * HD))
                args = p.dev(x, "q_gate", "k", "v")
                if all(t == 1 for t in tokens):
                    p.c.attn_decode(0, seqs, *args, out)
                else:
                    p.c.attn_prefill(0, seqs, tokens, *args, out)
                p.put(seqs, tokens, x)
                want = p.attend(seqs, tokens, x)
                got = out.download()
                close_to(got, want)
                at = 0
                for s, t in zip(seqs, tokens):
                    ref = flat.array((t, p.nh * HD))
                    flat.attn_prefill(0, s, t, *[flat.array((t, v.shape[1]), v[at:at + t]) for v in
                                                 (x["q_gate"], x["k"], x["v"])], ref)
                    # an fp16 cache differs by the rounding of its rows: 2^-11 a value of K moves a score (of
                    # deviation 4 here) by up to 16 x 2^-11 x 2 = 1.6e-2, a value of V by 2^-11 of itself
                    close_to(got[at:at + t], ref.download().astype(np.float64), 1e-4 if kv_type == KV_F32 else 2e-2)
                    flat.advance(s, t)
                    at += t
                p.c.advance(seqs, tokens)
                for s, t in zip(seqs, tokens):
                    p.len[s] += t

            both([0], [40], 80)                     # a prompt's first chunk
            both([0, 2], [25, 9], 81)               # its second beside another prompt
            # sequence 1 shares the first two pages (32 rows) of sequence 0
            own = p.table[1].copy()
            p.table[1][:2] = p.table[0][:2]
            p.c.map(1, 0, p.table[1][:2])
            p.c.advance([1], [2 * R])
            p.len[1] = 2 * R
            rows = [flat.state_read(0, 0, kind, 2 * R) for kind in (STATE_KEYS, STATE_VALUES)]
            for kind, r in zip((STATE_KEYS, STATE_VALUES), rows):
                flat.state_write(0, 1, kind, r)
            flat.advance(1, 2 * R)
            both([1], [21], 82)
            # a prompt whose attention nobody reads but its last token's
            x = p.inputs(30, salt=83)
            p.c.append(0, [2], [30], *p.dev(x, "k", "v"))
            p.put([2], [30], x)
            p.c.advance([2], [30])
            p.len[2] += 30
            scratch = flat.array((30, p.nh * HD))
            flat.attn_prefill(0, 2, 30, *[flat.array((30, v.shape[1]), v) for v in (x["q_gate"], x["k"], x["v"])], scratch)
            flat.advance(2, 30)
            for step in range(18):                  # over a page border of each
                both([2, 0, 1], [1, 1, 1], 90 + step)
            p.c.truncate(0, 70)
            p.len[0] = 70
            flat.truncate(0, 70)
            both([0, 1], [3, 1], 120)
            assert [p.c.length(s) for s in range(S)] == p.len
            # a write into the shared pages is refused, and the page is free again once remapped
            p.c.truncate(1, 20)
            with pytest.raises(q35mix.Q35Error) as e:
                p.c.append(0, [1], [1], *p.dev(x, "k", "v"))
            assert e.value.code == q35mix.ERR_INVALID and "read-only" in str(e.value)
            p.c.map(1, 0, own[:2])
            p.c.append(0, [1], [1], *p.dev(x, "k", "v"))
            p.ctx.sync()


def test_layers_keep_their_own_pages():
    """Two full-attention layers beside a linear one: the same page ids, each layer's own rows."""
    cfg = q35mix.qwen35_config(num_layers=3, is_recurrent=[0, 1, 0])
    with q35mix.Context(cfg, n_seqs=1, kv_capacity=16) as ctx:
        for l in (0, 2):
            ctx.set_attn_weights(l, synth.attn_weights(HD, salt=l))
        with q35mix.PagedCache(ctx, 1, 64, 4, 16, KV_F32) as c:
            c.map(0, 0, [3, 1, 0, 2])
            xs = [synth.attn_inputs(20, 16, 4, HD, salt=l) for l in (0, 2)]
            for l, x in zip((0, 2), xs):
                c.append(l, [0], [20], ctx.array(x["k"].shape, x["k"]), ctx.array(x["v"].shape, x["v"]))
            for l, x in zip((0, 2), xs):
                ptr, n = c.device_ptr(l, STATE_VALUES)
                a = np.empty((4, 4, 16, HD), np.float32)
                q35mix.check(q35mix.lib().q35m_copy_d2h(ctx.handle, a.ctypes.data, ptr, n))
                got = np.concatenate([a[3].transpose(1, 0, 2), a[1].transpose(1, 0, 2)[:4]]).reshape(20, -1)
                assert np.array_equal(got, x["v"])
                assert not a[[0, 2]].any() and not a[1, :, 4:].any()   # pages begin as zeros
            for call in (lambda: c.append(1, [0], [1], *[ctx.array((1, 1024))] * 2), lambda: c.device_ptr(1, STATE_KEYS)):
                with pytest.raises(q35mix.Q35Error):
                    call()


# ------------------------------------------------------------------ graphs

def capture(ctx, call):
    hip = q35mix.hip()
    stream, graph, exe = ctypes.c_void_p(ctx.stream), ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    try:
        call()
    finally:
        r = hip.hipStreamEndCapture(stream, ctypes.byref(graph))
    assert r == 0
    assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
    return graph, exe


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
def test_captured_calls_follow_lengths_and_pages(kv_type):
    """A decode step and a two-sequence chunk captured at short lengths and
    replayed over growing ones, across pages mapped after the capture, with
    eager calls between the replays: each replay equals the eager call."""
    hip = q35mix.hip()
    with Paged(kv_type, n_seqs=2, max_rows=2000, page_rows=32, salt=4) as p:
        p.seed_rows([3, 40], salt=8)
        p.c.unmap(0, 4, len(p.table[0]) - 4)
        x1, x2 = p.inputs(2, salt=65), p.inputs(9, salt=66)
        d1, d2 = p.dev(x1, "q_gate", "k", "v"), p.dev(x2, "q_gate", "k", "v")
        o1, o2 = p.ctx.array((2, p.nh * HD)), p.ctx.array((9, p.nh * HD))
        e1, e2 = p.ctx.array((2, p.nh * HD)), p.ctx.array((9, p.nh * HD))
        p.c.attn_decode(0, [0, 1], *d1, o1)
        graphs = [capture(p.ctx, lambda: p.c.attn_decode(0, [0, 1], *d1, o1)),
                  capture(p.ctx, lambda: p.c.attn_prefill(0, [1, 0], [4, 5], *d2, o2))]
        stream = ctypes.c_void_p(p.ctx.stream)
        try:
            for extra in (0, 30, 700, 1):
                need = -(-(p.c.length(0) + extra + 6) // 32)
                p.c.map(0, 0, p.table[0][:need])
                p.c.advance([0, 1], [extra, 2 * extra])
                for (g, exe), o, e, eager in ((graphs[0], o1, e1, lambda: p.c.attn_decode(0, [0, 1], *d1, e1)),
                                              (graphs[1], o2, e2, lambda: p.c.attn_prefill(0, [1, 0], [4, 5], *d2, e2))):
                    o.upload(np.zeros(o.shape, np.float32))
                    assert hip.hipGraphLaunch(exe, stream) == 0
                    p.ctx.sync()
                    got = o.download()
                    rows = p.pull()
                    eager()
                    want = e.download()
                    again = p.pull()
                    # rows never written are NaN behind `advance`: both sides see the same
                    assert np.array_equal(got.view(np.uint32), want.view(np.uint32))
                    assert all(np.array_equal(bits(a), bits(b)) for a, b in zip(rows, again))
        finally:
            for g, exe in graphs:
                assert hip.hipGraphExecDestroy(exe) == 0
                assert hip.hipGraphDestroy(g) == 0


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
@pytest.mark.parametrize("rows", [100, 127, 128, 129, 255, 256, 257, 511, 512])
def test_short_sequences_eager_and_replayed(kv_type, rows):
    """Lengths at which an eager call stops leaving a sequence to one workgroup; a replayed call, captured at another
    length, never does: both against the restatement."""
    hip = q35mix.hip()
    with Paged(kv_type, nh=8, nkv=2, n_seqs=2, max_rows=520, page_rows=32, salt=2) as p:
        p.seed_rows([rows - 1, rows - 3], salt=4)
        x1, x2 = p.inputs(2, salt=71), p.inputs(4, salt=72)
        d1, d2 = p.dev(x1, "q_gate", "k", "v"), p.dev(x2, "q_gate", "k", "v")
        o1, o2 = p.ctx.array((2, p.nh * HD)), p.ctx.array((4, p.nh * HD))
        calls = [lambda: p.c.attn_decode(0, [0, 1], *d1, o1), lambda: p.c.attn_prefill(0, [0, 1], [1, 3], *d2, o2)]
        p.c.truncate(0, 1)
        p.c.truncate(1, 1)
        graphs = [capture(p.ctx, c) for c in calls]
        p.c.advance([0, 1], [rows - 2, rows - 4])
        stream = ctypes.c_void_p(p.ctx.stream)
        try:
            for tokens, x, o, call, (_, exe) in (([1, 1], x1, o1, calls[0], graphs[0]), ([1, 3], x2, o2, calls[1], graphs[1])):
                p.put([0, 1], tokens, x)
                want = p.attend([0, 1], tokens, x)
                for run in (call, lambda exe=exe: hip.hipGraphLaunch(exe, stream)) * 2:
                    o.upload(np.zeros(o.shape, np.float32))
                    assert run() in (None, 0)
                    p.ctx.sync()
                    close_to(o.download(), want)
            p.check_pages()
        finally:
            for g, exe in graphs:
                assert hip.hipGraphExecDestroy(exe) == 0
                assert hip.hipGraphDestroy(g) == 0


def test_changes_are_refused_while_capturing():
    hip = q35mix.hip()
    with Paged(KV_F32, max_rows=64) as p:
        stream, graph = ctypes.c_void_p(p.ctx.stream), ctypes.c_void_p()
        assert hip.hipStreamBeginCapture(stream, 0) == 0
        try:
            for call in (lambda: p.c.map(0, 0, [1]), lambda: p.c.advance([0], [1]), lambda: p.c.truncate(0, 0)):
                with pytest.raises(q35mix.Q35Error) as e:
                    call()
                assert e.value.code == q35mix.ERR_INVALID and "captured" in str(e.value)
        finally:
            assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
            if graph.value:
                assert hip.hipGraphDestroy(graph) == 0
        p.c.advance([0], [1])
        assert p.c.length(0) == 1


# ------------------------------------------------------------------ refusals

def refused(code, call, word=""):
    with pytest.raises(q35mix.Q35Error) as e:
        call()
    assert e.value.code == code and word in str(e.value), str(e.value)


def test_refusals():
    """Nothing is enqueued for a refused call, and nothing changes."""
    cfg = q35mix.qwen35_config(num_layers=2, is_recurrent=[1, 0])
    with q35mix.Context(cfg, n_seqs=1, kv_capacity=16) as ctx:
        make = lambda **k: q35mix.PagedCache(ctx, **{**dict(n_seqs=2, max_rows=100, n_pages=8, page_rows=16,  # noqa: E731
                                                            kv_type=KV_F16), **k})
        for bad in ({"n_seqs": 0}, {"max_rows": 0}, {"n_pages": 0}, {"kv_type": 2}):
            refused(q35mix.ERR_INVALID, lambda: make(**bad))
        for bad in ({"page_rows": 8}, {"page_rows": 24}, {"page_rows": 2048}, {"page_rows": 0}, {"max_rows": (1 << 24) + 1}):
            refused(q35mix.ERR_UNSUPPORTED, lambda: make(**bad))
        with make() as c:
            k, q, out = ctx.array((8, 1024)), ctx.array((8, 8192)), ctx.array((8, 4096))
            refused(q35mix.ERR_INVALID, lambda: c.append(1, [0], [1], k, k), "weights")
            ctx.set_attn_weights(1, synth.attn_weights(HD))
            refused(q35mix.ERR_INVALID, lambda: c.append(0, [0], [1], k, k), "DeltaNet")
            refused(q35mix.ERR_INVALID, lambda: c.append(2, [0], [1], k, k), "layer")
            refused(q35mix.ERR_CAPACITY, lambda: c.append(1, [0], [1], k, k), "mapped")
            c.map(0, 0, range(7))
            c.map(1, 0, [7])
            refused(q35mix.ERR_INVALID, lambda: c.map(0, 0, [8]), "page")
            refused(q35mix.ERR_INVALID, lambda: c.map(0, 0, [-1]), "page")
            refused(q35mix.ERR_INVALID, lambda: c.map(2, 0, [1]), "sequence")
            refused(q35mix.ERR_RANGE, lambda: c.map(0, 6, [1, 2]))
            refused(q35mix.ERR_RANGE, lambda: c.map(0, -1, [1]))
            refused(q35mix.ERR_INVALID, lambda: c.append(1, [0, 0], [1, 1], k, k), "repeated")
            refused(q35mix.ERR_INVALID, lambda: c.append(1, [0], [-1], k, k), "tokens")
            refused(q35mix.ERR_INVALID, lambda: c.append(1, [2], [1], k, k), "sequence")
            refused(q35mix.ERR_CAPACITY, lambda: c.append(1, list(range(65)), [1] * 65, k, k), "64")
            refused(q35mix.ERR_CAPACITY, lambda: c.append(1, [1], [17], k, k), "mapped")
            refused(q35mix.ERR_CAPACITY, lambda: c.append(1, [0], [101], k, k), "exceed")
            refused(q35mix.ERR_CAPACITY, lambda: c.advance([0], [101]))
            refused(q35mix.ERR_INVALID, lambda: c.advance([0, 0], [1, 1]), "repeated")
            refused(q35mix.ERR_INVALID, lambda: c.advance([0], [-1]))
            refused(q35mix.ERR_CAPACITY, lambda: c.advance([], []))
            refused(q35mix.ERR_RANGE, lambda: c.truncate(0, 1))
            refused(q35mix.ERR_INVALID, lambda: c.truncate(0, -1))
            refused(q35mix.ERR_INVALID, lambda: c.truncate(5, 0))
            refused(q35mix.ERR_INVALID, lambda: c.length(-1))
            refused(q35mix.ERR_INVALID, lambda: c.device_ptr(1, q35mix.STATE_CONV))
            off = q35mix.DeviceView(q, 1, (4, 1024))
            null = type("Null", (), {"ptr": None})()
            for a in (off, null):
                refused(q35mix.ERR_INVALID, lambda: c.append(1, [0], [1], a, k))
                refused(q35mix.ERR_INVALID, lambda: c.append(1, [0], [1], k, a))
                refused(q35mix.ERR_INVALID, lambda: c.attn_decode(1, [0], a, k, k, out))
                refused(q35mix.ERR_INVALID, lambda: c.attn_decode(1, [0], q, k, k, a))
                refused(q35mix.ERR_INVALID, lambda: c.attn_prefill(1, [0], [2], q, a, k, out))
                refused(q35mix.ERR_INVALID, lambda: c.attn_prefill(1, [0], [2], q, k, k, a))
            c.append(1, [0, 1], [0, 0], k, k)                     # no rows: nothing to do
            c.attn_prefill(1, [0], [0], q, k, k, out)
            assert c.length(0) == 0 and c.length(1) == 0
            c.advance([0], [100])
            refused(q35mix.ERR_CAPACITY, lambda: c.attn_decode(1, [0], q, k, k, out), "exceed")
            ctx.sync()
    with q35mix.Context(q35mix.qwen35_config(num_layers=1, is_recurrent=[1]), n_seqs=1, kv_capacity=16) as ctx:
        refused(q35mix.ERR_INVALID, lambda: q35mix.PagedCache(ctx, 1, 16, 1, 16, KV_F32), "full-attention")


def test_kernel_timers():
    """Which kernels a call runs: parts are joined only where a sequence went to several workgroups."""
    with Paged(KV_F16, n_seqs=2, max_rows=700) as p:
        p.seed_rows([600, 5], salt=3)
        x = p.inputs(2)
        out = p.ctx.array((2, p.nh * HD))
        d = p.dev(x, "q_gate", "k", "v")

        def ran(seq):
            p.ctx.profile(True)
            p.c.attn_prefill(0, [seq], [2], *d, out)
            p.c.attn_decode(0, [seq], *d, out)
            names = sorted(p.ctx.profile_read())
            p.ctx.profile(False)
            return names

        assert ran(0) == ["paged_append_rows", "paged_decode", "paged_decode_merge", "paged_prefill", "paged_prefill_merge"]
        assert ran(1) == ["paged_append_rows", "paged_decode", "paged_prefill"]
