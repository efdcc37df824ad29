"""Paged K/V cache on the GPU: values at which an output could lose bits, range or its sign, against the plain
restatement in 64 bits of test_gpu_paged.py.  Each test states its own tolerance.

That file's bound of 2e-5 of the largest output counts fp32's roundings, a deviation of 9e-6.  Over an fp16 cache two
more belong to it, q and the weights to 2^-23 of themselves: 256 products of about 2 (a score of 32 in size) each off by
2^-23 of itself with random signs move the score by 16 * 2^-23 * 2 / sqrt(3) = 2.2e-6, and a weight's own rounding is
1.2e-7 of it.  In squares that is 9.3e-6, twice which the bound still covers."""
import numpy as np
import pytest

import q35mix
from q35mix import KV_F16, KV_F32
from test_gpu_paged import HD, TOL, Paged, cast, close_to, say

pytestmark = pytest.mark.gpu


def put_rows(p, seq, which, rows):
    """Cached rows 0 .. of a sequence: [n][kv head][256]."""
    t = np.arange(len(rows))
    p.pages[which][p.table[seq][t // p.R], :, t % p.R] = cast(rows, p.type)


def levels(p, n, tokens, score, salt=0):
    """A cache of n rows whose scores are score[j] in every head whatever the query, and inputs whose new rows score 0:
    every q row is 16 times the unit vector over the dims that are not rotated."""
    p.w = {"q_norm": np.zeros(HD, np.float32), "k_norm": np.full(HD, -1, np.float32)}
    p.ctx.set_attn_weights(0, p.w)
    dims = HD - 64
    K = np.zeros((n, p.nkv, HD), np.float32)
    K[..., 64:] = (np.asarray(score, np.float32) / np.sqrt(dims))[:, None, None]
    put_rows(p, 0, 0, K)
    x = {k: v.copy() for k, v in p.inputs(tokens, salt=salt).items()}
    qg = x["q_gate"].reshape(tokens, p.nh, 2, HD)
    qg[:, :, 0, :64], qg[:, :, 0, 64:] = 0, 1
    return x


def start(p, n):
    p.push()
    p.c.advance([0], [n])
    p.len[0] = n


# ------------------------------------------------------------------ weights far below the largest

@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
def test_prefill_weights_far_below_the_largest(kv_type):
    """One row 18.5 nats above 15000 others, 512 tokens (a workgroup keeps a tile for thousands of rows): together the
    others are 1.4e-4 of the output, half of whose dims hold nothing else.

    Tolerance, of the largest output (one): an fp16 weight's smallest step is 2^-24 with the largest at 2^6, so each is
    off by at most 2^-31 of the largest, 15500 * 2^-31 = 7.2e-6; the sums are fp32, and adding a unit's rows (an fp32
    cache: a step's), 16 a lane, to a sum that holds the large weight rounds by at most 2^-24 of it, 130 (260) times in
    the 8300 rows of a workgroup: 7.8e-6 (1.5e-5)."""
    n, T, sink = 15000, 512, 5
    with Paged(kv_type, max_rows=n + T, page_rows=256, spare=0) as p:
        score = np.zeros(n)
        score[sink] = 18.5
        x = levels(p, n, T, score, salt=74)
        rs = np.random.RandomState(1)
        V = rs.standard_normal((n, p.nkv, HD)).astype(np.float32)
        V[..., :128] = 1 + 0.5 * V[..., :128]
        V[sink, :, :128], V[sink, :, 128:] = 0, np.sign(V[sink, :, 128:])
        put_rows(p, 0, 1, V)
        start(p, n)
        out = p.ctx.array((T, p.nh * HD))
        p.c.attn_prefill(0, [0], [T], *p.dev(x, "q_gate", "k", "v"), out)
        p.put([0], [T], x)
        some = [0, 200, T - 1]
        want = p.attend([0], [T], x, some)[some]
        e = np.abs(out.download()[some] - want).max()
        say(f"weights of 2^-26.7, type {kv_type}: {e:.1e} of {np.abs(want).max():.2f}")
        assert e <= TOL


# ------------------------------------------------------------------ infinities

def same_kind(got, want, tol):
    """Infinities of the same sign, NaN where NaN, the rest within tol of the largest."""
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(np.isinf(got), inf) and np.array_equal(got[inf] > 0, want[inf] > 0)
    ok = np.isfinite(want)
    e = np.abs(got[ok] - want[ok]).max() / np.abs(want[ok]).max()
    assert e <= tol, e
    return int(inf.sum()), int(np.isnan(want).sum())


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
@pytest.mark.parametrize("n,T,sharp,nh", [(0, 30, 1, 16), (90, 40, 1, 16), (90, 40, 1, 4), (1700, 70, 1, 16), (1700, 70, 8, 16),
                                          (600, 20, 1, 64), (300, 1, 1, 16), (300, 1, 1, 4), (2500, 1, 8, 16), (2500, 1, 1, 64)])
def test_infinite_values(kv_type, n, T, sharp, nh):
    """A V of +-inf makes the output of every token that sees it that infinity in its dim and heads, however small its
    weight; infinities of both signs, or a NaN, make it NaN.  T = 1 runs the one-token kernels and a chunk of one.
    (sharp: cached K times 8, scores of deviation 32 nats.  TOL as in test_gpu_paged.py, scores 8 times the size.)"""
    with Paged(kv_type, nh=nh, n_seqs=2, max_rows=n + T, page_rows=32) as p:
        rs = np.random.RandomState(n + T)
        x = {k: v.copy() for k, v in p.inputs(T, salt=75).items()}
        xv = x["v"].reshape(T, p.nkv, HD)
        if n:
            K, V = (rs.standard_normal((n, p.nkv, HD)).astype(np.float32) for _ in range(2))
            K *= sharp
            V[n // 13, 0, 3] = np.inf                # seen by all
            V[n - 1, 1, 255] = -np.inf
            V[n // 2, 2, 9], V[n - 2, 2, 9] = np.inf, -np.inf
            V[n // 3, 3, 77] = np.nan
            V[3, 3, 200] = -1e6                      # infinite in fp16
            put_rows(p, 0, 0, K)
            put_rows(p, 0, 1, V)
            start(p, n)
        xv[T // 2, 1, 130] = np.inf                  # seen by some, of the other heads' rows by none
        xv[T - 1, 0, 4] = -np.inf
        xv[0, 2, 64], xv[T // 3, 2, 64] = -np.inf, np.inf if T > 1 else -np.inf
        xv[T // 4, 3, 8] = np.nan
        xv[T // 2, 3, 201] = 1e6
        args = p.dev(x, "q_gate", "k", "v")
        out = p.ctx.array((T, p.nh * HD))
        calls = [lambda: p.c.attn_prefill(0, [0], [T], *args, out)]
        if T == 1:
            calls.append(lambda: p.c.attn_decode(0, [0], *args, out))
        p.put([0], [T], x)
        with np.errstate(invalid="ignore"):
            want = p.attend([0], [T], x)
        # beside them what is finite, which for an fp32 cache holds values of 1e6 too
        big = np.abs(want) > 1e3
        for call in calls:
            out.upload(np.zeros(out.shape, np.float32))
            call()
            got = out.download()
            counts = same_kind(np.where(big & np.isfinite(want), 0, got), np.where(big & np.isfinite(want), 0, want), TOL * sharp)
            ok = big & np.isfinite(want)
            assert not ok.any() or np.abs(got[ok] - want[ok]).max() <= TOL * sharp * np.abs(want[ok]).max()
            say(f"infinities {T} behind {n} type {kv_type}: {counts[0]} infinite, {counts[1]} NaN")
            assert counts[0] and counts[1]
        p.check_pages()


# ------------------------------------------------------------------ the output gate

@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
@pytest.mark.parametrize("T", [1, 3, 40])
def test_gate_keeps_fp32_precision(kv_type, T):
    """V of ones, a first token that sees one row: its output is the gate's sigmoid, at -80 to 20.

    Tolerance, relative: the sigmoid's exponential and its reciprocal are an ulp off, 2^-23 each, the two sums between
    them, the product with it and the division by the sum of weights 2^-24 each: 2^-21."""
    with Paged(kv_type, max_rows=64) as p:
        x = {k: v.copy() for k, v in p.inputs(T, salt=76).items()}
        x["v"][:] = 1
        g = np.linspace(-80, 20, p.nh * HD).astype(np.float32).reshape(p.nh, HD)
        x["q_gate"].reshape(T, p.nh, 2, HD)[:, :, 1] = g
        args, out = p.dev(x, "q_gate", "k", "v"), p.ctx.array((T, p.nh * HD))
        want = (1 / (1 + np.exp(-g.astype(np.float64)))).ravel()
        calls = [lambda: p.c.attn_prefill(0, [0], [T], *args, out)]
        if T == 1:
            calls.append(lambda: p.c.attn_decode(0, [0], *args, out))
        for call in calls:
            call()
            e = np.abs(out.download()[0] / want - 1).max()
            say(f"gate, {T} tokens, type {kv_type}: {e / 2.0 ** -24:.2f} half steps")
            assert e <= 2.0 ** -21


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
def test_gates_without_bounds(kv_type):
    """Gates whose exponential overflows, infinite ones and NaN: 0, 1 and NaN."""
    gates = np.array([-np.inf, np.inf, np.nan, -1e30, 1e30, -3e38, 3e38, -200, 200, -1e5, 1e5, 0], np.float32)
    sig = np.array([0, 1, np.nan, 0, 1, 0, 1, 0, 1, 0, 1, 0.5], np.float32)
    for T in (1, 20):
        with Paged(kv_type, max_rows=32) as p:
            x = {k: v.copy() for k, v in p.inputs(T, salt=78).items()}
            x["v"][:] = 1
            x["q_gate"].reshape(T, p.nh, 2, HD)[:, :, 1] = np.resize(gates, HD)
            args, out = p.dev(x, "q_gate", "k", "v"), p.ctx.array((T, p.nh * HD))
            calls = [lambda: p.c.attn_prefill(0, [0], [T], *args, out)]
            if T == 1:
                calls.append(lambda: p.c.attn_decode(0, [0], *args, out))
            for call in calls:
                call()
                assert np.allclose(out.download().reshape(T, p.nh, HD), np.resize(sig, HD), rtol=2e-6, atol=1e-38, equal_nan=True)


# ------------------------------------------------------------------ fp32's range

def test_fp32_values_near_the_largest():
    """V of 2^119 over 230 rows (their sum with weights up to one stays below 2^127), in rows whose scores rise 9 nats
    past those of the rows before.  Tolerance: test_gpu_paged.py's."""
    n, T = 230, 3
    with Paged(KV_F32, max_rows=n + T, page_rows=16) as p:
        score = np.zeros(n)
        score[70:] = 9.0
        x = levels(p, n, T, score, salt=77)
        rs = np.random.RandomState(2)
        V = rs.uniform(1.0, 2.0, (n, p.nkv, HD)).astype(np.float32) * np.float32(2.0 ** 118)
        put_rows(p, 0, 1, V)
        start(p, n)
        x["v"][:] = rs.uniform(1.0, 2.0, x["v"].shape).astype(np.float32) * np.float32(2.0 ** 118)
        args = p.dev(x, "q_gate", "k", "v")
        out, one = p.ctx.array((T, p.nh * HD)), p.ctx.array((1, p.nh * HD))
        p.c.attn_decode(0, [0], *args, one)
        p.c.attn_prefill(0, [0], [T], *args, out)
        p.put([0], [T], x)
        want = p.attend([0], [T], x)
        close_to(one.download().astype(np.float64), want[:1])
        close_to(out.download().astype(np.float64), want)


# ------------------------------------------------------------------ prompts of many tiles

@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16])
@pytest.mark.parametrize("n,T,page", [(0, 2048, 64), (0, 1031, 16), (700, 1500, 128)])
def test_prompts_of_whole_and_cut_tiles(kv_type, n, T, page):
    """16 q heads on 4 kv heads: 2048 rows are two whole tiles a workgroup, paired first with last; the others are cut.
    Rows of tiles at both ends and in the middle.  Tolerance: test_gpu_paged.py's."""
    with Paged(kv_type, max_rows=n + T, page_rows=page, salt=7) as p:
        rs = np.random.RandomState(n + T)
        for which in range(2):
            put_rows(p, 0, which, rs.standard_normal((n, p.nkv, HD)).astype(np.float32))
        start(p, n)
        x = p.inputs(T, salt=79)
        out = p.ctx.array((T, p.nh * HD))
        p.c.attn_prefill(0, [0], [T], *p.dev(x, "q_gate", "k", "v"), out)
        p.put([0], [T], x)
        mid = T // 2 // 16 * 16
        some = sorted({*range(18), *range(mid - 2, mid + 18, 3), *range(T // 3, T // 3 + 33, 8), *range(T - 18, T)})
        e = close_to(out.download().astype(np.float64), p.attend([0], [T], x, some))
        say(f"prompt of {T} behind {n} type {kv_type}: {e:.1e}")
        p.check_pages()
