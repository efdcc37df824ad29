"""Paged K/V cache in 4 bits at its limits: weights far apart, rows and queries that are not finite, long caches, pools of
more than 2^32 bytes, prompts whose tiles come out whole, graphs in turn.  Tolerance: test_gpu_paged_mx4.py's, unless
a test says otherwise.
"""
import numpy as np
import pytest

import mx4_rows
import q35mix
import synth
from q35mix import KV_F16, KV_F32, KV_MXFP4
from test_gpu_paged import HD, TOL, Paged, close_to, say
from test_gpu_paged_mx4 import Mx4, capture, decode, prefill

pytestmark = pytest.mark.gpu


def make(kv_type, **kw):
    return Mx4(**kw) if kv_type == KV_MXFP4 else Paged(kv_type, **kw)


def put_rows(p, seq, which, rows):
    """Cached rows 0 .. of a sequence: [n][kv head][256]."""
    t = np.arange(len(rows))
    at = p.table[seq][t // p.R], slice(None), t % p.R
    p.codes[which][at], p.scales[which][at] = mx4_rows.encode(np.asarray(rows, np.float32))


def start(p, n):
    p.push()
    p.c.advance([0], [n])
    p.len[0] = n


def level_inputs(p, tokens, salt=0):
    """Inputs whose q rows are 16 times the unit vector over the dims that are not rotated, and whose new rows score 0."""
    p.w = {"q_norm": np.zeros(HD, np.float32), "k_norm": np.full(HD, -1, np.float32)}
    p.ctx.set_attn_weights(0, p.w)
    x = {k: v.copy() for k, v in p.inputs(tokens, salt=salt).items()}
    qg = x["q_gate"].reshape(tokens, p.nh, 2, HD)
    qg[:, :, 0, :64], qg[:, :, 0, 64:] = 0, 1
    return x


# ------------------------------------------------------------------ weights far apart

@pytest.mark.parametrize("T", [1, 512])
def test_weights_far_below_the_largest(T):
    """One row about 18.5 nats above 15000 others: together the others are 1.4e-4 of the output, half of whose dims hold
    nothing else.

    Tolerance, of the largest output (one): a weight's smallest step is 2^-24 with the largest at 2^6, so each is off by at
    most 2^-31 of the largest, 15500 * 2^-31 = 7.2e-6; adding a unit's rows to an fp32 sum that holds the large weight
    rounds by at most 2^-24 of it, 130 times in a workgroup's 8300 rows: 7.8e-6.  Together 1.5e-5."""
    n, sink = 15000, 5
    with Mx4(max_rows=n + T, page_rows=256, spare=0) as p:
        x = level_inputs(p, T, salt=74)
        K = np.zeros((n, p.nkv, HD), np.float32)
        for block, v in zip(range(2, 8), (1.5, 1.5, 1.0, 1.5, 1.5, 1.0)):       # (1.33 sqrt(192) = 18.5)
            K[sink, :, 32 * block:32 * block + 32] = v
        rs = np.random.RandomState(1)
        V = rs.standard_normal((n, p.nkv, HD)).astype(np.float32)
        V[..., :128] = 1 + 0.5 * V[..., :128]
        V[sink, :, :128], V[sink, :, 128:] = 0, np.sign(V[sink, :, 128:])
        put_rows(p, 0, 0, K)
        put_rows(p, 0, 1, V)
        start(p, n)
        out = p.ctx.array((T, p.nh * HD))
        d = p.dev(x, "q_gate", "k", "v")
        p.c.attn_decode(0, [0], *d, out) if T == 1 else p.c.attn_prefill(0, [0], [T], *d, out)
        p.put([0], [T], x)
        some = sorted({0, T // 2, T - 1})
        want = p.attend([0], [T], x, some)[some]
        e = np.abs(out.download()[some] - want).max()
        say(f"weights of 2^-26.7, {T} tokens: {e:.1e} of {np.abs(want).max():.2f}")
        assert e <= TOL


@pytest.mark.parametrize("T", [1, 70])
@pytest.mark.parametrize("order", ["up", "down", "saw"])
def test_scores_that_rise_and_fall(order, T):
    """Scores from -40 to 40 nats along the rows: the maximum that weights refer to moves all along.  Two rows' weights
    differ by the rounding of their scores alone: 58 in log2, whose sums of 20 products of blocks round by 2^-19 each, 5e-6
    with random signs; what is held of q is the same factor in all of them, 2^-20, and 1e-6 of a difference of one."""
    n = 3000
    with Mx4(max_rows=n + T, page_rows=64, spare=0) as p:
        x = level_inputs(p, T, salt=75)
        level = {"up": np.linspace(-40, 40, n), "down": np.linspace(40, -40, n), "saw": 40 * np.sin(np.arange(n) * 0.7)}[order]
        K = np.zeros((n, p.nkv, HD), np.float32)
        K[..., 64:] = (level / np.sqrt(192))[:, None, None]
        put_rows(p, 0, 0, K)
        put_rows(p, 0, 1, np.random.RandomState(2).standard_normal((n, p.nkv, HD)))
        start(p, n)
        out = p.ctx.array((T, p.nh * HD))
        d = p.dev(x, "q_gate", "k", "v")
        p.c.attn_decode(0, [0], *d, out) if T == 1 else p.c.attn_prefill(0, [0], [T], *d, out)
        p.put([0], [T], x)
        say(close_to(out.download().astype(np.float64), p.attend([0], [T], x)))


# ------------------------------------------------------------------ what is not finite

def test_keys_and_queries_that_are_not_finite():
    """A K row that is not finite reaches the tokens that see it, a query row its own head, a gate its own value."""
    T = 70
    with Mx4(max_rows=512, page_rows=16) as p:
        p.seed_rows([130], salt=5)
        x = p.inputs(T, salt=6)
        y = {k: v.copy() for k, v in x.items()}
        y["k"].reshape(T, 4, HD)[11, 0, 37] = np.inf
        y["k"].reshape(T, 4, HD)[40, 1, 200] = np.nan
        qg = y["q_gate"].reshape(T, 16, 2, HD)
        qg[20, 9, 0, 5], qg[21, 10, 0, 100], qg[22, 11, 1, 7] = np.inf, np.nan, np.nan
        out = p.ctx.array((T, p.nh * HD))
        p.c.attn_prefill(0, [0], [T], *p.dev(y, "q_gate", "k", "v"), out)
        with np.errstate(invalid="ignore"):
            p.put([0], [T], y)
        p.check_pages()
        got = out.download().reshape(T, 16, HD)
        any_value = np.zeros((T, 16, HD), bool)
        any_value[11:, :4] = any_value[40:, 4:8] = any_value[20, 9] = any_value[21, 10] = any_value[22, 11, 7] = True
        assert np.isnan(got[20, 9]).all() and np.isnan(got[21, 10]).all() and np.isnan(got[22, 11, 7])
        for s in p.scales:
            s[s == 255] = 127                                   # (what the others' results are made of stays)
        close_to(got, np.where(any_value, np.nan, p.attend([0], [T], x).reshape(T, 16, HD)))


def test_one_token_s_queries_that_are_not_finite():
    with Mx4(n_seqs=3, max_rows=1024, page_rows=64) as p:
        p.seed_rows([900, 33, 400], salt=7)
        x = p.inputs(3, salt=8)
        y = {k: v.copy() for k, v in x.items()}
        qg = y["q_gate"].reshape(3, 16, 2, HD)
        qg[0, 3, 0, 250], qg[1, 6, 0, 0], qg[2, 15, 1, 9] = np.nan, -np.inf, np.nan
        y["k"].reshape(3, 4, HD)[1, 2, 8] = np.nan
        out = p.ctx.array((3, p.nh * HD))
        p.c.attn_decode(0, [0, 1, 2], *p.dev(y, "q_gate", "k", "v"), out)
        with np.errstate(invalid="ignore"):
            p.put([0, 1, 2], [1, 1, 1], y)
        p.check_pages()
        got = out.download().reshape(3, 16, HD)
        any_value = np.zeros((3, 16, HD), bool)
        any_value[0, 3] = any_value[1, 6] = any_value[2, 15, 9] = any_value[1, 8:12] = True
        assert np.isnan(got[0, 3]).all() and np.isnan(got[1, 6]).all() and np.isnan(got[2, 15, 9])
        for s in p.scales:
            s[s == 255] = 127
        close_to(got, np.where(any_value, np.nan, p.attend([0, 1, 2], [1, 1, 1], x).reshape(3, 16, HD)))


# ------------------------------------------------------------------ long caches, large pools

def test_a_long_cache():
    with Mx4(nh=8, nkv=1, n_seqs=2, max_rows=70100, page_rows=256) as p:
        p.seed_rows([70001, 33], salt=3)
        say(decode(p, [1, 0], p.len, 4))
        p.step([1, 1])
        say(prefill(p, [0, 1], [40, 3], 5, some=[0, 1, 2, 39]))


def test_a_pool_of_more_than_4_gib():
    """The last pages of a pool give what the first pages of a small one do."""
    with q35mix.Context(q35mix.qwen35_config(num_layers=1, num_heads=16, num_kv_heads=4, is_recurrent=[0]), n_seqs=1,
                        kv_capacity=16) as ctx:
        ctx.set_attn_weights(0, synth.attn_weights(HD, salt=1))
        x = synth.attn_inputs(1500, 16, 4, HD, salt=2)
        d = [ctx.array(x[k].shape, x[k]) for k in ("q_gate", "k", "v")]
        got = []
        for n_pages, pages in ((8000, [7999, 7998, 7993]), (3, [0, 1, 2])):
            with q35mix.PagedCache(ctx, n_seqs=1, max_rows=3000, n_pages=n_pages, page_rows=1024, kv_type=KV_MXFP4) as c:
                assert n_pages == 3 or c.device_ptr(0, q35mix.STATE_KEYS)[1] > 2 ** 32
                c.map(0, 0, pages[:3])
                a, b, e = ctx.array((1500, 4096)), ctx.array((1, 4096)), ctx.array((1500, 4096))
                held = ctx.array((2501, 1024)), ctx.array((2501, 1024))
                c.attn_prefill(0, [0], [1500], *d, a)
                c.advance([0], [1500])
                c.attn_decode(0, [0], *d, b)
                c.advance([0], [1])
                c.append(0, [0], [1000], d[1], d[2])
                c.rows(0, [0], [0], [2501], *held)
                c.advance([0], [1000])
                c.attn_prefill(0, [0], [400], *d, e)
                got.append([t.download() for t in (a, b, *held)] + [e.download()[:400]])
        for one, other in zip(*got):
            assert np.isfinite(one).all() and np.array_equal(one, other)


# ------------------------------------------------------------------ prompts of whole and cut tiles

@pytest.mark.parametrize("n,T,page", [(0, 2048, 64), (64, 2048, 16), (700, 1500, 128), (0, 1000, 32), (0, 1100, 64), (2000, 1500, 256),
                                      (30, 2500, 1024), (3000, 64, 16)])
def test_prompts_of_whole_and_cut_tiles(n, T, page):
    """16 q heads on 4 kv heads: one to three whole tiles a workgroup, in pairs of first and last, or tiles cut anywhere."""
    with Mx4(max_rows=n + T, page_rows=page, salt=7) as p:
        p.seed_rows([n], salt=n)
        mid = T // 2 // 16 * 16
        some = sorted({*range(18), *range(mid - 2, mid + 18, 3), *range(T // 3, T // 3 + 33, 8), *range(T - 18, T)})
        say(prefill(p, [0], [T], 79, some=some))


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16, KV_MXFP4])
@pytest.mark.parametrize("lens,tokens", [([0], [2048]), ([0, 0], [1024, 1024]), ([0, 64], [1024, 1024]), ([32, 32], [1024, 1024]),
                                         ([0, 0, 0], [1024, 0, 1023]), ([17, 17], [1024, 1024])])
def test_prompts_joined_or_not(kv_type, lens, tokens):
    """A call whose tiles all come out whole ends with them; a replay, whose host cannot know, launches the joining too:
    the same."""
    with make(kv_type, n_seqs=len(lens), max_rows=2112, page_rows=64) as p:
        p.seed_rows(lens, salt=1)
        seqs, rows = list(range(len(lens))), sum(tokens)
        x = p.inputs(rows, salt=80)
        d = p.dev(x, "q_gate", "k", "v")
        out, again = (p.ctx.array((rows, p.nh * HD), np.full((rows, p.nh * HD), 3, np.float32)) for _ in range(2))
        p.c.attn_prefill(0, seqs, tokens, *d, out)
        launch, end = capture(p, lambda: p.c.attn_prefill(0, seqs, tokens, *d, again))
        want = out.download()
        for _ in range(3):
            launch()
            assert np.array_equal(again.download(), want)
        end()
        assert np.isfinite(want).all()


@pytest.mark.parametrize("lens", [[600] * 16, [511, 0, 700], [1100] * 40 + [7] * 24, [3000] * 3, [2000] * 20, [130, 500, 900, 1300]])
def test_sequences_joined_or_not(lens):
    """One new token: sequences left whole and cut; a replay decides alike, from the lengths of its time."""
    with Mx4(n_seqs=len(lens), max_rows=max(lens) + 1, page_rows=128, nh=8, nkv=4) as p:
        p.seed_rows(lens, salt=2)
        decode(p, range(len(lens)), lens, 9)
        x, n = p.inputs(len(lens), salt=9), len(lens)
        d, out, again = p.dev(x, "q_gate", "k", "v"), p.ctx.array((n, p.nh * HD)), p.ctx.array((n, p.nh * HD))
        p.c.attn_decode(0, list(range(n)), *d, out)
        launch, end = capture(p, lambda: p.c.attn_decode(0, list(range(n)), *d, again))
        for _ in range(2):
            launch()
            assert np.array_equal(again.download(), out.download())
        p.c.truncate(0, lens[0] // 3)                           # (the graph's first choice may no longer hold)
        p.c.attn_decode(0, list(range(n)), *d, out)
        launch()
        assert np.array_equal(again.download(), out.download())
        end()


# ------------------------------------------------------------------ graphs in turn

def test_two_graphs_and_eager_calls_in_turn():
    """They share a workspace, in order."""
    with Mx4(n_seqs=2, max_rows=1500, page_rows=32) as p:
        p.seed_rows([900, 40], salt=1)
        x, y = p.inputs(2, salt=2), p.inputs(300, salt=3)
        out, outp, eager = p.ctx.array((2, p.nh * HD)), p.ctx.array((300, p.nh * HD)), p.ctx.array((300, p.nh * HD))
        d, e = p.dev(x, "q_gate", "k", "v"), p.dev(y, "q_gate", "k", "v")
        held = p.ctx.array((300, p.nkv * HD)), p.ctx.array((300, p.nkv * HD))
        p.c.attn_decode(0, [0, 1], *d, out)
        p.c.attn_prefill(0, [1, 0], [100, 200], *e, outp)
        one, end_one = capture(p, lambda: p.c.attn_decode(0, [0, 1], *d, out))
        two, end_two = capture(p, lambda: (p.c.attn_prefill(0, [1, 0], [100, 200], *e, outp), p.c.rows(0, [0], [900], [200], *held)))
        some = [0, 63, 99, 150, 199]
        for step in range(3):
            one()
            p.put([0, 1], [1, 1], x)
            close_to(out.download(), p.attend([0, 1], [1, 1], x))
            two()
            p.put([1, 0], [100, 200], y)
            want = p.attend([1, 0], [100, 200], y, some=some)
            close_to(outp.download(), want)
            p.c.attn_prefill(0, [1, 0], [100, 200], *e, eager)
            close_to(eager.download(), want)
            for which, h in enumerate(held):
                assert np.array_equal(h.download()[:200 - step], p.rows_of(0, 1100 - step, which)[900:].reshape(-1, 1024))
            p.check_pages()
            p.step([1, 1])
        end_one()
        end_two()


def test_timers_name_the_kernels():
    with Mx4(n_seqs=1, max_rows=4096, page_rows=64) as p:
        p.seed_rows([4000], salt=1)
        x = p.inputs(9, salt=2)
        d, out = p.dev(x, "q_gate", "k", "v"), p.ctx.array((9, p.nh * HD))
        p.ctx.profile(True)
        p.c.attn_decode(0, [0], *d, out)
        p.c.attn_prefill(0, [0], [9], *d, out)
        p.c.rows(0, [0], [0], [9], d[1], d[2])
        ran = p.ctx.profile_read()
        p.ctx.profile(False)
        assert sorted(ran) == ["paged_append_rows", "paged_decode", "paged_decode_merge", "paged_prefill", "paged_prefill_merge",
                               "paged_rows"]


@pytest.mark.parametrize("lens,tokens", [([0], [300]), ([0], [1500]), ([900, 3, 0, 40], [100, 0, 700, 33]), ([1700], [16]),
                                         ([1000, 1900], [1, 2]), ([0] * 6, [290, 301, 16, 1, 205, 300])])
def test_replayed_chunks_are_divided_alike(lens, tokens):
    """Tiles are left whole or cut by a rule on the lengths, which a replay reads where they are."""
    with Mx4(n_seqs=len(lens), max_rows=2000, page_rows=64, nh=16, nkv=4) as p:
        p.seed_rows(lens, salt=1)
        seqs, rows = list(range(len(lens))), sum(tokens)
        x = p.inputs(rows, salt=81)
        d = p.dev(x, "q_gate", "k", "v")
        out, again = p.ctx.array((rows, p.nh * HD)), p.ctx.array((rows, p.nh * HD))
        launch, end = capture(p, lambda: p.c.attn_prefill(0, seqs, tokens, *d, again))
        for shorter in (1, 3):
            p.c.attn_prefill(0, seqs, tokens, *d, out)
            launch()
            assert np.array_equal(again.download(), out.download()) and np.isfinite(out.download()).all()
            for s, n in enumerate(lens):
                p.c.truncate(s, n // 3)
        end()


# ------------------------------------------------------------------ queries of every size

@pytest.mark.parametrize("T", [1, 40])
def test_queries_of_every_size(T):
    """q rows of zeros, of values whose squares vanish in fp32, of one value among zeros, of sizes 2^-12 apart within a
    block, and norm weights of 8.  The last make scores 8 times test_gpu_paged_mx4.py's, and so 8 times what q's rounding
    leaves of them, 1.9e-5, with the sums' 9e-6: 6e-5 covers two deviations of both together."""
    with Mx4(max_rows=512, page_rows=32) as p:
        p.w["q_norm"][:] = 7
        p.ctx.set_attn_weights(0, p.w)
        p.seed_rows([333], salt=2)
        x = {k: v.copy() for k, v in p.inputs(T, salt=3).items()}
        q = x["q_gate"].reshape(T, p.nh, 2, HD)[:, :, 0]
        q[:, 0] = 0
        q[:, 1] *= np.float32(1e-30)
        q[:, 2, 1:] = 0
        q[:, 3] *= np.exp2(np.random.RandomState(4).randint(-12, 1, (T, HD))).astype(np.float32)
        q[:, 4] *= np.float32(1e15)
        out = p.ctx.array((T, p.nh * HD))
        d = p.dev(x, "q_gate", "k", "v")
        p.c.attn_decode(0, [0], *d, out) if T == 1 else p.c.attn_prefill(0, [0], [T], *d, out)
        p.put([0], [T], x)
        say(close_to(out.download(), p.attend([0], [T], x), tol=6e-5))
