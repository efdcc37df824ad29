"""Paged K/V cache in 4 bits: what the attention holds of the softmax weights and of q, each shown where nothing else of the
result covers it.  Every tolerance is the promise of include/q35mix.h worked out for the test's rows.
"""
import numpy as np
import pytest

import mx4_queries as mq
from test_gpu_paged import HD, say
from test_gpu_paged_mx4 import Mx4
from test_gpu_paged_mx4_values import level_inputs, put_rows, start

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ weights

@pytest.mark.parametrize("nh,nkv", [(16, 4), (8, 1), (16, 1)])
@pytest.mark.parametrize("n", [127, 4063])
def test_one_token_s_weights_far_below_the_largest(nh, nkv, n):
    """Every 32nd row is 23.09 nats, 33.32 in log2, above the others, which alone hold something in half of the dims.

    A weight is held to 2^-40 of the row's largest, so these dims are off by 2^-40 / 2^-33.32 = 2^-6.68 of themselves, 0.98 %,
    if all weights are rounded the same way, as they are where all scores are equal.  The fp32 sums and scores (33.32 to
    2^-24 of itself) are beside that 1e-4 at most."""
    with Mx4(nh=nh, nkv=nkv, max_rows=n + 1, page_rows=64, spare=0) as p:
        x = level_inputs(p, 1, salt=76)
        top = np.arange(0, n, 32)
        K = np.zeros((n, nkv, HD), np.float32)
        for block, v in zip(range(2, 8), (2, 2, 1.5, 1.5, 1.5, 1.5)):            # 320 / sqrt(192) = 23.09
            K[top, :, 32 * block:32 * block + 32] = v
        V = np.random.RandomState(1).standard_normal((n, nkv, HD)).astype(np.float32)
        V[..., :128] = 1 + 0.5 * V[..., :128]
        V[..., 128:] = 0
        V[top, :, :128], V[top, :, 128:] = 0, 1
        put_rows(p, 0, 0, K)
        put_rows(p, 0, 1, V)
        start(p, n)
        x["v"].reshape(1, nkv, HD)[..., 128:] = 0
        out = p.ctx.array((1, nh * HD))
        p.c.attn_decode(0, [0], *p.dev(x, "q_gate", "k", "v"), out)
        p.put([0], [1], x)
        got, want = (a.reshape(nh, HD)[:, :128] for a in (out.download().astype(np.float64), p.attend([0], [1], x)))
        e = np.abs(got - want).max() / np.abs(want).max()
        say(f"weights of 2^-33.3, {nh} heads on {nkv}, {n} rows: {e:.1e} of {np.abs(want).max():.1e}")
        assert e <= 2.0 ** -6.68 + 1e-4


# ------------------------------------------------------------------ q

def small_beside_large(p, seqs, tokens, seed):
    """Three cached rows a sequence, each with one K value, at a dim where every q row is small beside its block's largest;
    new rows score 0, and every V value is of size 1."""
    rng = np.random.RandomState(seed)
    p.w = {"q_norm": np.zeros(HD, np.float32), "k_norm": np.full(HD, -1, np.float32)}
    p.ctx.set_attn_weights(0, p.w)
    for s in range(seqs):
        K, V = np.zeros((3, p.nkv, HD), np.float32), rng.choice([-1.0, 1.0], (3, p.nkv, HD))
        np.put_along_axis(K, mq.places(rng, p.nkv, 3)[..., None], mq.K_OF, -1)
        put_rows(p, s, 0, K)
        put_rows(p, s, 1, V)
        p.len[s] = 3
    p.push()
    p.c.advance(list(range(seqs)), [3] * seqs)
    rows = seqs * tokens
    x = {k: v.copy() for k, v in p.inputs(rows, salt=seed).items()}
    x["q_gate"].reshape(rows, p.nh, 2, HD)[:, :, 0] = mq.queries(rng, rows, p.nh)
    x["v"][:] = rng.choice([-1.0, 1.0], x["v"].shape)
    return x


@pytest.mark.parametrize("nh,nkv", [(16, 4), (8, 4), (4, 4), (8, 1), (16, 1), (24, 1)])
@pytest.mark.parametrize("T", [1, 50])
def test_all_of_q_takes_part(nh, nkv, T):
    """The tolerances of tests/mx4_queries.py, which a lost digit or part misses by ten times (test_paged_mx4_queries.py)."""
    seqs = 24 if T == 1 else 2
    with Mx4(nh=nh, nkv=nkv, n_seqs=seqs, max_rows=3 + T, page_rows=16) as p:
        x = small_beside_large(p, seqs, T, seed=nh + T)
        out = p.ctx.array((seqs * T, nh * HD))
        d = p.dev(x, "q_gate", "k", "v")
        p.c.attn_decode(0, list(range(seqs)), *d, out) if T == 1 else p.c.attn_prefill(0, list(range(seqs)), [T] * seqs, *d, out)
        p.put(range(seqs), [T] * seqs, x)
        p.check_pages()
        e = np.abs(out.download() - p.attend(range(seqs), [T] * seqs, x)).max()
        tol = mq.TOL_ONE if T == 1 else mq.TOL_CHUNK
        say(f"q small beside large, {T} tokens, {nh} heads on {nkv}: {e:.1e} of {tol:.1e}")
        assert e <= tol
