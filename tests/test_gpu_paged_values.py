"""Paged K/V cache on the GPU: values at which an output could lose bits, range or its sign, against the plain
restatement in 64 bits of test_gpu_paged.py.  Each test states its own tolerance."""
import numpy as np
import pytest

from q35mix import KV_F16, KV_F32
from test_gpu_paged import HD, TOL, Paged, cast, say

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
