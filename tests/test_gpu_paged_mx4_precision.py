"""Paged K/V cache in 4 bits: what the attention holds of the softmax weights and of q, each shown where nothing else of the
result covers it.  Every tolerance is the promise of include/q35mix.h worked out for the test's rows.
"""
import numpy as np
import pytest

from test_gpu_paged import HD, say
from test_gpu_paged_mx4 import Mx4
from test_gpu_paged_mx4_values import level_inputs, put_rows, start

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ weights

@pytest.mark.parametrize("nh,nkv", [(16, 4), (8, 1), (16, 1)])
@pytest.mark.parametrize("n", [127, 4063])
def test_one_token_s_weights_far_below_the_largest(nh, nkv, n):
    """Every 32nd row is 23.09 nats, 33.32 in log2, above the others, which alone hold something in half of the dims.

    A weight is held to 2^-38 of the row's largest, so these dims are off by 2^-38 / 2^-33.32 = 2^-4.68 of themselves, 3.9 %,
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
        assert e <= 2.0 ** -4.68 + 1e-4
