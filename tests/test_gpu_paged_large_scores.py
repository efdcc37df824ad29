"""Paged attention at scores of two millions and more (large norm weights, K values near the top of their type), where fp32
holds a score to a quarter and two scores differ by whole quarters: a softmax weight is then off by much, but every output is
a mean of the V values that its token sees, times a gate below one, and must be finite as they are (include/q35mix.h).
"""
import numpy as np
import pytest

import mx4_rows
from q35mix import KV_F16, KV_F32, KV_MXFP4
from test_gpu_paged import HD, Paged, cast, say
from test_gpu_paged_mx4 import Mx4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16, KV_MXFP4])
@pytest.mark.parametrize("base", [16384.0, -16384.0, 40960.0])
@pytest.mark.parametrize("T", [1, 48])
def test_scores_of_millions(kv_type, base, T):
    """All rows have the same large part of a score, 160 * 0.83 * base = 2.2e6 (in log2; 5.5e6) in size, and a random one of
    some tens, so the maximum moves on by every number of quarters."""
    n, nh, nkv = 30000, 16, 4
    kw = dict(nh=nh, nkv=nkv, max_rows=n + T, page_rows=256, spare=0)
    with (Mx4(**kw) if kv_type == KV_MXFP4 else Paged(kv_type, **kw)) as p:
        rng = np.random.RandomState(3)
        p.w = {"q_norm": np.full(HD, 7, np.float32), "k_norm": np.zeros(HD, np.float32)}
        p.ctx.set_attn_weights(0, p.w)
        x = {k: v.copy() for k, v in p.inputs(T, salt=77).items()}
        q = x["q_gate"].reshape(T, nh, 2, HD)[:, :, 0]
        q[..., :64], q[..., 64:224] = 0, 1
        q[..., 224:] = rng.choice([-1.0, 1.0], q[..., 224:].shape)
        K = np.zeros((n, nkv, HD), np.float32)
        K[..., 64:224] = base
        K[..., 224:] = rng.standard_normal((n, nkv, 32))
        V = rng.standard_normal((n, nkv, HD)).astype(np.float32)
        at = p.table[0][np.arange(n) // p.R], slice(None), np.arange(n) % p.R
        for which, rows in enumerate((K, V)):
            if kv_type == KV_MXFP4:
                p.codes[which][at], p.scales[which][at] = mx4_rows.encode(rows)
            else:
                p.pages[which][at] = cast(rows, kv_type)
        p.push()
        p.c.advance([0], [n])
        out = p.ctx.array((T, nh * HD))
        d = p.dev(x, "q_gate", "k", "v")
        p.c.attn_decode(0, [0], *d, out) if T == 1 else p.c.attn_prefill(0, [0], [T], *d, out)
        got = out.download()
        most = max(np.abs(V).max(), np.abs(x["v"]).max()) * 1.2          # (a 4-bit value is up to a seventh above its own)
        say(f"{int((~np.isfinite(got)).sum())} of {got.size} not finite")
        assert np.isfinite(got).all() and np.abs(got).max() <= most
