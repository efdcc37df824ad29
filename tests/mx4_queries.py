"""What the attention over a 4-bit cache holds of q, restated: a block of 32 dims as parts of few bits, each what the ones
before it left, a power of 16 below.  And rows at which that alone decides the outputs.

With u the power of two for which the block's largest value is in [4 u, 8 u):
  one new token   six digits, whole numbers of u, u / 16, ..: what is left is u / 2 16^-5 = 2^-21 u at most
  chunks          five values of 4 significant bits up to 7.5, from u, u / 16, .. on (3 bits behind the leading one,
                  steps of 1/8 below 2): a value below 2 u leaves 1/16 u, and so does each part after it of its own unit, so
                  that after five there is 16^-5 u = 2^-20 u left at most
"""
import numpy as np

HD, K_OF = 256, 384.0                # a K row's one value: 6 2^6


def unit(q):
    """u of each block of q [..., 256], as [..., 8, 1], and q in blocks."""
    b = q.reshape(*q.shape[:-1], 8, 32).astype(np.float64)
    return 2.0 ** (np.floor(np.log2(np.maximum(np.abs(b).max(-1, keepdims=True), 1e-30))) - 2), b


def digits(q, n=6):
    u, b = unit(q)
    got, left = np.zeros_like(b), b / u
    for k in range(n):
        d = np.rint(left)
        got += d * 16.0 ** -k * u
        left = (left - d) * 16
    return got.reshape(q.shape)


def parts(q, n=5):
    u, b = unit(q)
    got = np.zeros_like(b)
    for k in range(n):
        x = (b - got) / (u * 16.0 ** -k)
        step = 2.0 ** (np.clip(np.floor(np.log2(np.maximum(np.abs(x), 1e-30))), 0, 2) - 3)
        got += np.clip(np.rint(x / step) * step, -7.5, 7.5) * u * 16.0 ** -k
    return got.reshape(q.shape)


def queries(rng, rows, heads):
    """q rows with one value of about 6.5 in each block of the dims that are not rotated, a thirtieth of it elsewhere there:
    normed to 16 as they are (the norm's weights being zeros)."""
    q = rng.uniform(0.6, 1.0, (rows, heads, HD)) * rng.choice([-1, 1], (rows, heads, HD)) * 0.22
    q[..., :64] = 0
    q[..., 64::32] = 6.5 * np.sign(q[..., 64::32])
    q *= 16 / np.sqrt((q * q).sum(-1, keepdims=True))
    return q.astype(np.float32)


def places(rng, kv_heads, rows):
    """Dims of small values, one for each K row of each kv head: [rows][kv_heads]."""
    d = rng.randint(1, 32, (rows, kv_heads)) + 32 * rng.randint(2, 8, (rows, kv_heads))
    return d


# A score is q_d 384 / 16, up to 0.25 24 = 6; the largest value of a block is 6.3 to 6.7, u = 1.
# What is left of q moves a score by 24 of it; fp32's sum of squares, root and products by 4 half steps of 2^-24 of the score,
# 1.5e-6, and its weights, sums and quotient by as many of the output.  An output, of values V of size 1, moves by no more than
# the scores do (sum of p |V - o| <= 1), and the gate is below one.
TOL_ONE = 24 * 2.0 ** -21 + 4e-6
TOL_CHUNK = 24 * 2.0 ** -20 + 4e-6
