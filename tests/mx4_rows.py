"""Rows of a 4-bit cache, restated in numpy from the format's definition: blocks of 32 values share a power of two 2^s,
the smallest with the largest value at most 7 2^s, -23 <= s <= 13; a value is the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6
times it, a tie the one of even code, at most 6; a block with a value that is not finite is NaN."""
import numpy as np

LEVELS = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])


def encode(x):
    """x [..., 256] fp32: (codes [..., 128], scales [..., 8]), uint8."""
    b = np.ascontiguousarray(x, np.float32).reshape(*x.shape[:-1], 8, 32).astype(np.float64)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    top = np.abs(b).max(-1)
    m, e = np.frexp(np.where(top > 0, top, 2.0 ** -100) / 7)       # top / 7 = m 2^e, 1/2 <= m < 1: s = e - 1 at m = 1/2
    s = np.clip(np.where(m == 0.5, e - 1, e), -23, 13)
    y = np.abs(b) / 2.0 ** s[..., None]
    code = np.zeros(y.shape, np.uint8)
    for i in range(7):
        border = (LEVELS[i] + LEVELS[i + 1]) / 2
        code += (y >= border) if i % 2 else (y > border)
    code |= np.signbit(np.where(bad[..., None], 0.0, np.asarray(x, np.float32).reshape(b.shape))).astype(np.uint8) << 3
    code = code.reshape(*x.shape[:-1], 128, 2)
    return code[..., 0] | code[..., 1] << 4, np.where(bad, 255, s + 127).astype(np.uint8)


def decode(codes, scales):
    """The values that codes [..., 128] and scales [..., 8] stand for, fp32."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], 8, 32)
    v = np.where(c & 8, -LEVELS[c & 7], LEVELS[c & 7])
    unit = np.where(scales == 255, np.nan, 2.0 ** (np.where(scales == 255, 127, scales).astype(np.float64) - 127))
    return (v * unit[..., None]).astype(np.float32).reshape(*codes.shape[:-1], 256)


def to_pool(which, codes, scales):
    """codes [pages][kv heads][R][128], scales [..][8] as the library lays a layer's pages out: bytes [pages][heads][136 R]."""
    p, h, r = codes.shape[:3]
    s = scales.reshape(p, h, r // 16, 16, 8).transpose(0, 1, 2, 4, 3) if which else scales
    return np.ascontiguousarray(np.concatenate([codes.reshape(p, h, -1), np.ascontiguousarray(s).reshape(p, h, -1)], -1))


def from_pool(which, pool, rows):
    p, h = pool.shape[:2]
    codes = pool[..., :128 * rows].reshape(p, h, rows, 128)
    s = pool[..., 128 * rows:]
    s = s.reshape(p, h, rows // 16, 8, 16).transpose(0, 1, 2, 4, 3).reshape(p, h, rows, 8) if which else s.reshape(p, h, rows, 8)
    return codes.copy(), np.ascontiguousarray(s)
