"""The restatement of what the attention over a 4-bit cache holds of q (tests/mx4_queries.py): its bounds, and that the rows at
which the kernels are held to them would tell a part that is lost.
"""
import numpy as np
import pytest

import mx4_queries as mq


@pytest.mark.parametrize("seed", range(4))
def test_what_is_left(seed):
    rng = np.random.RandomState(seed)
    q = (rng.standard_normal((200, 256)) * 2.0 ** rng.randint(-20, 20, (200, 1))).astype(np.float32)
    u, b = mq.unit(q)
    assert ((4 * u <= np.abs(b).max(-1, keepdims=True)) & (np.abs(b).max(-1, keepdims=True) < 8 * u)).all()
    left = lambda got: (np.abs(got.reshape(b.shape) - b) / u)           # noqa: E731
    for n in (4, 5, 6):
        assert left(mq.digits(q, n)).max() <= 16.0 ** (1 - n) / 2
        # (4 significant bits: a value of 4 .. 7.5 leaves a quarter, of which the next part leaves an eighth of its unit, ..;
        # one next to 8 is cut at 7.5, and so may the ones after it be)
        e = left(mq.parts(q, n))
        assert e.max() <= 16.0 ** (1 - n) / 2 and (e[np.abs(b) < 2 * u] <= 16.0 ** -n).all()
    # of the block's largest value
    assert (left(mq.digits(q)) * u / np.abs(b).max(-1, keepdims=True)).max() <= 2.0 ** -23
    assert (left(mq.parts(q)) * u / np.abs(b).max(-1, keepdims=True)).max() <= 2.0 ** -19.95


def output(q, rows_of_k, V):
    """[rows][heads][256] in 64 bits: softmax over the K rows (one value each) and a row that scores 0."""
    s = np.take_along_axis(q[:, :, None], rows_of_k[None, :, :, None], 3)[..., 0] * mq.K_OF / 16
    s = np.concatenate([s, np.zeros(s.shape[:2] + (1,))], -1)
    p = np.exp(s - s.max(-1, keepdims=True))
    return np.einsum("rhk,hkd->rhd", p / p.sum(-1, keepdims=True), V)


@pytest.mark.parametrize("held,n,tol", [(mq.digits, 6, mq.TOL_ONE), (mq.parts, 5, mq.TOL_CHUNK)])
def test_a_lost_part_would_be_seen(held, n, tol):
    """All parts are well within the tolerance, one fewer is past twice as much."""
    rng = np.random.RandomState(7)
    q = mq.queries(rng, 64, 16).astype(np.float64)
    top = np.abs(q).max(-1)
    assert 6.2 < top.min() and top.max() < 6.8 and np.abs(q).reshape(64, 16, 8, 32)[..., 1:].max() < 0.25
    at = np.stack([mq.places(rng, 3, 1)[0] for _ in range(16)])                     # [heads][3 rows]
    V = rng.choice([-1.0, 1.0], (16, 4, 256))
    want = output(q, at, V)
    off = [np.abs(output(held(q.astype(np.float32), k), at, V) - want).max() for k in (n, n - 1)]
    print(off, tol)
    assert off[0] <= tol and off[1] > 2 * tol
