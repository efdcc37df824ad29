"""Attention of sequences whose lengths and tables the device alone has, at sizes where work is cut and joined: chunks and
single tokens behind hundreds and thousands of rows that a plan says are there, eager and replayed at the lengths of the
replay's time, over all three cache types; requests behind a shared prefix.  Against the restatement in 64 bits, with the
tolerance of test_gpu_paged.py (4 bits: test_gpu_paged_mx4.py's, the same number).
"""
import numpy as np
import pytest

import mx4_rows
import q35mix
import synth
from q35mix import KV_F16, KV_F32, KV_MXFP4
from test_gpu_paged import HD, Paged, cast, close_to, say
from test_gpu_paged_mx4 import Mx4, capture
from test_gpu_paged_plan import Ints, read

pytestmark = pytest.mark.gpu

TYPES = [KV_F32, KV_F16, KV_MXFP4]


def make(kv_type, **kw):
    return Mx4(**kw) if kv_type == KV_MXFP4 else Paged(kv_type, **kw)


def fill(p, rows):
    """rows[s] cached rows of normal values, of which the host's lengths (0) know nothing."""
    for s, n in enumerate(rows):
        for which in range(2):
            x = synth.normal(9000 + 2 * s + which, n * p.nkv * HD).reshape(n, p.nkv, HD).astype(np.float32)
            t = np.arange(n)
            at = p.table[s][t // p.R], slice(None), t % p.R
            if p.type == KV_MXFP4:
                p.codes[which][at], p.scales[which][at] = mx4_rows.encode(x)
            else:
                p.pages[which][at] = cast(x, p.type)
    p.push()


class Plan:
    """A plan's arrays on the device.  The free pages are the ones that the restatement's table has for the new rows."""

    def __init__(self, p, n, most):
        self.p, self.n = p, n
        self.rows, self.tokens, self.taken = (Ints(p.ctx, [0] * n) for _ in range(3))
        self.free, self.listed = Ints(p.ctx, [0] * (n * p.table.shape[1])), Ints(p.ctx, [0])
        self.slots = Ints(p.ctx, [0] * most, np.int64)

    def set(self, lens, tokens):
        p = self.p
        have, end = [-(-a // p.R) for a in lens], [-(-(a + t) // p.R) for a, t in zip(lens, tokens)]
        free = [int(e) for s in range(self.n) for e in p.table[s][have[s]:end[s]]]
        self.rows.set(lens)
        self.tokens.set(tokens)
        self.free.set((free + [0] * self.free.n)[:self.free.n])
        self.listed.set([len(free)])
        p.len = list(lens)
        # (a plan before has left no entry behind its requests' rows)
        table = np.ascontiguousarray(p.table, np.int32)
        q35mix.check(q35mix.lib().q35m_copy_h2d(p.ctx.handle, p.c.tables()[0], table.ctypes.data, table.nbytes))
        self.want = [b - a for a, b in zip(have, end)]

    def call(self):
        self.p.c.plan(self.n, self.rows, self.tokens, self.free, self.slots, self.taken, self.listed)


def steps(p, lens_of_steps, tokens, decode):
    """The first step eager, the others replays of one graph; the plan and the attention together."""
    n, total = len(tokens), sum(tokens)
    fill(p, [max(a) for a in zip(*lens_of_steps)])
    plan = Plan(p, n, total)
    x = p.inputs(total, salt=5)
    d = p.dev(x, "q_gate", "k", "v")
    out = p.ctx.array((total + 1, p.nh * HD), np.full((total + 1, p.nh * HD), 5, np.float32))

    def step():
        plan.call()
        if decode:
            p.c.attn_decode(0, list(range(n)), *d, out)
        else:
            p.c.attn_prefill(0, list(range(n)), tokens, *d, out)

    some = None if decode else sorted({0, 1, min(tokens) // 2, 15, 63, 64, max(tokens) // 3, max(tokens) - 2, max(tokens) - 1})
    launch = end = None
    for k, lens in enumerate(lens_of_steps):
        plan.set(lens, tokens)
        if k == 0:
            step()
        else:
            if launch is None:
                launch, end = capture(p, step)
            launch()
        assert list(plan.taken.get()) == plan.want
        p.put(range(n), tokens, x)
        got = out.download()
        say(close_to(got[:-1], p.attend(range(n), tokens, x, some=some)))
        assert (got[-1] == 5).all()
        p.check_pages()
    end()


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("lens", [[[3000, 5, 1700], [640, 2999, 0], [127, 128, 129]], [[16000], [8191], [383]],
                                  [[600] * 12, [100] * 6 + [2000] * 6, [1] * 12]], ids=["ragged", "one", "many"])
def test_planned_tokens(kv_type, lens):
    n = len(lens[0])
    with make(kv_type, nh=8 if n > 3 else 16, nkv=4, n_seqs=n, max_rows=max(map(max, lens)) + 1, page_rows=64, salt=n) as p:
        steps(p, lens, [1] * n, True)


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("lens,tokens", [([[700, 0, 3], [0, 1500, 64], [64, 65, 2000]], [100, 40, 65]), ([[2000], [0], [333]], [600]),
                                         ([[3000, 1000], [17, 0], [2048, 2047]], [16, 1])], ids=["ragged", "chunk", "short"])
def test_planned_chunks(kv_type, lens, tokens):
    n = len(tokens)
    with make(kv_type, nh=16, nkv=4, n_seqs=n, max_rows=max(max(a) + t for a, t in zip(zip(*lens), tokens)), page_rows=32, salt=n) as p:
        steps(p, lens, tokens, False)


@pytest.mark.parametrize("kv_type", TYPES)
def test_requests_behind_a_shared_prefix(kv_type):
    """A prefix of 40 rows: its two whole pages are shared, and each request has its own copy of the third, in which it ends.
    Their tokens go on there, each in its own."""
    prefix, R, N = 40, 16, 3
    with make(kv_type, n_seqs=N, max_rows=128, page_rows=R, salt=2) as p:
        fill(p, [prefix] + [0] * (N - 1))
        for s in range(1, N):
            own, p.table[s][:2] = p.table[s][2], p.table[0][:2]
            for kept in (p.codes + p.scales if kv_type == KV_MXFP4 else p.pages):
                kept[own] = kept[p.table[0][2]]
        p.push()
        table_ptr, _, per = p.c.tables()
        plan = Plan(p, N, N * 20)
        lens = [prefix] * N
        for turn, tokens in enumerate(([20, 3, 9], [1, 1, 1], [1, 1, 1])):
            total = sum(tokens)
            x = p.inputs(total, salt=30 + turn)
            out = p.ctx.array((total, p.nh * HD))
            plan.set(lens, tokens)
            plan.call()
            if turn == 0:
                p.c.attn_prefill(0, list(range(N)), tokens, *p.dev(x, "q_gate", "k", "v"), out)
            else:
                p.c.attn_decode(0, list(range(N)), *p.dev(x, "q_gate", "k", "v"), out)
            assert list(plan.taken.get()) == plan.want
            now = read(p.ctx, table_ptr, (N, per), np.int32)
            for s in range(N):
                used = -(-(lens[s] + tokens[s]) // R)
                assert np.array_equal(now[s][:used], p.table[s][:used]) and (now[s][used:] == -1).all()
            p.put(range(N), tokens, x)
            close_to(out.download(), p.attend(range(N), tokens, x))
            p.check_pages()
            lens = [a + t for a, t in zip(lens, tokens)]
