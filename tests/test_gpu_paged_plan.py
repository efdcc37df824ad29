"""Page tables and slots planned on the GPU from request lengths, against a plain restatement (whole numbers: equal), and
the attention of sequences whose tables and lengths a plan made, eager and captured.
"""
import ctypes
import random

import numpy as np
import pytest

import mx4_rows
import q35mix
import synth
from q35mix import KV_F16, KV_F32, KV_MXFP4
from test_gpu_paged import HD, Paged, close_to, refused
from test_gpu_paged_mx4 import Mx4, capture

pytestmark = pytest.mark.gpu


class Ints:
    """Whole numbers on the device, as the front end takes them."""

    def __init__(self, ctx, data, dtype=np.int32):
        self.ctx, self.dtype = ctx, np.dtype(dtype)
        data = np.ascontiguousarray(data, dtype)
        self.n, self.nbytes = data.size, data.nbytes
        self.buf = ctx.array((max(1, -(-data.nbytes // 4)),))
        self.ptr = self.buf.ptr
        self.set(data)

    def set(self, data):
        data = np.ascontiguousarray(data, self.dtype)
        assert data.nbytes == self.nbytes
        if data.nbytes:
            q35mix.check(q35mix.lib().q35m_copy_h2d(self.ctx.handle, self.ptr, data.ctypes.data, data.nbytes))

    def get(self):
        return read(self.ctx, self.ptr, (self.n,), self.dtype)


def read(ctx, ptr, shape, dtype):
    a = np.empty(shape, dtype)
    if a.nbytes:
        q35mix.check(q35mix.lib().q35m_copy_d2h(ctx.handle, a.ctypes.data, ptr, a.nbytes))
    return a


def planned(rows, tokens, table, free, n_pages, page, max_rows, n_slots):
    """(table, lens, slots, taken) as a plan leaves them."""
    table, slots, lens, taken, at, used = table.copy(), [], [], [], 0, 0
    for i, (r, t) in enumerate(zip(rows, tokens)):
        r = min(max(int(r), 0), max_rows)
        t = min(max(int(t), 0), max_rows - r)
        have, end = -(-r // page), -(-(r + t) // page)
        used += end - have
        ok = end == have or used <= len(free)
        new = free[used - (end - have):used] if ok else [-1] * (end - have)
        table[i, have:] = -1
        table[i, have:end] = [p if 0 <= p < n_pages else -1 for p in new]
        for j in range(r, r + t):
            p = table[i, j // page]
            slots.append(int(p) * page + j % page if 0 <= p < n_pages else -1)
        lens.append(r)
        taken.append(end - have if ok else -1)
    return table, np.array(lens), np.array(slots[:n_slots], np.int64), np.array(taken)


class Planner:
    def __init__(self, n_seqs, max_rows, page, n_pages, kv_type=KV_MXFP4):
        self.ctx = q35mix.Context(q35mix.qwen35_config(num_layers=1, num_heads=1, num_kv_heads=1, is_recurrent=[0]), n_seqs=1,
                                  kv_capacity=16)
        self.c = q35mix.PagedCache(self.ctx, n_seqs=n_seqs, max_rows=max_rows, n_pages=n_pages, page_rows=page, kv_type=kv_type)
        self.n, self.max_rows, self.page, self.n_pages = n_seqs, max_rows, page, n_pages
        self.table_ptr, self.lens_ptr, self.per = self.c.tables()

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.c.close()
        self.ctx.close()

    def table(self):
        return read(self.ctx, self.table_ptr, (self.n, self.per), np.int32)

    def set_table(self, t):
        t = np.ascontiguousarray(t, np.int32)
        q35mix.check(q35mix.lib().q35m_copy_h2d(self.ctx.handle, self.table_ptr, t.ctypes.data, t.nbytes))

    def lens(self):
        return read(self.ctx, self.lens_ptr, (self.n,), np.int32)

    def check(self, rows, tokens, free, n_slots=None, n=None):
        n = self.n if n is None else n
        before, lens = self.table(), self.lens()
        total = sum(min(max(int(t), 0), self.max_rows - min(max(int(r), 0), self.max_rows)) for r, t in zip(rows, tokens))
        n_slots = total if n_slots is None else n_slots
        slots = Ints(self.ctx, np.full(n_slots + 3, -77), np.int64)
        taken = Ints(self.ctx, np.full(n + 2, -78))
        view = type("View", (), {"ptr": slots.ptr, "nbytes": 8 * n_slots})()
        self.c.plan(n, Ints(self.ctx, rows), Ints(self.ctx, tokens), Ints(self.ctx, free), view, taken)
        want = planned(rows, tokens, before[:n], free, self.n_pages, self.page, self.max_rows, n_slots)
        table = self.table()
        assert np.array_equal(table[:n], want[0]) and np.array_equal(table[n:], before[n:])
        now = self.lens()
        assert np.array_equal(now[:n], want[1]) and np.array_equal(now[n:], lens[n:])
        got = slots.get()
        m = min(n_slots, total)
        assert np.array_equal(got[:m], want[2]) and (got[m:] == -77).all()          # behind the last token: as it was
        got = taken.get()
        assert np.array_equal(got[:n], want[3]) and (got[n:] == -78).all()
        return want


@pytest.mark.parametrize("n,max_rows,page", [(1, 16, 16), (1, 5000, 16), (3, 100, 32), (64, 700, 16), (65, 2048, 64), (300, 300, 256),
                                             (1000, 1024, 1024), (4, 100000, 16)])
def test_plans(n, max_rows, page):
    rng = random.Random(n + max_rows)
    per = -(-max_rows // page)
    with Planner(n, max_rows, page, n * per + 5) as p:
        for kind in range(6):
            rows = [rng.randint(0, max_rows) if rng.random() < 0.8 else 0 for _ in range(n)]
            tokens = [rng.choice([0, 1, 1, page, rng.randint(0, max_rows)]) for _ in range(n)]
            if kind == 1:
                rows, tokens = [0] * n, [max_rows] * n
            if kind == 2:
                rows = [r // page * page for r in rows]                 # every next token begins a page
            tokens = [min(t, max_rows - r) for r, t in zip(rows, tokens)]
            ids = list(range(p.n_pages))
            rng.shuffle(ids)
            table = np.full((n, per), -1, np.int32)
            for i, r in enumerate(rows):
                for e in range(-(-r // page)):
                    table[i, e] = ids.pop()
            p.set_table(table)
            need = sum(-(-(r + t) // page) - -(-r // page) for r, t in zip(rows, tokens))
            if kind in (3, 4):                                          # too few pages
                ids = ids[:max(0, need - rng.randint(1, max(1, need)))]
            total = sum(tokens)
            p.check(rows, tokens, ids, n_slots=None if kind != 5 else rng.randint(0, total))
            want = p.check(rows, tokens, ids)                           # the same again: the same
            if kind == 1:
                assert sorted(want[0].ravel()) == sorted(ids[:n * per])


def test_inputs_out_of_range():
    """Lengths and tokens are taken into range, page ids that are none are left out; other sequences stay."""
    with Planner(6, 100, 16, 40) as p:
        p.set_table(np.arange(42).reshape(6, 7) - 1)                    # (-1 and 40 among them)
        p.check([-5, 200, 30, 99, 2 ** 31 - 1, -2 ** 31], [20, 5, -3, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1],
                [39, 40, -1, 2 ** 31 - 1, -2 ** 31, 3, 2, 1, 0, 5, 6, 7, 8])
        p.check([16, 0], [16, 1], [], n=2)                              # no free pages at all
        p.check([16, 0, 5], [0, 0, 11], [], n=3)                        # nor any needed
        p.check([0], [0], [1, 2], n=1)                                  # nothing kept


def test_lengths_of_the_cache_itself():
    """rows may be the cache's own lengths: a plan of what it holds changes no length."""
    with Planner(5, 256, 16, 100) as p:
        p.check([3, 0, 100, 16, 250], [13, 40, 1, 16, 6], list(range(50, 90)))
        before = p.table()
        slots, taken = Ints(p.ctx, np.zeros(5), np.int64), Ints(p.ctx, np.zeros(5))
        rows = type("View", (), {"ptr": p.lens_ptr, "nbytes": 20})()
        p.c.plan(5, rows, Ints(p.ctx, [1] * 5), Ints(p.ctx, [1, 2, 3]), slots, taken)
        want = planned([3, 0, 100, 16, 250], [1] * 5, before, [1, 2, 3], 100, 16, 256, 5)
        assert np.array_equal(p.lens(), want[1]) and np.array_equal(p.table(), want[0])
        assert np.array_equal(slots.get(), want[2]) and np.array_equal(taken.get(), want[3])


def test_large_slots():
    """Slots are page * page_rows + row in 64 bits."""
    with Planner(1, 1024, 1024, 9) as p:
        p.check([0], [1024], [8])


# ------------------------------------------------------------------ with the attention

@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16, KV_MXFP4])
def test_planned_steps(kv_type):
    """A serving loop on the device: prompts, then tokens, each step planned from lengths that a kernel could have
    written; requests come and go, and the same loop captured once and replayed gives the same."""
    N, R, M = 3, 16, 128
    make = (lambda: Mx4(n_seqs=N, max_rows=M, page_rows=R)) if kv_type == KV_MXFP4 else \
        (lambda: Paged(kv_type, n_seqs=N, max_rows=M, page_rows=R))
    with make() as p:
        per = M // R
        free = list(np.random.RandomState(3).permutation(p.n_pages))
        rows, tokens = Ints(p.ctx, [0] * N), Ints(p.ctx, [0] * N)
        lst = Ints(p.ctx, free)
        slots, taken = Ints(p.ctx, np.zeros(N * M), np.int64), Ints(p.ctx, np.zeros(N))
        table_ptr, lens_ptr, _ = p.c.tables()
        x = p.inputs(N, salt=3)
        out = p.ctx.array((N, p.nh * HD))
        d = p.dev(x, "q_gate", "k", "v")
        held = p.ctx.array((N, p.nkv * HD)), p.ctx.array((N, p.nkv * HD))

        def plan(r, t):
            rows.set(r)
            tokens.set(t)
            lst.set(free + [-1] * (lst.n - len(free)))
            p.c.plan(N, rows, tokens, lst, slots, taken)

        def follow(r):
            """What the plan took leaves the free list; the restatement's tables and lengths become the device's."""
            got = taken.get()
            assert (got >= 0).all()
            del free[:int(got.sum())]
            p.table = read(p.ctx, table_ptr, (N, per), np.int32)
            p.len = list(r)
            assert list(read(p.ctx, lens_ptr, (N,), np.int32)) == list(r)

        # prompts of two requests
        plan([0, 0, 0], [20, 0, 33])
        y = p.inputs(53, salt=4)
        outp = p.ctx.array((53, p.nh * HD))
        p.c.attn_prefill(0, [0, 2], [20, 33], *p.dev(y, "q_gate", "k", "v"), outp)
        follow([0, 0, 0])
        p.put([0, 2], [20, 33], y)
        close_to(outp.download(), p.attend([0, 2], [20, 33], y))
        now = [20, 0, 33]
        refused(q35mix.ERR_INVALID, lambda: p.c.map(0, 0, [1]), "planned")
        refused(q35mix.ERR_INVALID, lambda: p.c.advance([0], [1]), "planned")
        refused(q35mix.ERR_INVALID, lambda: p.c.truncate(0, 0), "planned")
        refused(q35mix.ERR_INVALID, lambda: p.c.length(0), "planned")
        refused(q35mix.ERR_CAPACITY, lambda: p.c.append(0, [0], [M + 1], d[1], d[2]), "exceed")

        def step():
            p.c.plan(N, rows, tokens, lst, slots, taken)
            p.c.attn_decode(0, list(range(N)), *d, out)

        step_graph = None
        for k in range(40):
            if k == 18:                                    # the first request goes, another takes its place
                free += [int(e) for e in p.table[0] if e >= 0]
                now[0] = 0
            rows.set(now)
            tokens.set([1] * N)
            lst.set((free + [-1] * lst.n)[:lst.n])
            if k < 3:
                step()
            else:
                if step_graph is None:
                    step_graph = capture(p, step)
                step_graph[0]()
            follow(now)
            p.put(range(N), [1] * N, x)
            close_to(out.download(), p.attend(range(N), [1] * N, x))
            now = [a + 1 for a in now]
        p.c.rows(0, [0, 1, 2], [a - 1 for a in now], [1] * N, *held)
        for which, h in enumerate(held):
            want = np.stack([p.rows_of(s, now[s], which)[-1] for s in range(N)]).astype(np.float32).reshape(N, -1)
            assert np.array_equal(h.download(), want)
        p.check_pages()
        step_graph[1]()


def test_rows_without_pages():
    """A planned request that got no page: its rows are not written and read back as zeros, nobody else's change."""
    with Mx4(n_seqs=2, max_rows=64, page_rows=16) as p:
        rows, tokens = Ints(p.ctx, [0, 0]), Ints(p.ctx, [16, 40])
        slots, taken = Ints(p.ctx, np.zeros(56), np.int64), Ints(p.ctx, [0, 0])
        p.c.plan(2, rows, tokens, Ints(p.ctx, [3, 5, 7]), slots, taken)
        assert list(taken.get()) == [1, -1] and (slots.get()[16:] == -1).all()
        p.table = np.array([[3] * 4, [5] * 4])
        x = p.inputs(56, salt=1)
        out = p.ctx.array((56, p.nh * HD))
        p.c.attn_prefill(0, [0, 1], [16, 40], *p.dev(x, "q_gate", "k", "v"), out)
        p.put([0], [16], x)
        close_to(out.download()[:16], p.attend([0], [16], x))
        p.check_pages()
        k, v = p.ctx.array((50, 1024)), p.ctx.array((50, 1024))
        p.c.rows(0, [1, 0], [5, 6], [40, 10], k, v)
        assert (k.download()[:40] == 0).all() and (v.download()[:40] == 0).all()
        assert np.array_equal(v.download()[40:], p.rows_of(0, 16, 1)[6:].reshape(10, -1))


def test_refusals():
    with Planner(4, 64, 16, 20) as p:
        good = Ints(p.ctx, [0] * 4)
        slots = Ints(p.ctx, [0] * 8, np.int64)
        null = type("Null", (), {"ptr": None, "nbytes": 16})()
        none = type("None_", (), {"ptr": None, "nbytes": 0})()
        off = type("Off", (), {"ptr": good.ptr + 2, "nbytes": 16})()
        off8 = type("Off8", (), {"ptr": slots.ptr + 4, "nbytes": 16})()
        refused(q35mix.ERR_CAPACITY, lambda: p.c.plan(0, good, good, good, slots, good), "requests")
        refused(q35mix.ERR_CAPACITY, lambda: p.c.plan(5, *[Ints(p.ctx, [0] * 5)] * 3, slots, Ints(p.ctx, [0] * 5)), "requests")
        for bad in (null, off):
            refused(q35mix.ERR_INVALID, lambda: p.c.plan(4, bad, good, good, slots, good))
            refused(q35mix.ERR_INVALID, lambda: p.c.plan(4, good, bad, good, slots, good))
            refused(q35mix.ERR_INVALID, lambda: p.c.plan(4, good, good, bad, slots, good))
            refused(q35mix.ERR_INVALID, lambda: p.c.plan(4, good, good, good, slots, bad))
        refused(q35mix.ERR_INVALID, lambda: p.c.plan(4, good, good, good, null, good))
        refused(q35mix.ERR_INVALID, lambda: p.c.plan(4, good, good, good, off8, good))
        p.c.map(0, 0, [1])                                             # nothing was planned: the host's still
        assert p.c.length(0) == 0
        p.c.plan(4, good, good, none, none, Ints(p.ctx, [0] * 4))
        refused(q35mix.ERR_INVALID, lambda: p.c.map(0, 0, [1]), "planned")
        p.ctx.sync()


def test_arrays_that_overlap():
    """Requests are planned side by side: nothing that a plan writes may be what it reads or writes elsewhere, but the
    lengths, which are left as they are read."""
    with Planner(4, 64, 16, 20) as p:
        n = Ints(p.ctx, [0] * 16)
        def part(at, count, size=4):
            return type("Part", (), {"ptr": n.ptr + 4 * at, "nbytes": size * count})()
        rows, tokens, free, taken = part(0, 4), part(4, 4), part(8, 4), part(12, 4)
        slots = Ints(p.ctx, [0] * 8, np.int64)
        far = Ints(p.ctx, [0] * 4)
        inside = lambda ptr, size=16: type("Inside", (), {"ptr": ptr, "nbytes": size})()
        for bad in (dict(taken=part(3, 4)), dict(taken=rows), dict(taken=part(5, 4)), dict(taken=part(9, 4)),
                    dict(slots=inside(n.ptr)), dict(slots=inside(n.ptr + 24)), dict(slots=inside(n.ptr + 40)),
                    dict(slots=inside(n.ptr + 56)), dict(tokens=inside(p.lens_ptr)), dict(taken=inside(p.lens_ptr)),
                    dict(rows=inside(p.lens_ptr + 4)), dict(rows=inside(p.lens_ptr - 4)), dict(free=inside(p.lens_ptr)),
                    dict(free=inside(p.table_ptr + 60)), dict(rows=inside(p.table_ptr)), dict(slots=inside(p.table_ptr)),
                    dict(taken=inside(p.table_ptr + 48))):
            a = dict(rows=rows, tokens=tokens, free=free, slots=slots, taken=taken) | bad
            refused(q35mix.ERR_INVALID, lambda: p.c.plan(4, a["rows"], a["tokens"], a["free"], a["slots"], a["taken"]), "overlap")
        p.c.map(0, 0, [1])                                             # nothing was planned
        p.c.plan(4, rows, rows, rows, slots, taken)                    # what is only read may be one array
        p.c.plan(4, inside(p.lens_ptr), tokens, free, slots, far)
        p.ctx.sync()
