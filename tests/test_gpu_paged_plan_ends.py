"""Page tables planned on the GPU: the ends of what a plan takes and gives.  Whole numbers, which must be equal, and the
attention of sequences whose lengths the device alone has, against the restatement in 64 bits (test_gpu_paged.py).
"""
import numpy as np
import pytest

import q35mix
from q35mix import KV_F16, KV_F32, KV_MXFP4, STATE_KEYS, STATE_VALUES
from test_gpu_paged import close_to, refused
from test_gpu_paged_mx4 import Mx4, capture
from test_gpu_paged_plan import Ints, Planner, planned, read

pytestmark = pytest.mark.gpu


def inside(ptr, nbytes=32):
    return type("Inside", (), {"ptr": ptr, "nbytes": nbytes})()


@pytest.mark.parametrize("kv_type", [KV_F32, KV_F16, KV_MXFP4])
def test_a_plan_writes_nothing_of_the_cache_but_tables_and_lengths(kv_type):
    """slots or taken in the cache's pages, at their first and last bytes and across their ends, or in its tables."""
    with Planner(4, 64, 16, 20, kv_type=kv_type) as p:
        a = [Ints(p.ctx, [0] * 4) for _ in range(3)]
        slots, taken = Ints(p.ctx, [0] * 8, np.int64), Ints(p.ctx, [0] * 4)
        for kind in (STATE_KEYS, STATE_VALUES):
            at, size = p.c.device_ptr(0, kind)
            for to in (at - 8, at, at + 4096, at + size - 8):
                refused(q35mix.ERR_INVALID, lambda: p.c.plan(4, *a, inside(to), taken), "overlap")
                refused(q35mix.ERR_INVALID, lambda: p.c.plan(4, *a, slots, inside(to)), "overlap")
        for to in (p.table_ptr, p.table_ptr + 4 * 4 * 4 - 8, p.lens_ptr, p.lens_ptr + 8):
            refused(q35mix.ERR_INVALID, lambda: p.c.plan(4, *a, inside(to), taken), "overlap")
            refused(q35mix.ERR_INVALID, lambda: p.c.plan(4, *a, slots, inside(to)), "overlap")
        p.c.map(0, 0, [1])                                      # nothing was planned
        at, size = p.c.device_ptr(0, STATE_VALUES)
        p.c.plan(4, a[0], a[1], inside(at, 16), slots, taken)   # what is only read may be anywhere
        p.ctx.sync()


# ------------------------------------------------------------------ lists whose length the device has

def test_listed_pages():
    """Plans of the first pages of a list, as many as a number on the device says: as plans of a list of that length."""
    n, page, max_rows = 5, 16, 96
    rng = np.random.RandomState(4)
    with Planner(n, max_rows, page, 40) as p:
        free, listed = Ints(p.ctx, [0] * 16), Ints(p.ctx, [0])
        rows, tokens, slots, taken = (Ints(p.ctx, [0] * k, t) for k, t in ((n, np.int32), (n, np.int32), (n * max_rows, np.int64), (n, np.int32)))
        for count in (0, 1, 2, 5, 7, 15, 16, 17, -1, 2 ** 31 - 1, -2 ** 31):
            r, t = rng.randint(0, 50, n), rng.randint(0, 40, n)
            ids = rng.permutation(40)[:16]
            before = p.table()
            for to, v in ((rows, r), (tokens, t), (free, ids), (listed, [count]), (slots, [-77] * (n * max_rows))):
                to.set(v)
            p.c.plan(n, rows, tokens, free, slots, taken, listed)
            want = planned(r, t, before, list(ids[:min(max(count, 0), 16)]), 40, page, max_rows, n * max_rows)
            assert np.array_equal(p.table(), want[0]) and np.array_equal(p.lens(), want[1])
            assert np.array_equal(slots.get()[:t.sum()], want[2]) and (slots.get()[t.sum():] == -77).all()
            assert np.array_equal(taken.get(), want[3])
        p.c.plan(n, rows, tokens, free, slots, taken)              # no such number: all of them
        assert np.array_equal(taken.get(), planned(r, t, p.table(), list(ids), 40, page, max_rows, 0)[3])
        bad = type("Bad", (), {"ptr": listed.ptr + 2, "nbytes": 4})()
        refused(q35mix.ERR_INVALID, lambda: p.c.plan(n, rows, tokens, free, slots, taken, bad), "aligned")
        refused(q35mix.ERR_INVALID, lambda: p.c.plan(n, rows, tokens, free, slots, taken, inside(taken.ptr + 4, 4)), "overlap")
        refused(q35mix.ERR_INVALID, lambda: p.c.plan(n, rows, tokens, free, slots, taken, inside(slots.ptr, 4)), "overlap")
        refused(q35mix.ERR_INVALID, lambda: p.c.plan(n, rows, tokens, free, slots, taken, inside(p.table_ptr, 4)), "overlap")


def test_a_captured_plan_whose_list_runs_short():
    """A step captured once: between replays the list gets shorter and longer.  A request that needs two pages with one left
    gets none and says so; those that need none are served, and their attention is right."""
    N, R, M, tokens = 4, 16, 128, [1, 40, 1, 17]
    at = np.cumsum([0] + tokens)
    with Mx4(n_seqs=N, max_rows=M, page_rows=R) as p:
        rows, toks, taken = Ints(p.ctx, [0] * N), Ints(p.ctx, tokens), Ints(p.ctx, [0] * N)
        lst, listed, slots = Ints(p.ctx, [0] * 12), Ints(p.ctx, [0]), Ints(p.ctx, [0] * at[-1], np.int64)
        table_ptr, _, per = p.c.tables()
        x = p.inputs(at[-1], salt=3)
        out = p.ctx.array((at[-1], p.nh * 256))
        d = p.dev(x, "q_gate", "k", "v")

        def step():
            p.c.plan(N, rows, toks, lst, slots, taken, listed)
            p.c.attn_prefill(0, list(range(N)), tokens, *d, out)

        free, now, launch, end, all_taken = [7, 3, 30, 11, 5, 2, 19, 23], [0] * N, None, None, []
        for k in range(3):
            if k == 2:
                free += [8, 25]
            rows.set(now)
            lst.set((free + [31] * 12)[:12])                        # (what is behind the list's end is nobody's to take)
            listed.set([len(free)])
            before = read(p.ctx, table_ptr, (N, per), np.int32)
            if launch is None:
                launch, end = capture(p, step)
            launch()
            want = planned(now, tokens, before, free, p.n_pages, R, M, at[-1])
            got = taken.get()
            p.table = read(p.ctx, table_ptr, (N, per), np.int32)
            assert np.array_equal(p.table, want[0]) and np.array_equal(got, want[3]) and np.array_equal(slots.get(), want[2])
            assert not (p.table == 31).any()
            p.len = list(now)
            # (a request that is not served still writes the rows that its kept page has room for)
            fits = [t if g >= 0 else min(t, -(-a // R) * R - a) for a, t, g in zip(now, tokens, got)]
            some = np.concatenate([np.arange(at[s], at[s] + t) for s, t in enumerate(fits)])
            p.put(range(N), fits, {name: v[some] for name, v in x.items()})
            served = [s for s in range(N) if got[s] >= 0]
            some = np.concatenate([np.arange(at[s], at[s + 1]) for s in served])
            close_to(out.download()[some], p.attend(served, [tokens[s] for s in served], {name: v[some] for name, v in x.items()}))
            p.check_pages()
            all_taken.append(list(got))
            free = free[sum(g for g in got if g > 0):]
            now = [a + t if g >= 0 else a for a, t, g in zip(now, tokens, got)]
        assert all_taken == [[1, 3, 1, 2], [0, -1, 0, -1], [0, 2, 0, 1]]
        end()


# ------------------------------------------------------------------ many requests

def test_tens_of_thousands_of_requests():
    """Each request's pages and slots come behind the sums of all before it; as many requests as one plan takes."""
    n, max_rows, page = 65535, 32, 16
    rng = np.random.RandomState(6)
    rows, tokens = rng.randint(0, 25, n), rng.randint(0, 8, n)
    need = -(-(rows + tokens) // page) - -(-rows // page)
    with Planner(n + 1, max_rows, page, 3 * n) as p:
        ids = rng.permutation(3 * n)
        table = np.full((n + 1, 2), -1, np.int32)
        kept = -(-rows // page)
        for e in range(2):
            some = np.nonzero(kept > e)[0]
            table[some, e], ids = ids[:some.size], ids[some.size:]
        p.set_table(table)
        want = p.check(list(rows), list(tokens), list(ids[:need.sum() - 5]), n=n)
        assert (want[3][:-200] >= 0).all() and (want[3] == -1).any()
        a = Ints(p.ctx, np.zeros(n + 1, np.int32))
        refused(q35mix.ERR_UNSUPPORTED, lambda: p.c.plan(n + 1, a, a, a, Ints(p.ctx, [0], np.int64), Ints(p.ctx, np.zeros(n + 1))), "65535")
