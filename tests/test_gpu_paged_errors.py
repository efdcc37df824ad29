"""Paged K/V cache on the GPU: what a failed call, the library's or another's, leaves for the calls after it."""
import ctypes

import numpy as np
import pytest

import q35mix
from q35mix import KV_F16, KV_F32
from test_gpu_paged import HD, Paged, cast, refused, rope_norm

pytestmark = pytest.mark.gpu

HUGE = 1 << 45                                              # bytes no device has


def calls_work(p):
    """Every kind of call on a cache of one sequence of up to 64 rows, host and device agreeing afterwards."""
    p.c.unmap(0, 1, 1)
    refused(q35mix.ERR_CAPACITY, lambda: p.c.append(0, [0], [17], *p.dev(p.inputs(17), "k", "v")), "mapped")
    p.c.map(0, 0, p.table[0])
    x = p.inputs(20, salt=81)
    p.c.append(0, [0], [20], *p.dev(x, "k", "v"))
    p.put([0], [20], x)
    p.step([20])
    p.c.truncate(0, 19)
    p.len[0] = 19
    for T in (1, 3):
        x = p.inputs(T, salt=82 + T)
        out = p.ctx.array((T, p.nh * HD))
        call = p.c.attn_prefill if T > 1 else p.c.attn_decode
        call(0, [0], *([[T]] if T > 1 else []), *p.dev(x, "q_gate", "k", "v"), out)
        p.put([0], [T], x)
        want = p.attend([0], [T], x)
        assert np.abs(out.download() - want).max() <= 2e-5 * np.abs(want).max()
        p.step([T])
    assert p.c.length(0) == 23
    p.check_pages()


def test_a_cache_that_does_not_fit():
    """A pool larger than the device is refused as such, and neither a smaller one nor a cache that was there fails after it."""
    with Paged(KV_F32, max_rows=64) as p:
        pages = HUGE // (4 * 1024 * HD * 4)                 # of 1024 rows of 4 kv heads of 256 floats
        for _ in range(2):
            refused(q35mix.ERR_OOM, lambda: q35mix.PagedCache(p.ctx, 1, 64, pages, 1024, KV_F32))
        calls_work(p)
        refused(q35mix.ERR_OOM, lambda: q35mix.PagedCache(p.ctx, 1, 64, pages, 1024, KV_F32))
        with q35mix.PagedCache(p.ctx, 1, 64, 4, 16, KV_F32) as c:
            c.map(0, 0, [0])
            c.advance([0], [1])
            assert c.length(0) == 1


def test_errors_left_by_other_calls():
    """An allocation that failed elsewhere on the thread, by the library or by the program, is not a paged call's error."""
    hip, lib = q35mix.hip(), q35mix.lib()

    def fails():
        ptr = ctypes.c_void_p()
        assert hip.hipMalloc(ctypes.byref(ptr), ctypes.c_size_t(HUGE)) != 0
        ptr = ctypes.c_void_p()
        assert lib.q35m_malloc(ctypes.byref(ptr), ctypes.c_size_t(HUGE)) == q35mix.ERR_OOM

    with Paged(KV_F32, max_rows=64) as p:
        x = p.inputs(1)
        args, out = p.dev(x, "q_gate", "k", "v"), p.ctx.array((1, p.nh * HD))
        for call in (lambda: p.c.map(0, 0, p.table[0]), lambda: p.c.advance([0], [1]), lambda: p.c.truncate(0, 0),
                     lambda: p.c.append(0, [0], [1], *args[1:]), lambda: p.c.attn_decode(0, [0], *args, out),
                     lambda: p.c.attn_prefill(0, [0], [1], *args, out),
                     lambda: q35mix.PagedCache(p.ctx, 1, 64, 4, 16, KV_F32).close()):
            fails()
            call()
        calls_work(p)
        # and the library's own failure is nobody else's
        ptr = ctypes.c_void_p()
        assert lib.q35m_malloc(ctypes.byref(ptr), ctypes.c_size_t(HUGE)) == q35mix.ERR_OOM
        assert hip.hipGetLastError() == 0


# ------------------------------------------------------------------ the largest calls

def test_calls_of_too_many_rows():
    """Refused before anything is read (the arrays hold one row), whatever is mapped."""
    with Paged(KV_F32, nh=32, nkv=4, max_rows=64) as p:
        x = p.inputs(1)
        (q, k, v), out = p.dev(x, "q_gate", "k", "v"), p.ctx.array((1, p.nh * HD))
        refused(q35mix.ERR_UNSUPPORTED, lambda: p.c.append(0, [0], [(1 << 24) + 1], k, v), "16777216")
        refused(q35mix.ERR_CAPACITY, lambda: p.c.append(0, [0], [1 << 24], k, v), "exceed")
        refused(q35mix.ERR_UNSUPPORTED, lambda: p.c.attn_prefill(0, [0], [(1 << 22) + 1], q, k, v, out), "4194304")
        refused(q35mix.ERR_CAPACITY, lambda: p.c.attn_prefill(0, [0], [1 << 22], q, k, v, out), "exceed")
        refused(q35mix.ERR_INVALID, lambda: p.c.append(0, [0], [-1], k, v), "tokens")
        p.ctx.sync()
    with q35mix.Context(q35mix.qwen35_config(num_layers=1, num_heads=8192, num_kv_heads=1024, is_recurrent=[0]), n_seqs=1,
                        kv_capacity=1) as ctx:
        refused(q35mix.ERR_UNSUPPORTED, lambda: q35mix.PagedCache(ctx, 1, 16, 1, 16, KV_F32), "q heads")


def test_append_of_a_million_rows():
    """More (row, kv head) pairs than one launch takes: rows at the beginning, about the end of the first launch and at
    the end, from arrays of 4 GiB, bit for bit."""
    T, R = (1 << 20) + 5, 1024
    with Paged(KV_F16, nh=4, nkv=4, max_rows=T, page_rows=R, spare=0, layers=1) as p:
        kv = p.ctx.array((T, p.nkv * HD))
        windows = [0, 700_000, (1 << 20) - 4, T - 3]
        xs = [p.inputs(3, salt=90 + i)["k"] for i in range(len(windows))]
        for at, x in zip(windows, xs):
            q35mix.check(q35mix.lib().q35m_copy_h2d(p.ctx.handle, kv.ptr + at * p.nkv * HD * 4, x.ctypes.data, x.nbytes))
        p.c.append(0, [0], [T], kv, kv)
        p.ctx.sync()
        for at, x in zip(windows, xs):
            want = (rope_norm(x.reshape(3, p.nkv, HD), p.w["k_norm"], at + np.arange(3)), x.reshape(3, p.nkv, HD))
            for kind, rows in zip((q35mix.STATE_KEYS, q35mix.STATE_VALUES), want):
                ptr, _ = p.c.device_ptr(0, kind)
                for j in range(3):
                    r = at + j
                    for h in range(p.nkv):
                        got = np.empty(HD, np.float16)
                        where = ((int(p.table[0][r // R]) * p.nkv + h) * R + r % R) * HD * 2
                        q35mix.check(q35mix.lib().q35m_copy_d2h(p.ctx.handle, got.ctypes.data, ptr + where, got.nbytes))
                        assert np.array_equal(got.view(np.uint16), cast(rows[j, h], KV_F16).view(np.uint16)), (r, h, kind)
        kv.free()
