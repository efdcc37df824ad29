"""Page tables planned on the GPU: the ends of what a plan takes and gives.  Whole numbers, which must be equal, and the
attention of sequences whose lengths the device alone has, against the restatement in 64 bits (test_gpu_paged.py).
"""
import numpy as np
import pytest

import q35mix
from q35mix import KV_F16, KV_F32, KV_MXFP4, STATE_KEYS, STATE_VALUES
from test_gpu_paged import refused
from test_gpu_paged_plan import Ints, Planner

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
