"""Lists of sequences, tokens and rows at the entry points, without a device: what a list may be made of, from the paged C
functions' prototypes and from the front end's calls.
"""
import ctypes

import numpy as np
import pytest

import q35mix

LISTS = {"q35m_paged_advance": 2, "q35m_paged_append": 2, "q35m_paged_rows": 3, "q35m_paged_attn_decode": 1,
         "q35m_paged_attn_prefill": 2}


@pytest.mark.parametrize("name", LISTS)
def test_prototypes_take_pointers_to_c_ints_alone(name):
    """A number, bytes or floats in a list's place are no address of C ints."""
    call = getattr(q35mix.lib(), name)
    first = 2 if name == "q35m_paged_advance" else 3            # (handle, layer, n before the lists)
    for wrong in (5, b"\0\0\0\0", (ctypes.c_float * 1)(0), (ctypes.c_int64 * 1)(0), ctypes.c_void_p(8)):
        for at in range(first, first + LISTS[name]):
            args = [None] + [0] * (first - 1) + [(ctypes.c_int * 1)(0)] * LISTS[name]
            args += [None] * (len(call.argtypes) - len(args))
            assert call(*args) == q35mix.ERR_INVALID            # (a null handle)
            args[at] = wrong
            with pytest.raises(ctypes.ArgumentError):
                call(*args)


BIG = (2 ** 32, 2 ** 32 + 1, 2 ** 31, -2 ** 31 - 1, 2 ** 70)


@pytest.mark.parametrize("n", [1, 3, 8, 64, 65])
def test_calls_refuse_values_that_are_no_c_ints(n):
    """Cut to 32 bits they would be another conversation's number, or another count of rows."""
    c = object.__new__(q35mix.PagedCache)
    c.handle = None                                             # (what is not refused before ends at the null handle)
    x = type("Null", (), {"ptr": None})()
    good = list(range(n))

    def calls(lists):
        yield lambda: c.advance(lists(0), lists(1))
        yield lambda: c.append(0, lists(0), lists(1), x, x)
        yield lambda: c.rows(0, lists(0), lists(1), lists(2), x, x)
        yield lambda: c.attn_decode(0, lists(0), x, x, x, x)
        yield lambda: c.attn_prefill(0, lists(0), lists(1), x, x, x, x)

    for call in calls(lambda k: good):
        with pytest.raises(q35mix.Q35Error):
            call()
    for big in BIG:
        for where in (0, 1, 2):
            for kind in (list, tuple, np.array):
                if kind is np.array and abs(big) > 2 ** 40:
                    continue
                bad = kind(good[:-1] + [big])
                for k, call in enumerate(calls(lambda k: bad if k == where else good)):
                    if where < (2, 2, 3, 1, 2)[k]:
                        with pytest.raises(ValueError):
                            call()
    for wrong in ([1.5] * n, ["a"] * n, [None] * n):
        with pytest.raises(TypeError):
            c.advance(wrong, good)


@pytest.mark.parametrize("n", [1, 8])
def test_calls_over_the_context_s_own_caches_refuse_them_too(n):
    c = object.__new__(q35mix.Context)
    c.handle = None
    x = type("Null", (), {"ptr": None})()
    calls = (lambda v: c.deltanet_decode(0, v, x, x, x, x, x), lambda v: c.attn_decode(0, v, x, x, x, x),
             lambda v: c.attn_decode_noalloc(0, v, x, x, x, x), lambda v: q35mix.DecodeGraph(c, v, [], 16))
    for call in calls:
        with pytest.raises(q35mix.Q35Error):
            call(list(range(n)))
        for big in BIG:
            with pytest.raises(ValueError):
                call(list(range(n - 1)) + [big])
