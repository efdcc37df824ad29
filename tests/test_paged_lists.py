"""Lists of sequences, tokens and rows at the paged cache's entry points, without a device: what a list may be made of, from
the C functions' prototypes and from the front end's calls.
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
