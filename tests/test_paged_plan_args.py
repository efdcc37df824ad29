"""Entry points of plans and row reads without a device: null handles; what the page map lets a read touch."""
import ctypes
import os
import subprocess

import numpy as np

import mx4_rows
import q35mix

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_null_handles():
    L = q35mix.lib()
    one = (ctypes.c_int * 1)(0)
    p, n = ctypes.c_void_p(), ctypes.c_int()
    assert L.q35m_paged_rows(None, 0, 1, one, one, one, None, None) == q35mix.ERR_INVALID
    assert L.q35m_paged_plan(None, 1, None, None, None, 0, None, 0, None) == q35mix.ERR_INVALID
    assert L.q35m_paged_tables(None, ctypes.byref(p), ctypes.byref(p), ctypes.byref(n)) == q35mix.ERR_INVALID
    assert q35mix.KV_MXFP4 not in (q35mix.KV_F32, q35mix.KV_F16)


def test_readable_rows(tmp_path):
    """Rows may be read where their pages are mapped, beyond the length too, and up to max_rows in any case."""
    src = tmp_path / "r.cpp"
    src.write_text('''
#include <cstdio>
#include "page_map.h"
int main() {
    q35::PageMap m(2, 100, 8, 16);
    int ids[3] = {1, 2, 3};
    m.map(0, 0, 3, ids);
    m.map(0, 5, 1, ids);
    const int at[][3] = {{0, 0, 48}, {0, 47, 1}, {0, 48, 1}, {0, 40, 9}, {0, 80, 16}, {0, 79, 2}, {0, 96, 4}, {0, 100, 0},
                         {0, 100, 1}, {0, 101, 0}, {0, 2147483647, 16777216}, {0, 0, 2147483647}, {1, 0, 0}, {1, 0, 1}, {2, 0, 0}, {-1, 0, 0}};
    for (auto& a : at) std::printf("%d%d ", m.readable(a[0], a[1], a[2], false), m.readable(a[0], a[1], a[2], true));
}
''')
    exe = str(tmp_path / "r")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                    os.path.join(ROOT, "qwen3.5sharp_amd", "csrc"), str(src), "-o", exe], check=True)
    got = subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()
    ok, seq, unmapped, long = "0", "1", "5", "6"
    assert got == [ok + ok, ok + ok, unmapped + ok, unmapped + ok, ok + ok, unmapped + ok, unmapped + ok, ok + ok, long + long,
                   long + long, long + long, long + long, ok + ok, unmapped + ok, seq + seq, seq + seq]


def test_the_rows_restatement():
    """The tests' own encoder against a search over all codes and powers of two."""
    rng = np.random.RandomState(1)
    x = (rng.standard_normal((40, 256)) * 2.0 ** rng.randint(-30, 20, (40, 1))).astype(np.float32)
    codes, scales = mx4_rows.encode(x)
    held = mx4_rows.decode(codes, scales).reshape(40, 8, 32).astype(np.float64)
    b = x.reshape(40, 8, 32).astype(np.float64)
    for r in range(40):
        for k in range(8):
            top = np.abs(b[r, k]).max()
            s = min([e for e in range(-23, 14) if top <= 7 * 2.0 ** e] or [13])
            assert scales[r, k] == s + 127
            grid = np.concatenate([mx4_rows.LEVELS, -mx4_rows.LEVELS]) * 2.0 ** s
            assert np.allclose(np.abs(held[r, k] - b[r, k]), np.abs(grid[None] - b[r, k][:, None]).min(1), rtol=0, atol=0)
    pool = mx4_rows.to_pool(1, codes.reshape(1, 1, 40, 128)[:, :, :32], scales.reshape(1, 1, 40, 8)[:, :, :32])
    assert pool.shape == (1, 1, 136 * 32) and pool[0, 0, 128 * 32 + 128 + 16 * 3 + 5] == scales[16 + 5, 3]
    back = mx4_rows.from_pool(1, pool, 32)
    assert np.array_equal(back[0][0, 0], codes[:32]) and np.array_equal(back[1][0, 0], scales[:32])


def test_lists_as_the_calls_take_them():
    """The front end's short and long lists: C ints of the same values, wrapped where too large, refused where not whole."""
    import pytest
    for n in (0, 1, 3, 7, 8, 64, 65, 200):
        v = [(37 * i) % 101 - 50 for i in range(n)]
        for given in (v, tuple(v), np.array(v, np.int64), np.array(v, np.int32)):
            assert np.array_equal(np.frombuffer(q35mix._ints(given), np.int32) if n else [], v)
            assert list(q35mix._seqs(given)) == v
    for n in (1, 8):
        assert list(q35mix._ints([2 ** 31] * n)) == list(q35mix._seqs([2 ** 31] * n)) == [-2 ** 31] * n
        for f in (q35mix._ints, q35mix._seqs):
            with pytest.raises(TypeError):
                f([1.5] * n)
