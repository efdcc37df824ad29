"""What a paged cache's calls may read and write (CPU; no device).

The library's rule (qwen3.5sharp_amd/csrc/page_map.h, which every paged call is
checked against before anything is enqueued) against a plain model: random
histories of maps, unmaps and lengths must agree on every answer.  Then the null
handles and bad arguments of the entry points that need no device.
"""
import ctypes
import os
import random
import subprocess

import pytest

import q35mix

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, BAD_SEQ, BAD_RANGE, BAD_PAGE, SHARED, UNMAPPED, TOO_LONG = range(7)


@pytest.fixture(scope="module")
def driver(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("pages") / "pages")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "qwen3.5sharp_amd", "csrc"),
                    os.path.join(ROOT, "tests", "page_map_driver.cpp"), "-o", exe], check=True)
    return exe


class Map:
    def __init__(self, exe, *dims):
        self.p = subprocess.Popen([exe], stdin=subprocess.PIPE, stdout=subprocess.PIPE, text=True, bufsize=1)
        self.p.stdin.write(" ".join(map(str, dims)) + "\n")

    def ask(self, *line):
        self.p.stdin.write(" ".join(map(str, line)) + "\n")
        self.p.stdin.flush()
        return int(self.p.stdout.readline())

    def close(self):
        self.p.stdin.close()
        assert self.p.wait() == 0


class Model:
    def __init__(self, n_seqs, max_rows, n_pages, page_rows):
        self.rows, self.n_pages, self.page_rows = max_rows, n_pages, page_rows
        self.table = [[None] * -(-max_rows // page_rows) for _ in range(n_seqs)]
        self.len = [0] * n_seqs

    def map(self, s, first, n, pages):
        if not 0 <= s < len(self.table):
            return BAD_SEQ
        if first < 0 or n < 0 or first + n > len(self.table[0]):
            return BAD_RANGE
        if pages is not None and any(not 0 <= p < self.n_pages for p in pages):
            return BAD_PAGE
        self.table[s][first:first + n] = [None] * n if pages is None else list(pages)
        return OK

    def usable(self, s, tokens):
        if not 0 <= s < len(self.table):
            return BAD_SEQ
        end = self.len[s] + tokens
        if end > self.rows:
            return TOO_LONG
        if any(self.table[s][r // self.page_rows] is None for r in range(end)):
            return UNMAPPED
        uses = [p for t in self.table for p in t if p is not None]
        written = {self.table[s][r // self.page_rows] for r in range(self.len[s], end)}
        return SHARED if any(uses.count(p) > 1 for p in written) else OK


@pytest.mark.parametrize("seed", range(6))
def test_random_histories(driver, seed):
    rng = random.Random(seed)
    dims = (rng.randint(1, 4), rng.randint(1, 70), rng.randint(1, 12), 16)
    m, ref = Map(driver, *dims), Model(*dims)
    seen = set()
    for _ in range(400):
        s = rng.randint(-1, dims[0]) if rng.random() < 0.05 else rng.randrange(dims[0])
        do = rng.random()
        if do < 0.35:
            top = len(ref.table[0])
            first = rng.randint(-1, top) if rng.random() < 0.1 else rng.randrange(top)
            n = rng.randint(0, top + 1 - max(first, 0))
            pages = [rng.randint(-1, dims[2]) if rng.random() < 0.02 else rng.randrange(dims[2]) for _ in range(n)]
            assert m.ask("map", s, first, n, *pages) == ref.map(s, first, n, pages)
        elif do < 0.45:
            first = rng.randrange(len(ref.table[0]))
            assert m.ask("unmap", s, first, 1) == ref.map(s, first, 1, None)
        elif do < 0.6 and 0 <= s < dims[0]:
            ref.len[s] = rng.randint(0, dims[1])
            m.ask("len", s, ref.len[s])
        else:
            tokens = rng.choice([0, 1, 1, 2, rng.randint(0, dims[1])])
            want = ref.usable(s, tokens)
            seen.add(want)
            assert m.ask("usable", s, tokens) == want, (dims, ref.table, ref.len, s, tokens)
        if 0 <= s < dims[0]:
            i = rng.randrange(len(ref.table[0]))
            assert m.ask("page", s, i) == (-1 if ref.table[s][i] is None else ref.table[s][i])
    assert OK in seen and len(seen) > 1
    m.close()


def test_shared_pages_are_read_only(driver):
    m = Map(driver, 2, 64, 8, 16)
    assert m.ask("map", 0, 0, 2, 5, 3) == OK
    assert m.ask("map", 1, 0, 2, 5, 4) == OK          # a common first page
    m.ask("len", 0, 16)
    m.ask("len", 1, 16)
    assert m.ask("usable", 0, 16) == OK and m.ask("usable", 1, 1) == OK
    m.ask("len", 1, 15)
    assert m.ask("usable", 1, 1) == SHARED            # row 15 lies in the shared page
    assert m.ask("usable", 1, 0) == OK                # reading it is fine
    assert m.ask("map", 0, 0, 1, 7) == OK             # the other entry moves away
    assert m.ask("usable", 1, 1) == OK
    assert m.ask("map", 1, 1, 1, 5) == OK             # twice in one sequence
    m.ask("len", 1, 16)
    assert m.ask("usable", 1, 1) == SHARED
    m.close()


def test_unmapped_and_too_long(driver):
    m = Map(driver, 1, 40, 4, 16)                      # 3 pages hold 48 rows, the sequence 40
    assert m.ask("usable", 0, 0) == OK
    assert m.ask("usable", 0, 1) == UNMAPPED
    assert m.ask("map", 0, 1, 2, 1, 2) == OK
    assert m.ask("usable", 0, 1) == UNMAPPED           # entry 0 is missing
    assert m.ask("map", 0, 0, 1, 0) == OK
    assert m.ask("usable", 0, 40) == OK
    assert m.ask("usable", 0, 41) == TOO_LONG
    assert m.ask("map", 0, 1, 3, 1, 2, 3) == BAD_RANGE
    assert m.ask("map", 0, 1, 2, 3, 4) == BAD_PAGE and m.ask("page", 0, 1) == 1      # nothing changed
    assert m.ask("unmap", 0, 1, 1) == OK
    assert m.ask("usable", 0, 17) == UNMAPPED and m.ask("usable", 0, 16) == OK
    m.close()


def test_null_handles_are_refused():
    L = q35mix.lib()
    one = (ctypes.c_int * 1)(0)
    h = ctypes.c_void_p(1234)
    assert L.q35m_paged_create(None, 1, 16, 1, 16, q35mix.KV_F16, ctypes.byref(h)) == q35mix.ERR_INVALID
    assert h.value is None and "context" in L.q35m_last_error().decode()
    assert L.q35m_paged_create(None, 1, 16, 1, 16, q35mix.KV_F16, None) == q35mix.ERR_INVALID
    assert L.q35m_paged_destroy(None) == q35mix.OK
    assert L.q35m_paged_map(None, 0, 0, 0, None) == q35mix.ERR_INVALID
    assert "paged" in L.q35m_last_error().decode()
    assert L.q35m_paged_advance(None, 1, one, one) == q35mix.ERR_INVALID
    assert L.q35m_paged_truncate(None, 0, 0) == q35mix.ERR_INVALID
    assert L.q35m_paged_len(None, 0, one) == q35mix.ERR_INVALID
    p, n = ctypes.c_void_p(), ctypes.c_size_t()
    assert L.q35m_paged_device_ptr(None, 0, 2, ctypes.byref(p), ctypes.byref(n)) == q35mix.ERR_INVALID
    assert L.q35m_paged_append(None, 0, 1, one, one, None, None) == q35mix.ERR_INVALID
    assert L.q35m_paged_attn_decode(None, 0, 1, one, None, None, None, None) == q35mix.ERR_INVALID
    assert L.q35m_paged_attn_prefill(None, 0, 1, one, one, None, None, None, None) == q35mix.ERR_INVALID
