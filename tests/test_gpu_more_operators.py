"""States of the performance cases of the 4-bit cache: a program makes its context and caches once and keeps them, so a new
state takes those that an earlier one has left, and gives what one of its own handles gives; two states' calls follow each
other on one stream.
"""
import importlib.util
import os

import pytest

import q35mix

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
A = {"nh": 16, "nkv": 4, "page": 16, "ragged": True, "n": 3}
CASES = [{"kind": "append", "rows": 40, "tokens": 20, **A}, {"kind": "decode", "rows": 300, "tokens": 1, **A},
         {"kind": "prefill", "rows": 90, "tokens": 33, **A}, {"kind": "plan", "rows": 200, "tokens": 30, "short": 1, **A}]


@pytest.fixture
def cases(monkeypatch):
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "more_operators.py")
    spec = importlib.util.spec_from_file_location("more_operators", at)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own, m.made = True, []

    class Counted(q35mix.PagedCache):
        def __init__(self, *a, **k):
            m.made.append(k)
            super().__init__(*a, **k)
    monkeypatch.setattr(q35mix, "PagedCache", Counted)
    yield m
    m._Owner.program = None


def answer(m, state):
    got = m.run(state)
    torch.cuda.synchronize()
    return {k: t.clone() for k, t in got.items()}


@pytest.mark.parametrize("case", CASES, ids=lambda c: c["kind"])
def test_a_new_state_takes_the_handles_that_are_free(cases, case):
    first = {seed: answer(cases, cases.prepare(case, seed)) for seed in (1, 2, 3)}
    assert len(cases.made) == 1
    a, b = cases.prepare(case, 1), cases.prepare(case, 2)           # two at once: handles of their own
    assert len(cases.made) == 2 and a["cache"] is not b["cache"] and a["owner"].ctx is b["owner"].ctx
    for _ in range(2):
        for seed, s in ((1, a), (2, b)):
            got = answer(cases, s)
            assert all(torch.equal(got[k], first[seed][k]) for k in got)
    del a, s
    c = cases.prepare(case, 3)
    assert len(cases.made) == 2
    got = answer(cases, c)
    assert all(torch.equal(got[k], first[3][k]) for k in got)
    assert any(not torch.equal(first[1][k], first[3][k]) for k in got)


def test_other_lengths_and_shapes(cases):
    """Fewer and more rows in the same handles; another shape closes those that nobody has."""
    short, long = {**CASES[2], "rows": 85}, {**CASES[2], "rows": 88}          # (8 pages a sequence at most, both)
    want = {}
    for c in (long, short, long):
        got = answer(cases, cases.prepare(c, 5))
        for k in got:
            assert torch.equal(want.setdefault((c["rows"], k), got[k]), got[k])
    assert len(cases.made) == 1
    answer(cases, cases.prepare({**CASES[2], "nh": 8}, 5))
    assert len(cases.made) == 2 and len(cases._Owner.program.caches) == 1


def test_more_states_than_a_program_has_places_for(cases):
    want = [answer(cases, cases.prepare(CASES[1], seed)) for seed in range(7)]
    states = [cases.prepare(CASES[1], seed) for seed in range(7)]
    assert len({id(s["owner"].ctx) for s in states}) == 2 and len({id(s["cache"]) for s in states}) == 7
    for s, w in zip(states, want):
        got = answer(cases, s)
        assert all(torch.equal(got[k], w[k]) for k in got)
