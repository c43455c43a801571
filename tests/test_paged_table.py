"""CPU: the page bookkeeping of fpga_qwen_b200/paged.py (no device)."""
import random

import pytest

from fpga_qwen_b200.paged import PageTable
from fpga_qwen_b200.qattn import QA_ERR_CAPACITY, QA_ERR_INVALID, QA_ERR_STATE, QAttnError


def held(t):
    return [p for pages in t.pages if pages for p in pages]


def test_pages_are_handed_out_as_rows_come_and_returned():
    t = PageTable(n_pages=5, page_rows=16, max_seqs=2, max_rows=64)
    a = t.open()
    assert t.grow({a: 1}) == [(a, 0, 0)] and t.grow({a: 15}) == []
    assert t.grow({a: 1}) == [(a, 1, 1)]
    b = t.open()
    assert t.grow({a: 1, b: 33}) == [(b, 0, 2), (b, 1, 3), (b, 2, 4)]
    assert (t.rows, t.position) == ([18, 33], [18, 33])
    with pytest.raises(QAttnError) as err:
        t.open()
    assert err.value.status == QA_ERR_CAPACITY
    t.shrink(b, 16)                                     # an eviction: the position stays
    assert (t.rows[b], t.position[b], t.pages[b]) == (16, 33, [2]) and sorted(t.free) == [3, 4]
    assert t.grow({b: 1}) == [(b, 1, 3)]
    t.close(a)
    assert sorted(t.free) == [0, 1, 4] and t.live() == [b]
    assert t.open() == a and (t.rows[a], t.position[a]) == (0, 0)


def test_what_does_not_fit_changes_nothing():
    t = PageTable(n_pages=3, page_rows=16, max_seqs=3, max_rows=40)
    a, b = t.open(), t.open()
    t.grow({a: 20})
    before = ([list(p) if p is not None else None for p in t.pages], list(t.rows), list(t.position), list(t.free))
    for counts, status in [({a: 21}, QA_ERR_CAPACITY), ({a: 1, b: 17}, QA_ERR_CAPACITY), ({a: 0}, QA_ERR_INVALID),
                           ({2: 1}, QA_ERR_STATE), ({-1: 1}, QA_ERR_STATE), ({3: 1}, QA_ERR_STATE)]:
        with pytest.raises(QAttnError) as err:
            t.grow(counts)
        assert err.value.status == status
    for call in (lambda: t.shrink(a, 21), lambda: t.shrink(a, -1), lambda: t.shrink(2, 0), lambda: t.close(2)):
        with pytest.raises(QAttnError) as err:
            call()
        assert err.value.status == QA_ERR_STATE
    assert before == (t.pages, t.rows, t.position, t.free)
    for bad in ((0, 16, 1, 1), (1, 0, 1, 1), (1, 16, 0, 1), (1, 16, 1, 0)):
        with pytest.raises(QAttnError):
            PageTable(*bad)


def test_random_life_never_shares_or_loses_a_page():
    r = random.Random(5)
    t = PageTable(n_pages=40, page_rows=32, max_seqs=6, max_rows=300)
    for _ in range(4000):
        live = t.live()
        try:
            what = r.random()
            if what < 0.1:
                t.open()
            elif what < 0.15 and live:
                t.close(r.choice(live))
            elif what < 0.25 and live:
                s = r.choice(live)
                t.shrink(s, r.randrange(0, t.rows[s] + 1))
            elif live:
                t.grow({s: r.randrange(1, 40) for s in r.sample(live, r.randrange(1, len(live) + 1))})
        except QAttnError as e:
            assert e.status == QA_ERR_CAPACITY
        assert sorted(held(t) + t.free) == list(range(40))
        for pages, rows, pos in zip(t.pages, t.rows, t.position):
            assert rows == 0 if pages is None else len(pages) == -(-rows // 32) and rows <= min(pos, 300)
