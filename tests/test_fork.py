"""Forked requests in the cache manager: shared pages, copies, pages that go back when the last holder does, without a GPU."""
import random

import pytest

from celeg_b200.cache import NO_PAGE, CacheManager, OutOfPages, PageError, PagedNeed, StateLayout


def manager(pages=20, slots=6, window=None, page_tokens=4, cleared=None):
    needs = [PagedNeed(2, 8), PagedNeed(1, 8, window=window)]
    return CacheManager(page_tokens, [pages, pages], [(need.group_key() + (i,), need) for i, need in enumerate(needs)], StateLayout(), slots,
                        clear_slot=(cleared.append if cleared is not None else None), table_capacity=16)


def fill(m, name, tokens):
    cache = m.find(name) or m.open(name)
    m.reserve(cache, cache.tokens + tokens)
    m.advance(cache, cache.tokens + tokens)
    return cache


@pytest.mark.parametrize("tokens", [0, 1, 3, 4, 5, 8, 11])
def test_fork_shares_full_pages_and_copies_the_last(tokens):
    m = manager()
    a = fill(m, "a", tokens)
    b, copies = m.fork("a", "b")
    m.check_invariants()
    full, rest = divmod(tokens, 4)
    for g in range(2):
        assert b.tables[g][:full] == a.tables[g][:full]
        assert all(m.groups[g].pool.ref_count(page) == 2 for page in b.tables[g][:full])
        assert len(b.tables[g]) == full + (rest > 0)
        assert list(b.table_array(g)) == b.tables[g] and list(m.table_mirrors[g][b.slot][:len(b.tables[g])]) == b.tables[g]
        assert copies[g] == ([(a.tables[g][full], b.tables[g][full], rest)] if rest else [])
    assert b.tokens == tokens and b.slot != a.slot and b.capacity == 4 * (full + (rest > 0))
    fill(m, "a", 3)
    fill(m, "b", 6)
    m.check_invariants()
    m.close("a")
    m.check_invariants()
    assert [m.groups[0].pool.ref_count(page) for page in b.tables[0]] == [1] * len(b.tables[0])
    m.close("b")
    m.check_invariants()
    assert all(group.pool.free_pages == 20 for group in m.groups)


def test_fork_does_not_take_pages_that_were_only_reserved():
    m = manager()
    a = m.open("a")
    m.reserve(a, 14)
    m.advance(a, 5)
    b, copies = m.fork("a", "b")
    assert len(b.tables[0]) == 2 and copies[0] == [(a.tables[0][1], b.tables[0][1], 1)]
    m.check_invariants()


def test_fork_under_a_window():
    m = manager(window=5)
    a = fill(m, "a", 18)                    # the next query sees positions 14 ..: pages 0, 1 and 2 of group 1 are back
    assert a.tables[1][:3] == [NO_PAGE] * 3
    b, copies = m.fork("a", "b")
    m.check_invariants()
    assert b.tables[1][:3] == [NO_PAGE] * 3 and b.tables[1][3] == a.tables[1][3] and b.first_live_page == a.first_live_page
    fill(m, "a", 9)                         # releases a's hold on what b still shares
    m.check_invariants()
    assert m.groups[1].pool.ref_count(b.tables[1][3]) == 1
    fill(m, "b", 9)
    m.check_invariants()
    m.close("a")
    m.close("b")
    m.check_invariants()


def test_fork_is_all_or_nothing():
    cleared = []
    m = manager(pages=3, slots=3, cleared=cleared)
    fill(m, "a", 6)
    fill(m, "c", 4)
    before = [group.pool.free_pages for group in m.groups]
    with pytest.raises(OutOfPages):
        m.fork("a", "b")                    # no page for the copy
    assert m.find("b") is None and [group.pool.free_pages for group in m.groups] == before
    m.check_invariants()
    m.fork("c", "b")                        # a full page is shared: no page needed
    m.check_invariants()
    with pytest.raises(OutOfPages):
        m.fork("c", "d")                    # no slot
    with pytest.raises(KeyError):
        m.fork("nobody", "e")
    with pytest.raises(ValueError):
        m.fork("c", "a")                    # the new one is there already
    m.check_invariants()
    assert m.groups[0].pool.ref_count(m.get("c").tables[0][0]) == 2
    # ... and pages that are held as often as nobody says are found
    m.groups[0].pool.retain([m.get("a").tables[0][0]])
    with pytest.raises(PageError):
        m.check_invariants()


@pytest.mark.parametrize("seed", range(6))
def test_random_traffic_with_forks(seed):
    rng = random.Random(seed)
    m = manager(pages=30, slots=8, window=rng.choice([None, 3, 9]))
    live, made = [], 0
    for _ in range(400):
        kind = rng.random()
        try:
            if kind < 0.15 or not live:
                made += 1
                fill(m, made, rng.randrange(0, 9))
                live.append(made)
            elif kind < 0.35:
                made += 1
                m.fork(rng.choice(live), made)
                live.append(made)
            elif kind < 0.75:
                fill(m, rng.choice(live), rng.randrange(1, 6))
            else:
                m.close(live.pop(rng.randrange(len(live))))
        except OutOfPages:
            if m.find(made) is not None and made not in live:
                m.close(made)
        m.check_invariants()
    for name in live:
        m.close(name)
    m.check_invariants()
    assert all(group.pool.free_pages == 30 for group in m.groups)
