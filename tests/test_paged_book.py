"""Pages that sequences have together, on the host: forked, kept in part, given back."""
import numpy as np
import pytest

from tensorcore_b200 import paged


def _users(book):
    """How many sequences have each page, counted from the table."""
    out = np.zeros(len(book._users), int)
    for s, n in enumerate(book.lengths):
        out[book.table[s, :-(-int(n) // book.page_tokens)]] += 1
    return out


def _sound(book):
    users = _users(book)
    assert (users == book._users).all() and sorted(book._free) == np.nonzero(users == 0)[0].tolist()
    for s, n in enumerate(book.lengths):
        assert (book.table[s, -(-int(n) // book.page_tokens):] == -1).all()


def test_forks_share_pages():
    book = paged.PageBook(n_pages=9, page_tokens=16, slots=4, max_pages=5)
    book.plan([40, 0, 0, 0])
    book.fork(0, 2)
    assert (book.table[0] == book.table[2]).all() and book.lengths.tolist() == [40, 0, 40, 0] and book.free_pages() == 6
    _sound(book)
    old = book.table[0, 2]
    plan = book.plan([8, 0, 3, 0])                           # the first to add has a copy, the other one the page
    assert plan.copies.tolist() == [[old, book.table[0, 2], 8]] and book.table[2, 2] == old and book.table[0, 2] != old
    assert plan.positions.tolist() == list(range(40, 48)) + [40, 41, 42] and book.free_pages() == 5
    _sound(book)
    assert len(book.plan([1, 0, 1, 0]).copies) == 0          # a new page, and one of its own
    _sound(book)
    book.fork(2, 1)
    plan = book.plan([0, 0, 1, 0])
    assert plan.copies.tolist() == [[old, book.table[2, 2], 12]] and book.table[1, 2] == old
    book.release(0)
    assert book.free_pages() == 9 - 2 - 2                    # two pages that both others have, and one of each
    _sound(book)
    book.release(2)
    book.release(1)
    assert book.free_pages() == 9
    _sound(book)
    book.plan([32, 0, 0, 0])
    book.fork(0, 3)
    assert len(book.plan([1, 0, 0, 1]).copies) == 0 and book.free_pages() == 5      # nothing to copy where the last page is full
    _sound(book)


def test_pages_enough_for_copies():
    """Sequences that add to one page need a copy each but for the last of its users; too few: nothing is changed."""
    for adders, needed in (([1, 1, 1], 2), ([1, 1, 0], 2), ([0, 1, 0], 1)):
        for free in (needed - 1, needed):
            book = paged.PageBook(n_pages=2 + free, page_tokens=16, slots=3, max_pages=3)
            book.plan([20, 0, 0])
            book.fork(0, 1)
            book.fork(0, 2)
            before = book.table.copy(), book.lengths.copy()
            if free < needed:
                with pytest.raises(paged.OutOfPages):
                    book.plan(adders)
                assert (book.table == before[0]).all() and (book.lengths == before[1]).all()
            else:
                assert len(book.plan(adders).copies) == needed and book.free_pages() == 0
            _sound(book)


def test_forks_that_cannot_be():
    book = paged.PageBook(n_pages=2, page_tokens=16, slots=3, max_pages=2)
    book.plan([20, 0, 0])
    for slot, to in ((0, 0), (1, 0)):
        with pytest.raises(ValueError):
            book.fork(slot, to)
    assert book.lengths.tolist() == [20, 0, 0]
    book.fork(1, 2)                                          # an empty sequence is one, too
    _sound(book)


def test_keeping_some_tokens():
    book = paged.PageBook(n_pages=8, page_tokens=16, slots=2, max_pages=6)
    book.plan([70, 0])
    assert book.keep(0, 64, [64, 66, 69]).tolist() == [64, 66, 69] and book.lengths[0] == 67 and book.free_pages() == 3
    assert book.keep(0, 4, list(range(40, 67))).tolist() == list(range(40, 67)) and book.lengths[0] == 31 and book.free_pages() == 6
    _sound(book)
    assert book.keep(0, 16, []).tolist() == [] and book.lengths[0] == 16 and book.free_pages() == 7
    _sound(book)
    for first, places in ((17, []), (-1, []), (0, [3, 3]), (0, [4, 3]), (2, [1]), (0, [16])):
        with pytest.raises(ValueError):
            book.keep(0, first, places)
    book.plan([24, 0])                                       # 40: two whole pages and eight tokens
    book.fork(0, 1)
    for first, places in ((0, [5, 6]), (32, [33, 39])):
        with pytest.raises(ValueError):
            book.keep(1, first, places)                      # would move tokens within the other's pages
    book.plan([0, 2])
    book.keep(1, 32, [33, 39, 41])                           # in its own
    assert book.lengths.tolist() == [40, 35]
    book.keep(1, 20, [])                                     # nothing moves: the page stays both's
    assert book.lengths.tolist() == [40, 20] and (book.table[0, :2] == book.table[1, :2]).all()
    _sound(book)
    plan = book.plan([0, 1])                                 # and is copied before it is written to
    assert plan.copies.tolist() == [[book.table[0, 1], book.table[1, 1], 4]]
    _sound(book)


def test_groups():
    book = paged.PageBook(n_pages=40, page_tokens=16, slots=7, max_pages=6)
    book.plan([50, 0, 0, 20, 0, 0, 5])
    for slot, to in ((0, 1), (0, 2), (3, 4)):
        book.fork(slot, to)
    start, shared = book.groups()
    assert start.tolist() == [0, 3, 5, 6, 7] and shared.tolist() == [48, 16, 0, 0]
    book.keep(2, 32, [])                                     # fewer in common: for all of the run
    assert book.groups()[1].tolist() == [32, 16, 0, 0]
    book.release(1)                                          # a slot in between that is empty ends a run
    assert book.groups()[0].tolist() == [0, 1, 2, 3, 5, 6, 7] and book.groups()[1].tolist() == [0, 0, 0, 16, 0, 0]
    assert start.dtype == shared.dtype == np.int32


def test_a_page_in_two_places_is_not_taken_for_a_group():
    book = paged.PageBook(n_pages=8, page_tokens=16, slots=2, max_pages=4)
    book.plan([32, 32])
    assert book.groups()[1].tolist() == [0, 0]


def test_the_length_without_what_others_may_have_more_of():
    b = paged.PageBook(8, 16, 3, 4)
    b.plan([40, 32, 0])
    assert [b.whole_or_own(s) for s in range(3)] == [40, 32, 0]
    b.fork(0, 2)
    assert [b.whole_or_own(s) for s in range(3)] == [32, 32, 32]
    b.plan([0, 0, 1])                                        # a copy of its own
    assert [b.whole_or_own(s) for s in range(3)] == [40, 32, 41]
