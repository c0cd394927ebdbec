"""What of the rotary, cache and paged-attention calls needs no GPU: page sizes, refusals without a context, descriptors, and the
bookkeeping of pages."""
import pytest

from tensorcore_b200 import paged


def test_page_bytes(tc):
    for heads, D, P in ((1, 32, 16), (8, 128, 64), (5, 96, 1024), (2, 64, 32)):
        assert tc.kv_page_bytes(tc.kv_desc(3, P, heads, D)) == heads * P * 2 * (D // 32) * 18
    for n, P, heads, D in ((0, 16, 1, 32), (1, 8, 1, 32), (1, 24, 1, 32), (1, 2048, 1, 32), (1, 16, 0, 32), (1, 16, 1, 48), (1, 16, 1, 160), (-1, 16, 1, 32)):
        assert tc.kv_page_bytes(tc.kv_desc(n, P, heads, D)) == 0


def test_without_a_context(tc):
    kv = tc.kv_desc(1, 16, 1, 32)
    calls = [lambda: tc.raw_rope(None, tc.rope_desc(1, 1, 32), 16, 16, 16, 16), lambda: tc.raw_rope_table(None, tc.rope_table_desc(4, 32), 16, 16),
             lambda: tc.raw_kv_append(None, kv, tc.kv_append_desc(1, 1, 1), 16, 16, 16, 0, 0, 0, 0, 16, 16, 16),
             lambda: tc.raw_kv_read(None, kv, tc.kv_read_desc(1, 1, 1), 16, 16, 16, 16, 16, 16),
             lambda: tc.raw_attention_paged(None, kv, tc.attention_paged_desc(1, 1, 1, 1), 16, 16, 16, 16, 0, 16)]
    for call in calls:
        with pytest.raises(tc.TensorcoreError) as e:
            call()
        assert e.value.status == tc.TC_ERR_NOT_INITIALIZED


def test_options_by_name(tc):
    with pytest.raises(ValueError):
        tc.rope_desc(1, 1, 32, layout="neighbours")
    with pytest.raises(ValueError):
        tc.rope_table_desc(1, 32, scaling="none")


def test_pages_are_given_and_taken_back():
    book = paged.PageBook(n_pages=5, page_tokens=16, slots=3, max_pages=4)
    a = book.plan([17, 16, 0])
    assert a.positions.tolist() == list(range(17)) + list(range(16)) and a.sequences.tolist() == [0] * 17 + [1] * 16
    assert a.starts.tolist() == [0, 17, 33, 33] and a.lengths.tolist() == [17, 16, 0]
    used = book.table[0, :2].tolist() + book.table[1, :1].tolist()
    assert sorted(set(used)) == sorted(used) and book.free_pages() == 2
    b = book.plan([0, 1, 16])
    assert b.positions.tolist() == [16] + list(range(16)) and b.lengths.tolist() == [17, 17, 16] and book.free_pages() == 0
    before = book.table.copy(), book.lengths.copy()
    with pytest.raises(paged.OutOfPages):
        book.plan([16, 1, 1])                               # a page for sequence 0 and one for 2: neither is taken
    assert (book.table == before[0]).all() and (book.lengths == before[1]).all()
    with pytest.raises(ValueError):
        book.plan([1, 2])
    with pytest.raises(ValueError):
        book.plan([1, -1, 0])
    book.release(0)
    assert book.free_pages() == 2 and book.lengths.tolist() == [0, 17, 16]
    with pytest.raises(paged.OutOfPages):
        book.plan([65, 0, 0])                               # longer than a sequence may be
    assert book.plan([15, 0, 1]).lengths.tolist() == [15, 17, 17]
