"""What of the calls for shared, moved and chosen pages needs no GPU: sizes, refusals without a context."""
import pytest


def test_bytes_of_bounds(tc):
    for D in (32, 64, 96, 128):
        assert tc.kv_bounds_bytes(tc.kv_desc(3, 16, 2, D)) == 2 * D + 16
    for n, P, heads, D in ((0, 16, 1, 32), (1, 8, 1, 32), (1, 16, 0, 32), (1, 16, 1, 48), (1, 16, 1, 160)):
        assert tc.kv_bounds_bytes(tc.kv_desc(n, P, heads, D)) == 0


def test_without_a_context(tc):
    kv = tc.kv_desc(1, 16, 1, 32)
    calls = [lambda: tc.raw_kv_copy(None, kv, tc.kv_copy_desc(1), 16, 16, 16), lambda: tc.raw_kv_compact(None, kv, tc.kv_compact_desc(1, 1, 1), 16, 16, 16, 16, 16),
             lambda: tc.raw_attention_shared(None, kv, tc.attention_shared_desc(1, 1, 1, 1, 1), 16, 16, 16, 16, 0, 16, 16, 16),
             lambda: tc.raw_kv_bounds(None, kv, tc.kv_bounds_desc(1, 1), 16, 16, 16, 16, 16), lambda: tc.raw_kv_select(None, kv, tc.kv_select_desc(1, 1, 1, 1, 1), *[16] * 8),
             lambda: tc.raw_attention_blocks(None, kv, tc.attention_blocks_desc(1, 1, 1), 16, 16, 16, 16, 16)]
    for call in calls:
        with pytest.raises(tc.TensorcoreError) as e:
            call()
        assert e.value.status == tc.TC_ERR_NOT_INITIALIZED
