"""Rotary tables at the ends of their scalings."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rot,base,original,factor", [(128, 10000.0, 131072, 4), (64, 10000.0, 262144, 8), (128, 500000.0, 8192, 16), (32, 100.0, 65536, 2), (8, 10.0, 10 ** 9, 2)])
def test_by_parts_where_every_pair_turns_often(tc, ctx, rot, base, original, factor):
    """The frequencies go over linearly up to the pair that turns `slow` times, also where that one is past the last pair (but no further than rot - 1)."""
    k = np.arange(rot // 2)
    f = base ** (-2.0 * k / rot)
    pair = lambda turns: rot * np.log(original / (turns * 2 * np.pi)) / (2 * np.log(base))
    low, high = max(np.floor(pair(32.0)), 0.0), min(np.ceil(pair(1.0)), rot - 1.0)
    kept = 1 - np.clip((k - low) / max(high - low, 1e-3), 0, 1)
    f = kept * f + (1 - kept) * f / factor
    rows, first, size = 7, 1000, 0.1 * np.log(factor) + 1
    bc, bs = ctx.buffer(rows * rot * 2), ctx.buffer(rows * rot * 2)
    tc.rope_table(ctx, tc.rope_table_desc(rows, rot, freq_base=base, scaling="by_parts", factor=factor, original_context=original, first_row=first), bc, bs)
    a = np.arange(first, first + rows)[:, None] * f
    for b, want in ((bc, np.cos(a)), (bs, np.sin(a))):
        assert np.all(abs(b.to_numpy((rows, rot // 2), np.float32) - size * want) <= size * (2.0 ** -24 + 2.0 ** 10 * 2.0 ** -50))
