"""Attention over the paged cache where it can go wrong: values at the ends of their types, NaN, windows without an end, rows that a call
declares wrongly, lengths at the end of 32 bits."""
import ctypes

import numpy as np
import pytest

from paged_reference import attention64, numbers, pack, quantise
from test_gpu_attention_paged import Case, _cuda, _torch

pytestmark = pytest.mark.gpu


def put(c, s, keys, which, x=None, nan=(), inf=()):
    """Row x [Hkv, D] (or the one there) for `keys` of sequence s, K (0) or V (1); blocks in `nan` and `inf` with such a scale instead."""
    nb, shape = c.D // 32, (1, c.Hkv, 16)
    pages = c.pages.cpu().numpy()
    for key in keys:
        page, at, r = int(c.table[s, key // c.P]), key % c.P // 16, key % 16
        codes, scales = quantise(np.asarray(x, np.float32)) if x is not None else (None, None)
        full = [np.zeros(shape + (c.D,), np.uint8), np.zeros(shape + (nb,), np.uint16), np.zeros(shape + (c.D,), np.uint8), np.zeros(shape + (nb,), np.uint16)]
        mask = [a.copy() for a in full]
        blocks = list(nan) + list(inf) if x is None else range(nb)
        mask[2 * which + 1][0, :, r, list(blocks)] = 0xFFFF
        if x is not None:
            mask[2 * which][0, :, r] = 15
            full[2 * which][0, :, r] = codes
            full[2 * which + 1][0, :, r] = scales.view(np.uint16)
            (c.k, c.v)[which][s][:, key] = numbers(codes, scales)
        for b in nan:
            full[2 * which + 1][0, :, r, b] = 0x7E00
        for b in inf:
            full[2 * which + 1][0, :, r, b] = 0x7C00
        value, gone = (pack(a[0], a[1].view(np.float16), a[2], a[3].view(np.float16))[0, :, 0] for a in (full, mask))
        pages[page, :, at] = pages[page, :, at] & ~gone | value
    c.pages = _cuda(pages)


def same(a, b, rows=slice(None)):
    torch, _ = _torch()
    return all(torch.equal(x[rows], y[rows]) for x, y in zip(a, b))


def test_lengths_at_the_end_of_32_bits(tc, ctx):
    """A table may hold 2^31 - 4096 keys of a sequence, so that a step past the last key is still an int; the last length that there is, all on one page."""
    torch, _ = _torch()
    P, D, st = 1024, 64, torch.cuda.current_stream().cuda_stream
    c = Case(tc, [P], [1], 2, 1, D, P, seed=1)
    want, want_lse = c.run(tc, ctx)
    n = (2 ** 31 - 4096) // P
    table = torch.full((n + 1,), int(c.table[0, 0]), dtype=torch.int32, device="cuda")
    o, lse = torch.zeros_like(c.q), torch.zeros(1, 2, device="cuda")

    def status(pages, length):
        d = tc.attention_paged_desc(1, 1, pages, 2, max_q=1)
        lens = _cuda(np.array([length], np.int32))
        rc = tc.lib().tcx_raw_attention_paged(ctx.handle, ctypes.byref(c.kv), ctypes.byref(d), c.pages.data_ptr(), c.q.data_ptr(), table.data_ptr(), lens.data_ptr(), None,
                                              o.data_ptr(), lse.data_ptr(), st)
        torch.cuda.synchronize()
        return rc
    assert status(n + 1, 1) == tc.TC_ERR_INVALID_SHAPE
    assert status(n, n * P) == tc.TC_OK and tc.take_device_error(ctx) == 0
    # Every key n times as often.  A warp adds up 2^25 / 1776 steps of four products, each cut at 2^-23 of the sum.
    off = (2 ** 25 / 1776 + 64) * 4 * 2.0 ** -23
    assert (o.float() - want.float()).abs().max() <= (off + 2.0 ** -10) * want.float().abs().max()
    assert (lse - want_lse - np.log(n)).abs().max() <= off


def test_nan_in_a_query_of_a_prompt_in_chunks(tc, ctx):
    """A row whose scores are all NaN is NaN, not a row without keys, however many chunks its keys are cut into."""
    torch, _ = _torch()
    for keys, queries in (([5000], [130]), ([200], [130]), ([200, 300], [1, 3])):
        c = Case(tc, keys, queries, 2, 1, 128, 64, seed=3)
        want = c.run(tc, ctx)
        q = c.q.clone()
        q[0, 1, 5] = float("nan")
        o, lse = c.run(tc, ctx, q=q)
        assert o[0, 1].isnan().all() and lse[0, 1].isnan()
        assert torch.equal(o[:, 0], want[0][:, 0]) and torch.equal(o[1:], want[0][1:]) and torch.equal(lse[1:], want[1][1:])


def test_a_chunk_of_keys_that_are_nan(tc, ctx):
    """The first 512 keys - one chunk of nine - have NaN scales: rows that see them are NaN; rows whose window begins behind them keep their bits."""
    torch, _ = _torch()
    c = Case(tc, [5000], [130], 2, 1, 128, 64, seed=4)
    inside = c.run(tc, ctx, window=4300)
    put(c, 0, range(512), 0, nan=(0, 1, 2, 3))
    o, lse = c.run(tc, ctx)
    assert o.isnan().all() and lse.isnan().all()
    assert same(c.run(tc, ctx, window=4300), inside)
    assert c.run(tc, ctx, window=4860)[0].isnan().any(dim=(1, 2)).cpu().tolist() == [i - 4860 < 512 for i in range(4870, 5000)]
