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


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("queries,keys,H,Hkv,D,window", [([200], [300], 4, 2, 128, 0), ([130], [5000], 2, 1, 128, 0), ([90, 130, 1, 20], [200, 131, 40, 300], 8, 2, 64, 0),
                                                         ([64] * 20, [100] * 20, 32, 8, 96, 30), ([100, 70], [100, 90], 4, 1, 32, 25), ([1, 5], [200, 90], 8, 2, 128, 40),
                                                         ([3, 8, 2], [700, 64, 2], 4, 2, 64, 0)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_magnitudes_beyond_half_precision(tc, ctx, queries, keys, H, Hkv, D, window, which, dtype):
    """K and V up to 2^19 (rows appended from bf16 or fp32): rows that do not see them keep their bits, rows that do are right."""
    torch, _ = _torch()
    c = Case(tc, keys, queries, H, Hkv, D, 16, dtype, seed=D + which)
    scale = 1e-5 if which == 0 else 0.0                                # scores of large keys near one
    before = c.run(tc, ctx, window=window, scale=scale)
    rng = np.random.default_rng(7)
    at = {}
    for s, (q, k) in enumerate(zip(queries, keys)):
        if k - 1 - q // 2 >= 0:
            at[s] = k - 1 - q // 2                                     # seen from the middle query on
            x = rng.standard_normal((Hkv, D))
            x[:, 5] = -7.0                                             # a scale above 8192 in the first block
            put(c, s, [at[s]], which, x * (3.0e4 if dtype == "bf16" or which == 0 else 1.2e4))
    o, lse = c.run(tc, ctx, window=window, scale=scale)
    pos = np.concatenate([np.arange(k - q, k) for q, k in zip(queries, keys)])
    key = np.concatenate([np.full(q, at.get(s, 1 << 30)) for s, q in enumerate(queries)])
    sees = (pos >= key) & ((pos - key <= window) if window else True)
    assert sees.any() and not sees.all()
    assert same((o, lse), before, torch.from_numpy(~sees).cuda())
    if dtype == "bf16":
        c.check(o, lse, window=window, scale=scale or None)
    else:                                                              # results may be above 65504 themselves
        want = torch.cat([torch.from_numpy(attention64(c.q[c.start[s]:c.start[s + 1]].double().cpu().numpy(), c.k[s], c.v[s], scale or D ** -0.5, True, window)[0])
                          for s in range(len(keys))])
        small = want.abs() < 6.0e4
        assert small.float().mean() > 0.9 and (o.cpu().double() - want)[small].abs().max() <= 2.0 ** -9 * want[small].abs().max()
    assert tc.take_device_error(ctx) == 0


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30])
@pytest.mark.parametrize("queries,keys,H,Hkv", [([150, 150, 150], [75, 0, 148], 4, 2), ([3, 4, 5], [1, 2, 0], 4, 2), ([40, 40], [10, 38], 2, 2), ([1, 1], [90, 7], 8, 1)])
def test_windows_that_hide_nothing(tc, ctx, queries, keys, H, Hkv, window, causal):
    """Windows up to the largest int, also where queries are more than keys and the first ones lie before position zero."""
    c = Case(tc, keys, queries, H, Hkv, 64, 16, seed=sum(queries))
    want = c.run(tc, ctx, causal=causal)
    c.check(*want, causal=causal)
    assert same(c.run(tc, ctx, causal=causal, window=window), want)


@pytest.mark.parametrize("used", [0, 1, 3, 20])
@pytest.mark.parametrize("keys", [60, 4000])
def test_one_sequence_of_fewer_queries_than_tokens(tc, ctx, keys, used):
    """A step padded to 64 tokens (a captured one) whose only sequence has few queries: they are answered, what is behind them is left."""
    torch, _ = _torch()
    c = Case(tc, [keys], [used], 4, 2, 64, 16, seed=used + 1)
    q = torch.zeros(64, 4, 64, device="cuda").half()
    q[:used] = c.q
    o = torch.full_like(q, 3.0)
    lse = torch.full((64, 4), 3.0, device="cuda")
    t, l, b = _cuda(c.table), _cuda(np.array([keys], np.int32)), _cuda(c.start)
    for max_q in (0, 64):
        o.fill_(3.0)
        lse.fill_(3.0)
        tc.raw_attention_paged(ctx, c.kv, tc.attention_paged_desc(64, 1, c.table.shape[1], 4, max_q=max_q), c.pages.data_ptr(), q.data_ptr(), t.data_ptr(), l.data_ptr(),
                               b.data_ptr(), o.data_ptr(), lse.data_ptr(), torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        c.check(o[:used], lse[:used])
        assert (o[used:] == 3).all() and (lse[used:] == 3).all()
    assert tc.take_device_error(ctx) == 0


@pytest.mark.parametrize("queries,max_q", [([300, 20, 260], 40), ([20, 700], 100), ([513], 100), ([100] * 12 + [140], 100)])
def test_more_queries_than_declared(tc, ctx, queries, max_q):
    """max_q below a sequence's queries: either every row is right, or the error word says that rows may be missing."""
    c = Case(tc, [q + 30 for q in queries], queries, 4, 2, 64, 16, seed=len(queries))
    got = c.run(tc, ctx, max_q=max_q)
    error = tc.take_device_error(ctx)
    assert error in (0, 2)
    if error == 0:
        c.check(*got)
    c.check(*c.run(tc, ctx, max_q=max(queries)))
    assert tc.take_device_error(ctx) == 0


@pytest.mark.parametrize("queries", [[1, 1, 1], [5, 2, 1], [40, 3, 60], [130, 1, 1]])
@pytest.mark.parametrize("extra", [150, 5000])
def test_values_that_are_nan_show_however_small_their_weight(tc, ctx, queries, extra):
    """Scores hundreds apart: the weight of a key is zero in fp32, its value NaN or infinite, and a row that sees it is NaN in that block."""
    torch, _ = _torch()
    keys = [q + extra for q in queries]
    c = Case(tc, keys, queries, 8, 2, 128, 64, seed=12, size=20.0)
    for s in range(3):
        put(c, s, [3], 1, nan=(0,))
        put(c, s, [4], 1, x=np.concatenate([np.ones((2, 96)), np.full((2, 32), np.inf)], axis=1))      # as an infinity is appended: codes of zero
    o, lse = c.run(tc, ctx, scale=1.0)
    assert o[..., :32].isnan().all() and o[..., 96:].isnan().all() and o[..., 32:96].isfinite().all() and lse.isfinite().all()
    o, lse = c.run(tc, ctx, scale=1.0, window=100)                     # the first keys are out of sight
    assert o.isfinite().all() and lse.isfinite().all()


@pytest.mark.parametrize("queries,keys,H,Hkv,D", [([1] * 8, [1, 2, 3, 5, 9, 40, 300, 2000], 32, 8, 128), ([4] * 4, [5, 40, 300, 1100], 8, 2, 64), ([130, 64, 33], [130, 500, 40], 8, 2, 128),
                                                  ([100], [3000], 4, 1, 128), ([64] * 19, [64 + 5 * i for i in range(19)], 32, 8, 96)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_scores_are_exact_but_for_fp32_sums(tc, ctx, queries, keys, H, Hkv, D, dtype):
    """The log-sum-exp shows the scores: products of whole queries and keys summed in fp32 (a K rounded to 11 bits is off by ten times the bound)."""
    c = Case(tc, keys, queries, H, Hkv, D, 16, dtype, seed=D)
    o, lse = c.run(tc, ctx)
    q, got = c.q.double().cpu().numpy(), o.double().cpu().numpy()
    off = near = 0.0
    for s in range(len(keys)):
        rows = slice(c.start[s], c.start[s + 1])
        want, want_lse, _, score = attention64(q[rows], c.k[s], c.v[s], D ** -0.5, True, 0)
        # `score` is 2^-11 of the sum of a row's largest terms.  Up to 16 products of 16 terms are added up, each time cut at
        # 2^-22 of the terms: 2^-18; exponentials and their sum 2^-21, the logarithm and its product 2^-22 of the result.
        assert np.all(abs(lse.cpu().numpy()[rows] - want_lse) <= 2.0 ** -7 * score + 2.0 ** -21 + 2.0 ** -22 * abs(want_lse))
        off, near = off + np.sum((got[rows] - want) ** 2), near + np.sum(want ** 2)
    # the result's rounding, 2^-10 / sqrt(12) or 2^-7 / sqrt(12) of the power of two below (a factor of 0.72 over a binade), and for
    # fp16 that of values or weights to 11 bits, as much again at most; a fifth on top
    ulp = 2.0 ** -10 if dtype == "f16" else 2.0 ** -7
    assert np.sqrt(off / near) <= 1.2 * 0.72 * ulp / np.sqrt(12) * (np.sqrt(2) if dtype == "f16" else 1.0)
