"""The paged 4-bit cache: bytes written, rows read back, rotation on the way, odd places, refusals."""
import ctypes

import numpy as np
import pytest

from paged_reference import numbers, pack, quantise, turn32

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch, {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _cuda(a):
    torch, _ = _torch()
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _tables(rows, rot):
    a = np.arange(rows)[:, None] * 10000.0 ** (-np.arange(0, rot, 2) / rot)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


class Cache:
    """Sequences with pages in no order, and the same cache as codes and scales."""

    def __init__(self, tc, lens, kv_heads, D, P, seed):
        rng = np.random.default_rng(seed)
        n = [-(-k // P) for k in lens]
        self.kv, total = tc.kv_desc(sum(n) + 2, P, kv_heads, D), sum(n) + 2
        self.table, at, order = np.full((len(lens), max(1, max(n))), -1, np.int32), 0, rng.permutation(total)
        for s, k in enumerate(n):
            self.table[s, :k] = order[at:at + k]
            at += k
        shape = (total, kv_heads, P)
        self.codes = [np.zeros(shape + (D,), np.uint8) for _ in range(2)]
        self.scales = [np.zeros(shape + (D // 32,), np.float16) for _ in range(2)]
        assert tc.kv_page_bytes(self.kv) == kv_heads * P * D * 18 // 16
        torch, _ = _torch()
        self.pages = torch.zeros(total * tc.kv_page_bytes(self.kv), dtype=torch.uint8, device="cuda")
        self.P = P

    def put(self, seq, pos, k, v):
        for which, x in enumerate((k, v)):
            c, d = quantise(x)
            for t in range(len(pos)):
                if pos[t] >= 0:
                    page = self.table[seq[t], pos[t] // self.P]
                    self.codes[which][page, :, pos[t] % self.P] = c[t]
                    self.scales[which][page, :, pos[t] % self.P] = d[t]

    def bytes(self):
        return pack(self.codes[0], self.scales[0], self.codes[1], self.scales[1])


@pytest.mark.parametrize("D,P,heads,q_heads,rot,layout,dtype", [
    (32, 16, 1, 1, 32, "half", "f32"), (64, 32, 3, 6, 64, "half", "f16"), (96, 16, 2, 0, 96, "interleaved", "bf16"), (128, 64, 8, 32, 128, "half", "f16"),
    (128, 128, 1, 8, 64, "interleaved", "f32"), (96, 64, 5, 5, 40, "half", "f16"), (128, 16, 4, 4, 96, "half", "bf16"), (64, 16, 2, 4, 0, "half", "f16"),
])
@pytest.mark.parametrize("odd", [False, True])
def test_bytes_of_the_pages(tc, ctx, D, P, heads, q_heads, rot, layout, dtype, odd):
    """Ragged pieces of sequences, in rows of a fused projection (aligned, or at an odd element), against packing by hand."""
    torch, types = _torch()
    rng = np.random.default_rng(D + P + heads)
    lens = [1, 16, 17, 2 * P + 5, 40]
    cache = Cache(tc, lens, heads, D, P, 3)
    seq = np.concatenate([np.full(n, s) for s, n in enumerate(lens)]).astype(np.int32)
    pos = np.concatenate([np.arange(n) for n in lens]).astype(np.int32)
    order = rng.permutation(len(seq))                                        # tokens in no order
    seq, pos = seq[order], pos[order]
    T, n = len(seq), q_heads + 2 * heads
    flat = torch.from_numpy((rng.standard_normal(T * n * D + 1) * np.exp(rng.standard_normal(T * n * D + 1))).astype(np.float32)).cuda().to(types[dtype])
    x = flat[int(odd):int(odd) + T * n * D].view(T, n, D)
    q, k, v = x[:, :q_heads], x[:, q_heads:q_heads + heads], x[:, q_heads + heads:]
    rows = max(lens)
    cos, sin = _tables(rows, rot or 2)
    c, s = _cuda(cos), _cuda(sin)
    out = torch.zeros(T, max(1, q_heads), D, dtype=types[dtype], device="cuda")
    desc = tc.kv_append_desc(T, len(lens), cache.table.shape[1], q_heads=q_heads, rot_dim=rot, layout=layout, dtype=dtype, table_rows=rows,
                             k_strides=x.stride()[:2], v_strides=x.stride()[:2], q_strides=x.stride()[:2])
    ps, sq, tb = _cuda(pos), _cuda(seq), _cuda(cache.table)
    st = torch.cuda.current_stream().cuda_stream
    args = (c.data_ptr(), s.data_ptr()) if rot else (0, 0)
    tc.raw_kv_append(ctx, cache.kv, desc, cache.pages.data_ptr(), k.data_ptr(), v.data_ptr(), q.data_ptr() if q_heads else 0, out.data_ptr() if q_heads else 0,
                     *args, ps.data_ptr(), sq.data_ptr(), tb.data_ptr(), st)
    kf, vf, qf = (a.float().cpu().numpy() for a in (k, v, q))
    if rot:
        kf, qf = (turn32(a, cos, sin, pos, rot, layout) for a in (kf, qf))
    cache.put(seq, pos, kf, vf)
    assert np.array_equal(cache.pages.cpu().numpy().reshape(cache.bytes().shape), cache.bytes())
    if q_heads:
        assert torch.equal(out.cpu(), torch.from_numpy(qf).to(types[dtype]))
    # and back: every number is exact in fp32, and rounded once in the others
    for to in ("f32", "f16", "bf16"):
        rk, rv = (torch.zeros(T, heads, D, dtype=types[to], device="cuda") for _ in range(2))
        tc.raw_kv_read(ctx, cache.kv, tc.kv_read_desc(T, len(lens), cache.table.shape[1], dtype=to), cache.pages.data_ptr(), rk.data_ptr(), rv.data_ptr(),
                       ps.data_ptr(), sq.data_ptr(), tb.data_ptr(), st)
        for got, a in ((rk, kf), (rv, vf)):
            assert torch.equal(got.cpu(), torch.from_numpy(numbers(*quantise(a))).float().to(types[to]))
    assert tc.take_device_error(ctx) == 0


def test_same_codes_as_the_weight_quantiser(tc, ctx, oracle):
    """A row that is not turned holds what tc_quantize_weights makes of it (the oracle's bytes)."""
    rng = np.random.default_rng(8)
    T, D, P = 48, 128, 16
    x = (rng.standard_normal((T, 2, D)) * 3).astype(np.float16)
    x[5, 0, :64] = 0
    x[6, 1, 3] = 6e4
    q = oracle.quantize_weights(x.reshape(T * 2, D), 0).reshape(T, 2, D // 32, 18)
    codes = np.concatenate([q[..., 2:] & 15, q[..., 2:] >> 4], axis=-1)
    scales = np.ascontiguousarray(q[..., :2]).view(np.float16)[..., 0]
    kv = tc.kv_desc(T // P, P, 2, D)
    kb, pages = ctx.buffer_from_array(x), ctx.buffer(tc.kv_page_bytes(kv) * (T // P))
    pos, seq = ctx.buffer_from_array(np.arange(T, dtype=np.int32)), ctx.buffer_from_array(np.zeros(T, np.int32))
    table = ctx.buffer_from_array(np.arange(T // P, dtype=np.int32))
    tc.kv_append(ctx, kv, tc.kv_append_desc(T, 1, T // P), pages, kb, kb, None, None, None, None, pos, seq, table)
    rk, rv = ctx.buffer(T * 2 * D * 4), ctx.buffer(T * 2 * D * 4)
    tc.kv_read(ctx, kv, tc.kv_read_desc(T, 1, T // P, dtype="f32"), pages, rk, rv, pos, seq, table)
    want = ((codes.astype(np.float32) - 8) * scales.astype(np.float32)[..., None]).reshape(T, 2, D)
    for b in (rk, rv):
        assert np.array_equal(b.to_numpy((T, 2, D), np.float32), want)
    assert tc.cuda_last_kernel_name() == "kv_read_q4_0_sm100"


def test_single_tokens_without_sequences_and_queries_in_place(tc, ctx):
    torch, _ = _torch()
    rng = np.random.default_rng(9)
    n, H, Hq, D, P = 9, 2, 8, 128, 32
    lens = [int(v) for v in rng.integers(1, 100, n)]
    cache = Cache(tc, lens, H, D, P, 4)
    pos = np.array([k - 1 for k in lens], np.int32)
    pos[4] = -1                                                           # an idle slot
    x = torch.randn(n, Hq + 2 * H, D, device="cuda").half()
    before = x.clone()
    cos, sin = _tables(128, D)
    c, s, ps, tb = _cuda(cos), _cuda(sin), _cuda(pos), _cuda(cache.table)
    stride = x.stride()[:2]
    desc = tc.kv_append_desc(n, n, cache.table.shape[1], q_heads=Hq, table_rows=128, k_strides=stride, v_strides=stride, q_strides=stride, q_out_strides=stride)
    q, k, v = x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:]
    tc.raw_kv_append(ctx, cache.kv, desc, cache.pages.data_ptr(), k.data_ptr(), v.data_ptr(), q.data_ptr(), q.data_ptr(), c.data_ptr(), s.data_ptr(),
                     ps.data_ptr(), 0, tb.data_ptr(), torch.cuda.current_stream().cuda_stream)
    f = before.float().cpu().numpy()
    safe = np.maximum(pos, 0)
    cache.put(np.arange(n), pos, turn32(f[:, Hq:Hq + H], cos, sin, safe, D, "half"), f[:, Hq + H:])
    assert np.array_equal(cache.pages.cpu().numpy().reshape(cache.bytes().shape), cache.bytes())
    want = turn32(f[:, :Hq], cos, sin, safe, D, "half")
    want[4] = f[4, :Hq]
    assert torch.equal(x[:, :Hq].cpu(), torch.from_numpy(want).half()) and torch.equal(x[:, Hq:], before[:, Hq:])


def test_places_that_do_not_exist(tc, ctx):
    """A page, sequence or position that is not there: the token is passed over and the error word is set; the others are written."""
    torch, _ = _torch()
    H, D, P = 1, 64, 16
    kv = tc.kv_desc(4, P, H, D)
    pages = torch.full((4 * tc.kv_page_bytes(kv),), 0xAB, dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    x = torch.randn(6, 1, D, device="cuda").half()
    cos, sin = _tables(20, D)
    c, s = _cuda(cos), _cuda(sin)
    pos, seq = _cuda(np.array([3, 16, 40, 5, 21, 2], np.int32)), _cuda(np.array([0, 0, 0, 7, 1, -1], np.int32))
    table = _cuda(np.array([[2, 9], [-3, 1]], np.int32))
    # good; page 9 of 4; page slot 2 of 2; sequence 7; row 21 of 20 of the tables; sequence -1
    tc.raw_kv_append(ctx, kv, tc.kv_append_desc(6, 2, 2, table_rows=20), pages.data_ptr(), x.data_ptr(), x.data_ptr(), 0, 0, c.data_ptr(), s.data_ptr(),
                     pos.data_ptr(), seq.data_ptr(), table.data_ptr(), st)
    torch.cuda.synchronize()
    assert tc.take_device_error(ctx) == 2
    page = pages.view(4, -1)
    assert (page[[0, 1, 3]] == 0xAB).all() and (page[2] != 0xAB).sum() <= 2 * (32 + 4)
    out = torch.full((6, 1, D), 5.0, device="cuda")
    tc.raw_kv_read(ctx, kv, tc.kv_read_desc(6, 2, 2, dtype="f32"), pages.data_ptr(), out.data_ptr(), 0, pos.data_ptr(), seq.data_ptr(), table.data_ptr(), st)
    torch.cuda.synchronize()
    assert tc.take_device_error(ctx) == 2
    assert (out[[1, 2, 3, 5]] == 5).all() and not (out[0] == 5).any()


def test_infinities_and_nan(tc, ctx):
    """A NaN makes its block NaN, an infinity its block NaN or infinite, and no other block is touched."""
    x = np.ones((3, 1, 64), np.float32)
    x[0, 0, 7], x[1, 0, 40], x[2, 0, 0] = np.nan, np.inf, -1e38
    kv = tc.kv_desc(1, 16, 1, 64)
    pages, xb = ctx.buffer(tc.kv_page_bytes(kv)), ctx.buffer_from_array(x)
    pos, seq, table = (ctx.buffer_from_array(np.array(a, np.int32)) for a in ([0, 1, 2], [0, 0, 0], [0]))
    tc.kv_append(ctx, kv, tc.kv_append_desc(3, 1, 1, dtype="f32"), pages, xb, xb, None, None, None, None, pos, seq, table)
    for which in (0, 1):
        out = ctx.buffer(x.nbytes)
        tc.kv_read(ctx, kv, tc.kv_read_desc(3, 1, 1, dtype="f32"), pages, out if which == 0 else None, out if which else None, pos, seq, table)
        y = out.to_numpy(x.shape, np.float32)
        assert np.isnan(y[0, 0, :32]).all() and (y[0, 0, 32:] != 0).all() and np.isfinite(y[0, 0, 32:]).all()
        assert not np.isfinite(y[1, 0, 32:]).any() and np.isfinite(y[1, 0, :32]).all()
        assert not np.isfinite(y[2, 0, :32]).any() and np.isfinite(y[2, 0, 32:]).all()


def test_places_past_32_bits(tc, ctx):
    """Rows in pages that lie more than 4 GB into the cache."""
    torch, _ = _torch()
    kv = tc.kv_desc(1 << 15, 1024, 1, 128)
    each = tc.kv_page_bytes(kv)
    pages = torch.empty((1 << 15) * each, dtype=torch.uint8, device="cuda")
    table = _cuda(np.array([[1, (1 << 15) - 1]], np.int32))
    x = torch.randn(2, 1, 128, device="cuda").half()
    pos, seq = _cuda(np.array([1023, 2047], np.int32)), _cuda(np.zeros(2, np.int32))
    st = torch.cuda.current_stream().cuda_stream
    tc.raw_kv_append(ctx, kv, tc.kv_append_desc(2, 1, 2), pages.data_ptr(), x.data_ptr(), x.data_ptr(), 0, 0, 0, 0, pos.data_ptr(), seq.data_ptr(),
                     table.data_ptr(), st)
    small = tc.kv_desc(2, 1024, 1, 128)
    near = torch.cat([pages[each:2 * each], pages[-each:]])
    out = torch.zeros(2, 2, 1, 128, device="cuda")
    read = tc.kv_read_desc(2, 1, 2, dtype="f32")
    tc.raw_kv_read(ctx, kv, read, pages.data_ptr(), out[0].data_ptr(), 0, pos.data_ptr(), seq.data_ptr(), table.data_ptr(), st)
    near_table = _cuda(np.array([[0, 1]], np.int32))
    tc.raw_kv_read(ctx, small, read, near.data_ptr(), 0, out[1].data_ptr(), pos.data_ptr(), seq.data_ptr(), near_table.data_ptr(), st)
    want = torch.from_numpy(numbers(*quantise(x.float().cpu().numpy()))).float()
    assert torch.equal(out[0].cpu(), want) and torch.equal(out[1].cpu(), want) and tc.take_device_error(ctx) == 0


def test_refusals(tc, ctx):
    L, b = tc.lib(), ctx.buffer(1 << 16)
    kv, ok = tc.kv_desc(4, 16, 2, 64), dict(tokens=4, n_seqs=4, max_pages=1)
    h = b.handle

    def status(kv=kv, pages=h, k=h, q=None, q_out=None, cos=None, sin=None, **kw):
        return L.tcx_kv_append(ctx.handle, ctypes.byref(kv), ctypes.byref(tc.kv_append_desc(**{**ok, **kw})), pages, k, h, q, q_out, cos, sin, h, None, h)
    z = ctx.buffer_from_array(np.zeros(1 << 14, np.int32))
    assert L.tcx_kv_append(ctx.handle, ctypes.byref(kv), ctypes.byref(tc.kv_append_desc(**ok)), h, z.handle, z.handle, None, None, None, None, z.handle, None,
                           z.handle) == tc.TC_OK
    assert L.tcx_kv_append(None, *[None] * 12) == tc.TC_ERR_NOT_INITIALIZED
    assert L.tcx_kv_read(None, *[None] * 8) == tc.TC_ERR_NOT_INITIALIZED
    for bad in (dict(pages=None), dict(k=None), dict(tokens=0), dict(n_seqs=0), dict(max_pages=-1), dict(q_heads=-1), dict(q_heads=2), dict(q_heads=2, q=h),
                dict(cos=h), dict(cos=h, sin=h), dict(cos=h, sin=h, table_rows=4, rot_dim=3), dict(cos=h, sin=h, table_rows=4, rot_dim=66),
                dict(cos=h, sin=h, table_rows=4, layout=2), dict(k_strides=(-4, 0)), dict(q_heads=2, q=h, q_out=h, q_out_strides=(64, 0)),
                dict(kv=tc.kv_desc(0, 16, 2, 64)), dict(kv=tc.kv_desc(4, 16, 0, 64))):
        assert status(**bad) == tc.TC_ERR_INVALID_ARG, bad
    for bad in (dict(tokens=5), dict(tokens=4, n_seqs=4, k_strides=(1 << 20, 0)), dict(max_pages=1 << 20), dict(kv=tc.kv_desc(1 << 10, 16, 2, 64)),
                dict(kv=tc.kv_desc(4, 24, 2, 64)), dict(kv=tc.kv_desc(4, 8, 2, 64)), dict(kv=tc.kv_desc(4, 2048, 2, 64)), dict(kv=tc.kv_desc(4, 16, 2, 80)),
                dict(kv=tc.kv_desc(4, 16, 2, 160))):
        assert status(**bad) == tc.TC_ERR_INVALID_SHAPE, bad
    assert status(dtype=4) == tc.TC_ERR_UNSUPPORTED_DTYPE
    for kv_bad in (tc.kv_desc(4, 24, 2, 64), tc.kv_desc(-1, 16, 2, 64), tc.kv_desc(4, 16, 2, 33)):
        assert tc.kv_page_bytes(kv_bad) == 0
    p, d = b.device_ptr(), tc.kv_append_desc(**ok)
    good = [p, p, p, None, None, None, None, p, None, p]
    for at, off in ((0, 8), (1, 1), (2, 1), (7, 2), (9, 2)):
        args = list(good)
        args[at] += off
        assert L.tcx_raw_kv_append(ctx.handle, ctypes.byref(kv), ctypes.byref(d), *args, None) == tc.TC_ERR_INVALID_ARG
    r = tc.kv_read_desc(4, 4, 1)
    assert L.tcx_kv_read(ctx.handle, ctypes.byref(kv), ctypes.byref(r), h, None, None, h, None, h) == tc.TC_ERR_INVALID_ARG
    assert L.tcx_kv_read(ctx.handle, ctypes.byref(kv), ctypes.byref(tc.kv_read_desc(4, 4, 1, dtype=5)), h, h, None, h, None, h) == tc.TC_ERR_UNSUPPORTED_DTYPE
    assert L.tcx_kv_read(ctx.handle, ctypes.byref(kv), ctypes.byref(tc.kv_read_desc(5, 4, 1)), h, h, None, h, None, h) == tc.TC_ERR_INVALID_SHAPE


@pytest.mark.parametrize("D,heads,q_heads,rot,layout,dtype,odd", [(128, 3, 10, 128, "half", "f16", False), (128, 8, 0, 64, "interleaved", "bf16", False), (64, 5, 7, 64, "half", "f32", False),
                                                                  (96, 2, 9, 40, "half", "bf16", True), (32, 6, 6, 32, "half", "f16", False)])
def test_many_tokens(tc, ctx, D, heads, q_heads, rot, layout, dtype, odd):
    """Sizes from which a thread has several rows, numbers of heads that leave some over; queries turned in place."""
    torch, types = _torch()
    rng = np.random.default_rng(D + heads)
    n, P = q_heads + 2 * heads, 64
    T = -(-4 * 2048 * 148 // (n * {32: 4, 64: 8}.get(D, 16))) + 7
    lens = [T // 3, T - T // 3 - 1, 1]
    cache = Cache(tc, lens, heads, D, P, 3)
    seq = np.concatenate([np.full(k, i) for i, k in enumerate(lens)]).astype(np.int32)
    pos = np.concatenate([np.arange(k) for k in lens]).astype(np.int32)
    pos[::97] = -1                                                           # padding
    flat = torch.from_numpy((rng.standard_normal(T * n * D + 1) * 3).astype(np.float32)).cuda().to(types[dtype])
    flat[5 * n * D + q_heads * D:][:3] = float("nan")
    flat[6 * n * D + q_heads * D + 5] = float("inf")
    x = flat[int(odd):int(odd) + T * n * D].view(T, n, D)
    q, k, v = x[:, :q_heads], x[:, q_heads:q_heads + heads], x[:, q_heads + heads:]
    cos, sin = _tables(max(lens), rot)
    c, s, ps, sq, tb = _cuda(cos), _cuda(sin), _cuda(pos), _cuda(seq), _cuda(cache.table)
    st = torch.cuda.current_stream().cuda_stream
    desc = tc.kv_append_desc(T, len(lens), cache.table.shape[1], q_heads=q_heads, rot_dim=rot, layout=layout, dtype=dtype, table_rows=max(lens),
                             k_strides=x.stride()[:2], v_strides=x.stride()[:2], q_strides=x.stride()[:2], q_out_strides=x.stride()[:2] if q_heads else (0, 0))
    with np.errstate(all="ignore"):
        qf, kf = (turn32(a.float().cpu().numpy(), cos, sin, pos, rot, layout) for a in (q, k))
    vf, was = v.float().cpu().numpy(), q.cpu().clone()
    tc.raw_kv_append(ctx, cache.kv, desc, cache.pages.data_ptr(), k.data_ptr(), v.data_ptr(), q.data_ptr() if q_heads else 0, q.data_ptr() if q_heads else 0,
                     c.data_ptr(), s.data_ptr(), ps.data_ptr(), sq.data_ptr(), tb.data_ptr(), st)
    live = torch.from_numpy(pos >= 0)
    if q_heads:
        same = lambda a, b: np.array_equal(a.float().numpy(), b.float().numpy(), equal_nan=True)
        assert same(q.cpu()[live], torch.from_numpy(qf).to(types[dtype])[live]) and same(q.cpu()[~live], was[~live])
    rk, rv = (torch.full((T, heads, D), 7.0, device="cuda") for _ in range(2))
    tc.raw_kv_read(ctx, cache.kv, tc.kv_read_desc(T, len(lens), cache.table.shape[1], dtype="f32"), cache.pages.data_ptr(), rk.data_ptr(), rv.data_ptr(),
                   ps.data_ptr(), sq.data_ptr(), tb.data_ptr(), st)
    for got, a in ((rk, kf), (rv, vf)):
        with np.errstate(all="ignore"):
            want = numbers(*quantise(a)).astype(np.float32)
        assert np.array_equal(got.cpu().numpy()[pos >= 0], want[pos >= 0], equal_nan=True) and bool((got.cpu()[~live] == 7.0).all())
    assert tc.take_device_error(ctx) == 0


def test_pages_behind_four_gigabytes(tc, ctx):
    torch, _ = _torch()
    rng = np.random.default_rng(1)
    kv = tc.kv_desc(0, 64, 8, 128)
    kv.n_pages = 1
    far = (5 << 30) // tc.kv_page_bytes(kv)
    kv.n_pages = far + 2
    pages = torch.empty(kv.n_pages * tc.kv_page_bytes(kv), dtype=torch.uint8, device="cuda")
    T = 100
    k, v = (torch.from_numpy(rng.standard_normal((T, 8, 128)).astype(np.float32)).cuda() for _ in range(2))
    table, pos, seq = _cuda(np.array([[far + 1, far]], np.int32)), _cuda(np.arange(T, dtype=np.int32)), _cuda(np.zeros(T, np.int32))
    st = torch.cuda.current_stream().cuda_stream
    tc.raw_kv_append(ctx, kv, tc.kv_append_desc(T, 1, 2, dtype="f32"), pages.data_ptr(), k.data_ptr(), v.data_ptr(), 0, 0, 0, 0, pos.data_ptr(), seq.data_ptr(), table.data_ptr(), st)
    rk, rv = torch.zeros_like(k), torch.zeros_like(v)
    tc.raw_kv_read(ctx, kv, tc.kv_read_desc(T, 1, 2, dtype="f32"), pages.data_ptr(), rk.data_ptr(), rv.data_ptr(), pos.data_ptr(), seq.data_ptr(), table.data_ptr(), st)
    for got, a in ((rk, k), (rv, v)):
        assert np.array_equal(got.cpu().numpy(), numbers(*quantise(a.cpu().numpy())).astype(np.float32))
    assert tc.take_device_error(ctx) == 0
