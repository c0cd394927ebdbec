"""Rotary positions: layouts, part of a head, positions, strides, types, the way back, scaled tables, refusals."""
import numpy as np
import pytest

from paged_reference import turn32, turn64

pytestmark = pytest.mark.gpu
HALF_ULP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}      # relative, of a rounding to the type (bf16: 2^-9, doubled)


def _torch():
    import torch
    return torch, {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _tables(rows, rot, seed=0):
    rng = np.random.default_rng(seed)
    a = rng.uniform(0, 2 * np.pi, (rows, rot // 2))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def _cuda(a):
    torch, _ = _torch()
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.mark.parametrize("tokens,heads,D,rot,layout,dtype", [
    (1, 1, 2, 2, "half", "f16"), (1, 32, 128, 128, "half", "f16"), (3, 5, 128, 128, "interleaved", "bf16"), (7, 3, 96, 72, "half", "f32"),
    (17, 2, 80, 32, "half", "f16"), (33, 7, 64, 64, "half", "bf16"), (5, 4, 100, 50, "interleaved", "f32"), (129, 8, 128, 64, "interleaved", "f16"),
    (2000, 16, 128, 96, "half", "f16"), (2000, 33, 128, 128, "interleaved", "f32"), (2, 70, 256, 256, "half", "bf16"), (9, 3, 13, 6, "half", "f16"),
])
@pytest.mark.parametrize("inverse", [False, True])
def test_against_64_bits(tc, ctx, tokens, heads, D, rot, layout, dtype, inverse):
    torch, types = _torch()
    rng = np.random.default_rng(tokens * 7 + D)
    rows = 501
    cos, sin = _tables(rows, rot)
    x = torch.from_numpy(rng.standard_normal((tokens, heads, D)).astype(np.float32)).cuda().to(types[dtype])
    pos = rng.integers(0, rows, tokens).astype(np.int32)
    y = torch.full_like(x, 7.0)
    desc = tc.rope_desc(tokens, heads, D, rot_dim=rot, layout=layout, dtype=dtype, table_rows=rows, inverse=inverse)
    c, s, p = _cuda(cos), _cuda(sin), _cuda(pos)
    tc.raw_rope(ctx, desc, x.data_ptr(), y.data_ptr(), c.data_ptr(), s.data_ptr(), p.data_ptr(), torch.cuda.current_stream().cuda_stream)
    want, room = turn64(x.float().cpu().numpy(), cos, sin, pos, rot, layout, inverse)
    got = y.float().cpu().numpy().astype(np.float64)
    assert np.all(abs(got - want) <= room + HALF_ULP[dtype] * abs(want) + 2.0 ** -25)
    assert tc.take_device_error(ctx) == 0
    if not inverse and dtype == "f32":
        assert np.array_equal(y.cpu().numpy(), turn32(x.cpu().numpy(), cos, sin, pos, rot, layout))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient_is_the_way_back(tc, ctx, layout):
    """The gradient of sum(g . rope(x)) by x: against differences, and against the transposed map."""
    torch, _ = _torch()
    rng = np.random.default_rng(3)
    T, H, D, rot = 4, 2, 64, 48
    cos, sin = _tables(T, rot)
    c, s = _cuda(cos), _cuda(sin)
    x, g = (rng.standard_normal((T, H, D)).astype(np.float32) for _ in range(2))

    def go(a, inverse):
        a = _cuda(a)
        y = torch.empty_like(a)
        tc.raw_rope(ctx, tc.rope_desc(T, H, D, rot_dim=rot, layout=layout, dtype="f32", table_rows=T, inverse=inverse), a.data_ptr(), y.data_ptr(),
                    c.data_ptr(), s.data_ptr(), 0, torch.cuda.current_stream().cuda_stream)
        return y.cpu().numpy().astype(np.float64)
    dx = go(g, True)
    want, room = turn64(g, cos, sin, np.arange(T), rot, layout, True)
    assert np.all(abs(dx - want) <= room + 2.0 ** -24 * abs(want))
    # <g, R x> = <R^T g, x>: each side a sum of T H D terms, every term off by 4 roundings at most
    assert abs(np.sum(g * go(x, False)) - np.sum(dx * x)) <= 4 * 2.0 ** -24 * 2 * np.sum(abs(g) * np.sqrt(2) * abs(x).max())
    # differences of a linear map: the step may be large, so only roundings are left
    f0 = np.sum(g * go(x, False))
    for i in range(0, T * H * D, 37):
        e = np.zeros(T * H * D, np.float32)
        e[i] = 64.0
        diff = (np.sum(g * go(x + e.reshape(x.shape), False)) - f0) / 64.0
        assert abs(diff - dx.reshape(-1)[i]) <= 64 * 2.0 ** -22 * abs(g).max()


def test_strides_places_and_streams(tc, ctx):
    """Heads-major rows, rows of a wider matrix, odd addresses, in place, on a stream of their own."""
    torch, _ = _torch()
    rng = np.random.default_rng(5)
    T, H, D, rows = 37, 6, 128, 64
    cos, sin = _tables(rows, D)
    pos = rng.integers(0, rows, T).astype(np.int32)
    c, s, p = _cuda(cos), _cuda(sin), _cuda(pos)
    x = torch.from_numpy(rng.standard_normal((T, H, D)).astype(np.float32)).cuda().half()
    want = torch.from_numpy(turn32(x.float().cpu().numpy(), cos, sin, pos, D, "half")).half()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        heads_first = x.transpose(0, 1).contiguous()                       # [H, T, D]
        wide = torch.zeros(T, 3 * H * D + 8, dtype=torch.float16, device="cuda")
        odd = torch.zeros(T * H * D + 1, dtype=torch.float16, device="cuda")[1:]
        for src, xs in ((heads_first, (D, T * D)), (x, (0, 0))):
            for dst, ys in ((torch.zeros_like(heads_first), (D, T * D)), (wide, (wide.stride(0), D)), (odd, (0, 0))):
                desc = tc.rope_desc(T, H, D, dtype="f16", table_rows=rows, x_strides=xs, y_strides=ys)
                tc.raw_rope(ctx, desc, src.data_ptr(), dst.data_ptr(), c.data_ptr(), s.data_ptr(), p.data_ptr(), stream.cuda_stream)
                stream.synchronize()
                got = dst.transpose(0, 1) if dst.shape == heads_first.shape else (wide[:, :H * D] if dst is wide else dst).reshape(T, H, D)
                assert torch.equal(got.cpu(), want)
        assert not wide[:, H * D:].any()
        for layout in ("half", "interleaved"):
            a, b = x.clone(), torch.empty_like(x)
            desc = tc.rope_desc(T, H, D, layout=layout, dtype="f16", table_rows=rows)
            tc.raw_rope(ctx, desc, x.data_ptr(), b.data_ptr(), c.data_ptr(), s.data_ptr(), p.data_ptr(), stream.cuda_stream)
            tc.raw_rope(ctx, desc, a.data_ptr(), a.data_ptr(), c.data_ptr(), s.data_ptr(), p.data_ptr(), stream.cuda_stream)
            stream.synchronize()
            assert torch.equal(a, b)


def test_same_bits_as_the_whole_head_form(tc, ctx):
    """tc_rope_forward on [1, heads, tokens, D] is this with the half layout and no positions; and the form on buffers."""
    rng = np.random.default_rng(6)
    T, H, D = 19, 4, 64
    cos, sin = _tables(T, D)
    x = rng.standard_normal((H, T, D)).astype(np.float16)
    bx, by, bc, bs = ctx.buffer_from_array(x), ctx.buffer(x.nbytes), ctx.buffer_from_array(cos), ctx.buffer_from_array(sin)
    tc.rope(ctx, tc.rope_desc(T, H, D, table_rows=T, x_strides=(D, T * D), y_strides=(D, T * D)), bx, by, bc, bs)
    tc.rope_forward(ctx, bx, bc, bs, 1, H, T, D)
    assert np.array_equal(bx.to_numpy(x.shape, np.float16).view(np.uint16), by.to_numpy(x.shape, np.float16).view(np.uint16))
    assert tc.cuda_last_kernel_name() == "rope_forward_sm100" and tc.last_backend() == tc.TC_BACKEND_CUDA


@pytest.mark.parametrize("D,rot", [(128, 128), (36, 12)])
def test_tokens_without_a_position(tc, ctx, D, rot):
    """Below zero: passed over.  Past the tables: passed over, and the device error word says so."""
    torch, _ = _torch()
    cos, sin = _tables(8, rot)
    c, s = _cuda(cos), _cuda(sin)
    x = torch.randn(5, 3, D, device="cuda")
    y = torch.full_like(x, 9.0)
    st = torch.cuda.current_stream().cuda_stream
    desc = tc.rope_desc(5, 3, D, rot_dim=rot, dtype="f32", table_rows=8)
    pos = _cuda(np.array([0, -1, 7, -5, 3], np.int32))
    tc.raw_rope(ctx, desc, x.data_ptr(), y.data_ptr(), c.data_ptr(), s.data_ptr(), pos.data_ptr(), st)
    torch.cuda.synchronize()
    assert (y[[1, 3]] == 9).all() and not (y[[0, 2, 4]] == 9).any() and tc.take_device_error(ctx) == 0
    pos = _cuda(np.array([0, 8, 7, 1 << 30, 3], np.int32))
    tc.raw_rope(ctx, desc, x.data_ptr(), y.data_ptr(), c.data_ptr(), s.data_ptr(), pos.data_ptr(), st)
    torch.cuda.synchronize()
    assert (y[[1, 3]] == 9).all() and tc.take_device_error(ctx) == 2
    assert tc.take_device_error(ctx) == 0


def _frequencies(rot, base, scaling, factor, original, fast, slow):
    """Radians a position in 64 bits, from the definitions."""
    k = np.arange(rot // 2)
    if scaling == "base":
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2.0 * k / rot)
    if scaling == "linear":
        return f / factor
    if scaling == "by_parts":
        def pair(turns):
            return rot * np.log(original / (turns * 2 * np.pi)) / (2 * np.log(base))
        low, high = max(np.floor(pair(fast)), 0), min(np.ceil(pair(slow)), rot // 2 - 1)
        kept = 1 - np.clip((k - low) / max(high - low, 1e-3), 0, 1)
        return kept * f + (1 - kept) * f / factor
    if scaling == "by_wavelength":
        kept = np.clip((original * f / (2 * np.pi) - slow) / (fast - slow), 0, 1)
        return kept * f + (1 - kept) * f / factor
    return f


@pytest.mark.parametrize("rot", [2, 64, 128])
@pytest.mark.parametrize("scaling,factor,fast,slow", [("plain", 1, 0, 0), ("linear", 4, 0, 0), ("base", 8, 0, 0), ("by_parts", 16, 32, 1),
                                                      ("by_wavelength", 8, 4, 1)])
def test_tables(tc, ctx, rot, scaling, factor, fast, slow):
    if scaling == "base" and rot == 2:
        with pytest.raises(tc.TensorcoreError):
            tc.rope_table(ctx, tc.rope_table_desc(4, 2, scaling="base", factor=2), ctx.buffer(64), ctx.buffer(64))
        return
    for first, rows in ((0, 3), (131072 - 5, 9)):
        bc, bs = ctx.buffer(rows * rot * 2), ctx.buffer(rows * rot * 2)
        tc.rope_table(ctx, tc.rope_table_desc(rows, rot, freq_base=500000.0, scaling=scaling, factor=factor, original_context=8192, first_row=first), bc, bs)
        f = _frequencies(rot, 500000.0, scaling, factor, 8192, fast, slow)
        a = np.arange(first, first + rows)[:, None] * f
        size = 0.1 * np.log(factor) + 1 if scaling == "by_parts" else 1.0
        # fp32 rounding of numbers up to `size`, and 2^17 radians off by some roundings of 2^-53
        for b, want in ((bc, np.cos(a)), (bs, np.sin(a))):
            assert np.all(abs(b.to_numpy((rows, rot // 2), np.float32) - size * want) <= size * (2.0 ** -24 + 2.0 ** 17 * 2.0 ** -50))


def test_refusals(tc, ctx):
    L = tc.lib()
    import ctypes
    b = ctx.buffer(4096)

    def status(**kw):
        args = dict(tokens=4, heads=2, head_dim=16, table_rows=8)
        args.update(kw)
        return L.tcx_rope(ctx.handle, ctypes.byref(tc.rope_desc(**args)), b.handle, b.handle, b.handle, b.handle, None)
    assert status() == tc.TC_OK
    assert L.tcx_rope(None, None, None, None, None, None, None) == tc.TC_ERR_NOT_INITIALIZED
    assert L.tcx_rope(ctx.handle, None, b.handle, b.handle, b.handle, b.handle, None) == tc.TC_ERR_INVALID_ARG
    assert L.tcx_rope(ctx.handle, ctypes.byref(tc.rope_desc(1, 1, 8)), b.handle, None, b.handle, b.handle, None) == tc.TC_ERR_INVALID_ARG
    for bad in (dict(tokens=0), dict(heads=-1), dict(head_dim=0), dict(rot_dim=3), dict(rot_dim=18), dict(rot_dim=-2), dict(table_rows=-1),
                dict(layout=7), dict(x_strides=(-1, 0)), dict(y_strides=(8, 0)), dict(y_strides=(0, 15)), dict(head_dim=15)):
        assert status(**bad) == tc.TC_ERR_INVALID_ARG, bad
    assert status(dtype=3) == tc.TC_ERR_UNSUPPORTED_DTYPE
    for bad in (dict(tokens=9), dict(tokens=8, heads=64), dict(table_rows=1000), dict(y_strides=(1 << 20, 0))):
        assert status(**bad) == tc.TC_ERR_INVALID_SHAPE, bad
    raw = tc.rope_desc(1, 1, 8)
    p = b.device_ptr()
    for args in ((p + 1, p, p, p), (p, p + 1, p, p), (p, p, p + 2, p), (p, p, p, p + 2)):
        assert L.tcx_raw_rope(ctx.handle, ctypes.byref(raw), *args, None, None) == tc.TC_ERR_INVALID_ARG
    for bad in (dict(rows=0), dict(rot_dim=7), dict(scaling=9), dict(factor=0.5), dict(scaling="by_parts", factor=2), dict(freq_base=float("nan"))):
        with pytest.raises(tc.TensorcoreError):
            tc.rope_table(ctx, tc.rope_table_desc(**{**dict(rows=2, rot_dim=8), **bad}), b, b)


@pytest.mark.parametrize("tokens,heads,D,rot,layout,dtype", [(9000, 30, 64, 40, "half", "f16"), (5200, 37, 64, 64, "half", "bf16"), (4801, 34, 128, 128, "interleaved", "bf16"),
                                                             (9001, 19, 96, 72, "half", "f32"), (9001, 22, 36, 20, "interleaved", "f16"), (9001, 18, 64, 8, "interleaved", "f32")])
def test_many_tokens_in_place(tc, ctx, tokens, heads, D, rot, layout, dtype):
    """Sizes from which a thread has several heads, a number of heads that leaves some over, pieces of 8 and of 4 elements."""
    torch, types = _torch()
    rng = np.random.default_rng(D + rot)
    cos, sin = _tables(300, rot)
    x = torch.from_numpy(rng.standard_normal((tokens, heads, D), dtype=np.float32)).cuda().to(types[dtype])
    pos = rng.integers(-1, 300, tokens).astype(np.int32)
    c, s, p, y = _cuda(cos), _cuda(sin), _cuda(pos), torch.full_like(x, 5.0)
    desc = tc.rope_desc(tokens, heads, D, rot_dim=rot, layout=layout, dtype=dtype, table_rows=300)
    st = torch.cuda.current_stream().cuda_stream
    want = turn32(x.float().cpu().numpy(), cos, sin, pos, rot, layout)
    passed = torch.from_numpy(pos < 0)
    tc.raw_rope(ctx, desc, x.data_ptr(), y.data_ptr(), c.data_ptr(), s.data_ptr(), p.data_ptr(), st)
    got, was = y.cpu(), x.cpu()
    assert torch.equal(got[~passed], torch.from_numpy(want).to(types[dtype])[~passed]) and bool((got[passed] == 5.0).all())
    tc.raw_rope(ctx, desc, x.data_ptr(), x.data_ptr(), c.data_ptr(), s.data_ptr(), p.data_ptr(), st)
    assert torch.equal(x.cpu()[~passed], got[~passed]) and torch.equal(x.cpu()[passed], was[passed])
