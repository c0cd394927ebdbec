"""Attention over the paged 4-bit cache against 64 bits: lengths from nothing to long, ragged batches, masks, heads, refusals."""
import ctypes

import numpy as np
import pytest

from paged_reference import attention64, numbers, pack, quantise

pytestmark = pytest.mark.gpu
HALF_ULP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _torch():
    import torch
    return torch, {"f16": torch.float16, "bf16": torch.bfloat16}


def _cuda(a):
    torch, _ = _torch()
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Case:
    def __init__(self, tc, keys, queries, H, Hkv, D, P, dtype="f16", seed=0, size=1.0, spare=0xFF):
        """spare: the byte that everything is filled with which no sequence owns (0xFF: NaN scales)."""
        torch, types = _torch()
        rng = np.random.default_rng(seed)
        self.keys, self.queries, self.H, self.Hkv, self.D, self.P, self.dtype = keys, queries, H, Hkv, D, P, dtype
        n = [-(-k // P) for k in keys]
        total = sum(n) + 2
        self.table, at, order = np.full((len(keys), max(1, max(n))), 1 << 20, np.int32), 0, rng.permutation(total)
        shape = (total, Hkv, P)
        codes = [np.full(shape + (D,), spare & 15, np.uint8) for _ in range(2)]
        scales = [np.full(shape + (D // 32,), np.array([spare * 257], np.uint16).view(np.float16)[0], np.float16) for _ in range(2)]
        self.k, self.v = [], []
        for s, (m, nk) in enumerate(zip(n, keys)):
            own = order[at:at + m]
            self.table[s, :m] = own
            at += m
            for which, to in enumerate((self.k, self.v)):
                x = (rng.standard_normal((Hkv, nk, D)) * size).astype(np.float32)
                if which == 0:
                    x[:, :, ::17] *= 3                                        # some channels are larger
                c, d = quantise(x)
                to.append(numbers(c, d))
                for i in range(m):
                    j = slice(i * P, min(nk, (i + 1) * P))
                    codes[which][own[i], :, :j.stop - j.start] = c[:, j]
                    scales[which][own[i], :, :j.stop - j.start] = d[:, j]
        self.pages = _cuda(pack(codes[0], scales[0], codes[1], scales[1]))
        self.kv = tc.kv_desc(total, P, Hkv, D)
        self.q = torch.from_numpy(rng.standard_normal((sum(queries), H, D)).astype(np.float32)).cuda().to(types[dtype])
        self.start = np.concatenate([[0], np.cumsum(queries)]).astype(np.int32)

    def run(self, tc, ctx, causal=True, window=0, scale=0.0, lse=True, max_q=None, start=True, q=None, q_strides=(0, 0), o=None, o_strides=(0, 0), stream=None):
        torch, _ = _torch()
        q = self.q if q is None else q
        T = int(self.start[-1])
        o = torch.full_like(self.q, 3.0) if o is None else o
        out = torch.full((T, self.H), 3.0, device="cuda")
        t, l, b = _cuda(self.table), _cuda(np.array(self.keys, np.int32)), _cuda(self.start)
        if stream is not None:
            stream.wait_stream(torch.cuda.current_stream())
        desc = tc.attention_paged_desc(T, len(self.keys), self.table.shape[1], self.H, max_q=max(self.queries) if max_q is None else max_q, dtype=self.dtype,
                                       softmax_scale=scale, causal=causal, window_size=window, q_strides=q_strides, o_strides=o_strides)
        tc.raw_attention_paged(ctx, self.kv, desc, self.pages.data_ptr(), q.data_ptr(), t.data_ptr(), l.data_ptr(), b.data_ptr() if start else 0, o.data_ptr(),
                               out.data_ptr() if lse else 0, (stream or torch.cuda.current_stream()).cuda_stream)
        torch.cuda.synchronize()
        return o, out

    def check(self, o, lse, causal=True, window=0, scale=None, only=None):
        scale = scale or self.D ** -0.5
        o, q = o.float().cpu().numpy().astype(np.float64), self.q.float().cpu().numpy().astype(np.float64)
        off = near = 0.0
        for s in range(len(self.keys)) if only is None else only:
            rows = slice(self.start[s], self.start[s + 1])
            want, want_lse, room, score_off = attention64(q[rows], self.k[s], self.v[s], scale, causal, window)
            got = o[rows]
            assert np.isfinite(got).all()
            assert np.all(abs(got - want) <= room + HALF_ULP[self.dtype] * abs(want) + 2.0 ** -24), (s, self.keys[s], abs(got - want).max())
            off, near = off + np.sum((got - want) ** 2), near + np.sum(want ** 2)
            if lse is not None:
                g = lse.cpu().numpy()[rows]
                none = np.isinf(want_lse)
                assert np.all(g[none] == -np.inf)
                assert np.all(abs(g[~none] - want_lse[~none]) <= score_off[~none] + 2.0 ** -22 * (1 + abs(want_lse[~none])))
        # all together: the result's rounding (2^-11 / sqrt 3, 2^-8 / (2 sqrt 3)) and those of values, weights and scores to 11 bits, with room for half as much again
        assert np.sqrt(off) <= (1.0e-3 if self.dtype == "f16" else 3.0e-3) * np.sqrt(near) + 1e-12


@pytest.mark.parametrize("D,P,H,Hkv,dtype", [(32, 16, 1, 1, "f16"), (64, 16, 8, 2, "f16"), (96, 32, 6, 2, "bf16"), (128, 64, 32, 8, "f16"), (128, 128, 8, 8, "bf16"),
                                             (128, 16, 14, 2, "f16"), (64, 32, 16, 1, "f16"), (128, 64, 20, 1, "bf16"), (32, 64, 12, 4, "f16")])
def test_single_tokens(tc, ctx, D, P, H, Hkv, dtype):
    keys = [1, 0, 2, 15, 16, 17, 31, 33, 63, 64, 65, 128, 200, 511, 1000]
    c = Case(tc, keys, [1] * len(keys), H, Hkv, D, P, dtype, seed=D + H)
    for start in (True, False):
        c.check(*c.run(tc, ctx, start=start))
    assert tc.take_device_error(ctx) == 0


@pytest.mark.parametrize("keys,H,Hkv,D", [([5000], 8, 1, 128), ([20011], 4, 4, 64), ([3, 9000, 0, 40], 16, 2, 128), ([4097] * 3, 2, 1, 96), ([700] * 150, 4, 2, 64)])
def test_long_and_uneven(tc, ctx, keys, H, Hkv, D):
    c = Case(tc, keys, [1] * len(keys), H, Hkv, D, 64, seed=len(keys))
    c.check(*c.run(tc, ctx))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [0, 1, 16, 50])
@pytest.mark.parametrize("queries,H,Hkv,D", [([1, 1, 1, 1, 1], 4, 2, 64), ([3, 5, 0, 2, 8], 4, 2, 64), ([4, 4, 4, 4, 4], 7, 7, 128), ([17, 40, 1, 0, 33], 4, 1, 128),
                                             ([130, 2, 200, 1, 64], 8, 2, 128), ([70, 9, 300, 1, 12], 2, 2, 96), ([257, 1, 100, 3, 0], 4, 1, 64), ([40, 0, 90, 5, 160], 8, 2, 32)])
def test_masks(tc, ctx, queries, H, Hkv, D, causal, window):
    keys = [queries[0] + 77, queries[1] + 1, queries[2] + 130, queries[3], queries[4] + 400]
    c = Case(tc, keys, queries, H, Hkv, D, 32, seed=window + D, dtype="f16" if window else "bf16")
    c.check(*c.run(tc, ctx, causal=causal, window=window), causal=causal, window=window)
    c.check(*c.run(tc, ctx, causal=causal, window=window, max_q=0), causal=causal, window=window)
    assert tc.take_device_error(ctx) == 0


@pytest.mark.parametrize("q", [2, 40, 150])
def test_fewer_keys_than_queries(tc, ctx, q):
    """The first queries lie before the first key: without a key they see, zeros and minus infinity."""
    c = Case(tc, [q // 2, 0, q], [q, q, q], 4, 2, 64, 16, seed=q)
    c.check(*c.run(tc, ctx))


@pytest.mark.parametrize("queries", [[1, 1, 1], [6, 1, 3], [90, 130, 20]])
def test_what_is_not_seen_has_no_part(tc, ctx, queries):
    """NaN and infinite scales behind a sequence's end, in keys ahead of a query and before its window change no bit."""
    keys = [q + 150 for q in queries]
    a, b = (Case(tc, keys, queries, 8, 2, 64, 16, seed=5, spare=s) for s in (0xFF, 0x00))
    for causal, window in ((True, 0), (True, 20)):
        for x, y in zip(a.run(tc, ctx, causal=causal, window=window), b.run(tc, ctx, causal=causal, window=window)):
            assert _torch()[0].equal(x, y)
    # the last key's blocks are NaN: only the last query of each sequence sees it
    nb, tile = 2, a.pages.view(a.kv.n_pages, 2, 1, 1152)
    for s, k in enumerate(keys):
        page, r = int(a.table[s, (k - 1) // 16]), (k - 1) % 16
        at = 544 * nb + ((r // 8 * 4 + r % 8 // 2) * nb) * 4 + r % 2 * 2
        tile[page, :, :, at:at + 2] = 0xFF
        tile[page, :, :, 256 * nb + r * nb * 2:256 * nb + r * nb * 2 + 2] = 0xFF
    o, lse = a.run(tc, ctx)
    last = [int(v) - 1 for v in a.start[1:]]
    bad = _torch()[0].zeros(len(o), dtype=bool)
    bad[last] = True
    assert o[bad].isnan().any(dim=2).all() and o[~bad].isfinite().all() and lse[~bad].isfinite().all()
    assert _torch()[0].equal(o[~bad], b.run(tc, ctx)[0][~bad])


@pytest.mark.parametrize("queries", [[1, 1, 1], [5, 2, 1], [64, 80, 150]])
def test_large_and_small_values(tc, ctx, queries):
    """Values and keys far from one, scores far apart: nothing over- or underflows on the way."""
    keys = [q + 100 for q in queries]
    for size, scale in ((300.0, 1e-4), (1e-3, 10.0), (2000.0, 1e-6)):
        c = Case(tc, keys, queries, 8, 2, 128, 32, seed=11, size=size)
        c.check(*c.run(tc, ctx, scale=scale), scale=scale)
    # scores hundreds apart: one key has all the weight
    c = Case(tc, keys, queries, 8, 2, 128, 32, seed=12, size=20.0)
    o, lse = c.run(tc, ctx, scale=1.0)
    assert o.isfinite().all() and lse.isfinite().all()


@pytest.mark.parametrize("queries", [[1] * 6, [3] * 6, [50] * 6])
def test_strides_and_streams(tc, ctx, queries):
    torch, _ = _torch()
    c = Case(tc, [q + 60 for q in queries], queries, 8, 2, 64, 16, seed=2)
    want, lse = c.run(tc, ctx)
    T, H, D = c.q.shape
    stream = torch.cuda.Stream()
    wide = torch.zeros(T, 2 * H * D, dtype=torch.float16, device="cuda")
    wide[:, :H * D] = c.q.view(T, -1)
    out = torch.zeros(H, T, D, dtype=torch.float16, device="cuda")
    c.run(tc, ctx, q=wide, q_strides=(2 * H * D, D), o=out, o_strides=(D, T * D), stream=stream)
    assert torch.equal(out.transpose(0, 1), want)
    odd_q, odd_o = (torch.zeros(T * H * D + 1, dtype=torch.float16, device="cuda")[1:] for _ in range(2))
    odd_q.copy_(c.q.view(-1))
    c.run(tc, ctx, q=odd_q, o=odd_o, stream=stream)
    assert torch.equal(odd_o.view(T, H, D), want)


@pytest.mark.parametrize("queries", [[1] * 4, [2, 7, 1, 4], [100, 1, 60, 8]])
def test_repeats_bit_for_bit(tc, ctx, queries):
    """The order of sums does not depend on the run."""
    c = Case(tc, [q + 900 for q in queries], queries, 8, 2, 128, 64, seed=3)
    first = c.run(tc, ctx)
    for _ in range(5):
        for x, y in zip(first, c.run(tc, ctx)):
            assert _torch()[0].equal(x, y)


@pytest.mark.parametrize("queries", [[1] * 5, [4] * 5, [80] * 5])
def test_captured_in_a_graph(tc, ctx, queries):
    """Replays with other lengths and pages, beside calls on another stream."""
    torch, _ = _torch()
    c = Case(tc, [q + 300 for q in queries], queries, 8, 2, 128, 16, seed=4)
    want = c.run(tc, ctx)
    shorter = [k - 40 for k in c.keys]
    t, b = _cuda(c.table), _cuda(c.start)
    lens = _cuda(np.array(c.keys, np.int32))
    o, lse = torch.zeros_like(c.q), torch.zeros(len(c.q), 8, device="cuda")
    desc = tc.attention_paged_desc(len(c.q), 5, c.table.shape[1], 8, max_q=max(queries))

    def call(stream):
        tc.raw_attention_paged(ctx, c.kv, desc, c.pages.data_ptr(), c.q.data_ptr(), t.data_ptr(), lens.data_ptr(), b.data_ptr(), o.data_ptr(), lse.data_ptr(),
                               stream.cuda_stream)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    call(side)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        call(side)
    for keys in (c.keys, shorter, c.keys):
        lens.copy_(_cuda(np.array(keys, np.int32)))
        o.zero_()
        torch.cuda.synchronize()
        g.replay()
        beside = c.run(tc, ctx, stream=torch.cuda.Stream())
        assert torch.equal(beside[0], want[0])
        if keys is c.keys:
            assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
        else:
            assert not torch.equal(o, want[0])
    del g


def test_on_buffers(tc, ctx):
    c = Case(tc, [50, 7, 90], [1, 2, 1], 4, 2, 64, 16, seed=6)
    want, lse = c.run(tc, ctx)
    q, pages = ctx.buffer_from_array(c.q.cpu().numpy()), ctx.buffer_from_array(c.pages.cpu().numpy())
    t, l, b = (ctx.buffer_from_array(np.array(a, np.int32)) for a in (c.table, c.keys, c.start))
    o, s = ctx.buffer(c.q.numel() * 2), ctx.buffer(len(c.q) * 4 * 4)
    before = tc.launch_count()
    tc.attention_paged(ctx, c.kv, tc.attention_paged_desc(4, 3, c.table.shape[1], 4, max_q=2), pages, q, t, l, b, o, s)
    assert tc.launch_count() > before and "attention_paged" in tc.cuda_last_kernel_name() and tc.last_backend() == tc.TC_BACKEND_CUDA
    assert np.array_equal(o.to_numpy(c.q.shape, np.float16), want.cpu().numpy()) and np.array_equal(s.to_numpy((4, 4), np.float32), lse.cpu().numpy())


@pytest.mark.parametrize("queries", [[1, 1, 1], [60, 1, 70]])
def test_pages_and_lengths_that_do_not_exist(tc, ctx, queries):
    """A length past the table is cut to it, a page that is not there is passed over; the error word is set, the other sequences are right."""
    c = Case(tc, [queries[0] + 40, queries[1] + 30, queries[2] + 20], queries, 4, 2, 64, 16, seed=7)
    for table, keys in (((1, 0, c.kv.n_pages), None), ((1, 1, -1), None), (None, (1, 16 * c.table.shape[1] + 1)), (None, (1, 2 ** 31 - 1))):
        d = Case(tc, list(c.keys), queries, 4, 2, 64, 16, seed=7)
        if table:
            d.table[table[0], table[1]] = table[2]
        if keys:
            d.table[1, :] = 0
            d.keys[keys[0]] = keys[1]
        result = d.run(tc, ctx)
        assert tc.take_device_error(ctx) == 2
        c.check(*result, only=(0, 2))      # (not bit for bit: where a row's keys are cut depends on all lengths)
    d = Case(tc, list(c.keys), queries, 4, 2, 64, 16, seed=7)
    d.keys[1] = -5
    assert not d.run(tc, ctx)[0][d.start[1]:d.start[2]].any() and tc.take_device_error(ctx) == 0


def test_refusals(tc, ctx):
    L, b = tc.lib(), ctx.buffer(1 << 16)
    h, kv, ok = b.handle, tc.kv_desc(4, 16, 2, 64), dict(tokens=4, n_seqs=4, max_pages=1, q_heads=4)

    def status(kv=kv, q=h, o=h, start=h, **kw):
        return L.tcx_attention_paged(ctx.handle, ctypes.byref(kv), ctypes.byref(tc.attention_paged_desc(**{**ok, **kw})), h, q, h, h, start, o, None)
    assert L.tcx_attention_paged(None, *[None] * 9) == tc.TC_ERR_NOT_INITIALIZED
    for bad in (dict(q=None), dict(o=None), dict(tokens=0), dict(n_seqs=0), dict(max_pages=0), dict(q_heads=0), dict(q_heads=3), dict(max_q=-1), dict(window_size=-1),
                dict(tokens=5, start=None), dict(q_strides=(-1, 0)), dict(o_strides=(64, 0)), dict(kv=tc.kv_desc(4, 16, -2, 64))):
        assert status(**bad) == tc.TC_ERR_INVALID_ARG, bad
    for bad in (dict(tokens=1 << 12, n_seqs=1 << 12), dict(max_pages=1 << 28), dict(max_pages=1 << 14), dict(kv=tc.kv_desc(4, 16, 2, 256)), dict(kv=tc.kv_desc(4, 12, 2, 64)),
                dict(tokens=1 << 30)):
        assert status(**bad) == tc.TC_ERR_INVALID_SHAPE, bad
    assert status(dtype="f32") == tc.TC_ERR_UNSUPPORTED_DTYPE
    p, d = b.device_ptr(), tc.attention_paged_desc(**ok)
    for at, off in ((0, 8), (1, 1), (2, 2), (3, 1), (5, 1), (6, 2)):
        args = [p, p, p, p, None, p, None]
        args[at] = (args[at] or p) + off
        assert L.tcx_raw_attention_paged(ctx.handle, ctypes.byref(kv), ctypes.byref(d), *args, None) == tc.TC_ERR_INVALID_ARG


@pytest.mark.parametrize("n,q", [(257, 1), (600, 1), (300, 3)])
def test_more_sequences_than_a_launch_takes(tc, ctx, n, q):
    rng = np.random.default_rng(n)
    c = Case(tc, [int(k) for k in rng.integers(0, 90, n)], [q] * n, 4, 2, 64, 16, seed=n)
    c.check(*c.run(tc, ctx))
    assert tc.take_device_error(ctx) == 0


@pytest.mark.parametrize("keys,queries,H,Hkv,D,window", [([5000], [130], 2, 1, 128, 0), ([6001], [70], 4, 1, 64, 0), ([4100, 9, 3000], [40, 9, 1], 4, 2, 96, 0),
                                                         ([7000], [257], 1, 1, 32, 3000)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_prompts_whose_keys_are_cut_into_chunks(tc, ctx, keys, queries, H, Hkv, D, window, dtype):
    """Few rows over many keys, beside a sequence of one token; twice, for the pieces' room is used again."""
    c = Case(tc, keys, queries, H, Hkv, D, 64, dtype, seed=len(keys) + D)
    for _ in range(2):
        c.check(*c.run(tc, ctx, window=window), window=window)


@pytest.mark.parametrize("queries", [[1, 1, 1], [2, 5, 1], [130, 1, 40]])
def test_without_room_to_hand_sums_over(tc, ctx, queries):
    """While the context has an error pending no room is handed out: whole items to a CTA, prompts' keys in one piece."""
    c = Case(tc, [k + 2500 for k in queries], queries, 8, 2, 64, 16, seed=9)
    tc.set_device_error(ctx, 1)
    try:
        got = c.run(tc, ctx)
    finally:
        assert tc.take_device_error(ctx) == 1
    c.check(*got)


@pytest.mark.parametrize("queries", [[1, 1], [60, 1]])
def test_pages_behind_four_gigabytes(tc, ctx, queries):
    torch, _ = _torch()
    c = Case(tc, [300, 77], queries, 8, 8, 128, 64, seed=2)
    far = (5 << 30) // tc.kv_page_bytes(c.kv)
    pages = torch.empty((far * tc.kv_page_bytes(c.kv) + c.pages.nbytes,), dtype=torch.uint8, device="cuda")
    pages[far * tc.kv_page_bytes(c.kv):] = c.pages.view(torch.uint8).reshape(-1)
    c.table = np.where(c.table < 1 << 20, c.table + far, 1 << 20).astype(np.int32)
    c.kv.n_pages += far
    c.pages = pages
    c.check(*c.run(tc, ctx))


def test_small_launches_between_others(tc, ctx):
    """Calls that follow one another on a stream, each reading what the one before wrote: rows turned, appended, attended to, and the
    result turned back, as many times over without a wait on the host."""
    torch, _ = _torch()
    rng = np.random.default_rng(4)
    T, H, Hkv, D, P, steps = 3, 8, 2, 64, 16, 40
    kv, per = tc.kv_desc(T * 4, P, Hkv, D), 4
    table = _cuda(np.arange(T * per, dtype=np.int32).reshape(T, per))
    angles = np.arange(steps)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)
    cos, sin = _cuda(np.cos(angles).astype(np.float32)), _cuda(np.sin(angles).astype(np.float32))
    x = torch.from_numpy(rng.standard_normal((steps, T, H + 2 * Hkv, D)).astype(np.float32)).cuda().half()
    seq, places = _cuda(np.arange(T, dtype=np.int32)), _cuda(np.repeat(np.arange(steps, dtype=np.int32)[:, None], T, axis=1))
    lens = places + 1
    app = tc.kv_append_desc(T, T, per, q_heads=H, rot_dim=D, dtype="f16", table_rows=steps, k_strides=x.stride()[1:3], v_strides=x.stride()[1:3], q_strides=x.stride()[1:3])
    att, back = tc.attention_paged_desc(T, T, per, H, max_q=1, dtype="f16"), tc.rope_desc(T, H, D, dtype="f16", table_rows=steps, inverse=True)

    def go(wait):
        pages, q, o = torch.zeros(T * per * tc.kv_page_bytes(kv), dtype=torch.uint8, device="cuda"), torch.zeros(T, H, D, device="cuda").half(), torch.zeros(T, H, D, device="cuda").half()
        outs, st = torch.zeros(steps, T, H, D, device="cuda").half(), torch.cuda.current_stream().cuda_stream
        torch.cuda.synchronize()
        for i in range(steps):
            r, at = x[i], (places[i].data_ptr(), seq.data_ptr(), table.data_ptr())
            tc.raw_kv_append(ctx, kv, app, pages.data_ptr(), r[:, H:].data_ptr(), r[:, H + Hkv:].data_ptr(), r.data_ptr(), q.data_ptr(), cos.data_ptr(), sin.data_ptr(), *at, st)
            if wait:
                torch.cuda.synchronize()
            tc.raw_attention_paged(ctx, kv, att, pages.data_ptr(), q.data_ptr(), table.data_ptr(), lens[i].data_ptr(), 0, o.data_ptr(), 0, st)
            if wait:
                torch.cuda.synchronize()
            tc.raw_rope(ctx, back, o.data_ptr(), outs[i].data_ptr(), cos.data_ptr(), sin.data_ptr(), places[i].data_ptr(), st)
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return outs
    assert torch.equal(go(False), go(True))
    assert tc.take_device_error(ctx) == 0


@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 60), (False, 33)])
@pytest.mark.parametrize("G,Hkv,D,dtype", [(4, 8, 128, "f16"), (4, 8, 128, "bf16"), (3, 8, 64, "f16"), (5, 8, 96, "bf16"), (4, 8, 32, "f16")])
def test_prompts_enough_for_all_processors(tc, ctx, G, Hkv, D, dtype, causal, window):
    """Rows enough for tiles of twice the height: tiles that are full, half full, one row more than half, and sequences of few rows beside them."""
    queries = [64, 32, 33, 65, 96, 1, 100, 0, 128, 40, 64, 75, 90, 3, 64, 64, 70, 80, 31]
    keys = [q + extra for q, extra in zip(queries, (0, 200, 1, 300, 0, 77, 130, 5, 0, 400, 17, 0, 64, 1, 128, 127, 129, 31, 250))]
    c = Case(tc, keys, queries, G * Hkv, Hkv, D, 16, dtype, seed=D + G)
    c.check(*c.run(tc, ctx, causal=causal, window=window), causal=causal, window=window)
    assert tc.take_device_error(ctx) == 0


def test_many_prompts_and_what_they_do_not_see(tc, ctx):
    queries = [64] * 17 + [33, 1]
    keys = [q + 90 for q in queries]
    a, b = (Case(tc, keys, queries, 32, 8, 64, 16, seed=5, spare=s) for s in (0xFF, 0x00))
    for window in (0, 20):
        for x, y in zip(a.run(tc, ctx, window=window), b.run(tc, ctx, window=window)):
            assert _torch()[0].equal(x, y)
    first, second = (a.run(tc, ctx) for _ in range(2))
    assert all(_torch()[0].equal(x, y) for x, y in zip(first, second))
    for s, k in enumerate(keys):                                              # the last key's values are NaN: only the last query sees it
        tile = a.pages.view(a.kv.n_pages, 8, 1, 1152)
        page, r = int(a.table[s, (k - 1) // 16]), (k - 1) % 16
        at = 544 * 2 + ((r // 8 * 4 + r % 8 // 2) * 2) * 4 + r % 2 * 2
        tile[page, :, :, at:at + 2] = 0xFF
    o, lse = a.run(tc, ctx)
    last = np.zeros(sum(queries), bool)
    last[a.start[1:] - 1] = True
    torch = _torch()[0]
    assert torch.isnan(o[torch.from_numpy(last)][:, :, :32]).all() and torch.isfinite(o[torch.from_numpy(last)][:, :, 32:]).all()
    assert torch.equal(o[torch.from_numpy(~last)], first[0][torch.from_numpy(~last)]) and torch.equal(lse, first[1])
