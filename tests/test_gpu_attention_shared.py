"""Attention for sequences with the same first keys, and over lists of pages by K/V head, against 64 bits."""
import ctypes

import numpy as np
import pytest

from paged_reference import attention64, numbers, pack, quantise

pytestmark = pytest.mark.gpu
HALF_ULP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _torch():
    import torch
    return torch, {"f16": torch.float16, "bf16": torch.bfloat16}


def _cuda(a, dtype=np.int32):
    return _torch()[0].from_numpy(np.ascontiguousarray(np.asarray(a, dtype))).cuda()


class Family:
    """groups: (shared keys, [(own keys, queries) of each sequence]).  Whole pages of shared keys are the group's; what is left of them each sequence
    has on its own next page.  spare: the byte of everything that is no sequence's (0xFF: NaN scales)."""

    def __init__(self, tc, groups, H, Hkv, D, P, dtype="f16", seed=0, size=1.0, spare=0xFF):
        torch, types = _torch()
        rng = np.random.default_rng(seed)
        self.H, self.Hkv, self.D, self.P, self.dtype = H, Hkv, D, P, dtype
        self.shared, self.group_start, self.keys, self.queries, self.k, self.v = [], [0], [], [], [], []
        lists, content, free = [], {}, 0

        def rows(n, which):
            x = (rng.standard_normal((Hkv, n, D)) * size).astype(np.float32)
            if which == 0:
                x[:, :, ::17] *= 3
            return quantise(x)
        for n, members in groups:
            common = [rows(n, w) for w in (0, 1)]
            self.shared.append(n)
            whole = list(range(free, free + n // P))
            free += n // P
            for own, nq in members:
                kv = []
                for w in (0, 1):
                    c, d = rows(own, w)
                    kv.append((np.concatenate([common[w][0], c], axis=1), np.concatenate([common[w][1], d], axis=1)))
                m = -(-(n + own) // P)
                mine = whole + list(range(free, free + m - n // P))
                free += m - n // P
                for i, page in enumerate(mine):
                    content[page] = [(x[:, i * P:(i + 1) * P], d[:, i * P:(i + 1) * P]) for x, d in kv]
                lists.append(mine)
                self.keys.append(n + own)
                self.queries.append(nq)
                self.k.append(numbers(*kv[0]))
                self.v.append(numbers(*kv[1]))
            self.group_start.append(len(lists))
        total = free + 2
        order = rng.permutation(total)
        self.table = np.full((len(lists), max(1, max(map(len, lists)))), 1 << 20, np.int32)
        for s, mine in enumerate(lists):
            self.table[s, :len(mine)] = order[mine]
        codes = [np.full((total, Hkv, P, D), spare & 15, np.uint8) for _ in range(2)]
        scales = [np.full((total, Hkv, P, D // 32), np.array([spare * 257], np.uint16).view(np.float16)[0], np.float16) for _ in range(2)]
        for page, kv in content.items():
            for w, (c, d) in enumerate(kv):
                codes[w][order[page], :, :c.shape[1]] = c
                scales[w][order[page], :, :c.shape[1]] = d
        self.pages = torch.from_numpy(pack(codes[0], scales[0], codes[1], scales[1])).cuda()
        self.kv = tc.kv_desc(total, P, Hkv, D)
        self.q = torch.from_numpy(rng.standard_normal((sum(self.queries), H, D)).astype(np.float32)).cuda().to(types[dtype])
        self.start = np.concatenate([[0], np.cumsum(self.queries)]).astype(np.int32)

    def most(self):
        return max(int(self.start[b] - self.start[a]) for a, b in zip(self.group_start, self.group_start[1:]))

    def run(self, tc, ctx, causal=True, scale=0.0, max_q=None, max_group_q=None, start=True, q=None, q_strides=(0, 0), o=None, o_strides=(0, 0), stream=None, shared=None,
            group_start=None, lse=True, always=True):
        torch, _ = _torch()
        q = self.q if q is None else q
        T = len(self.q)
        o = torch.full_like(self.q, 3.0) if o is None else o
        out = torch.full((T, self.H), 3.0, device="cuda")
        group_start, shared = self.group_start if group_start is None else group_start, self.shared if shared is None else shared
        ints = [_cuda(a) for a in (self.table, self.keys, self.start, group_start, shared)]
        desc = tc.attention_shared_desc(T, len(self.keys), self.table.shape[1], self.H, len(shared), max_q=max(self.queries) if max_q is None else max_q,
                                        max_group_q=self.most() if max_group_q is None else max_group_q, dtype=self.dtype, softmax_scale=scale, causal=causal,
                                        q_strides=q_strides, o_strides=o_strides, always=always)
        torch.cuda.synchronize()
        t, l, b, g, n = (x.data_ptr() for x in ints)
        tc.raw_attention_shared(ctx, self.kv, desc, self.pages.data_ptr(), q.data_ptr(), t, l, b if start else 0, g, n, o.data_ptr(), out.data_ptr() if lse else 0,
                                (stream or torch.cuda.current_stream()).cuda_stream)
        torch.cuda.synchronize()
        return o, out

    def check(self, o, lse, causal=True, scale=None, only=None):
        scale = scale or self.D ** -0.5
        o, q = o.float().cpu().numpy().astype(np.float64), self.q.float().cpu().numpy().astype(np.float64)
        off = near = 0.0
        for s in range(len(self.keys)) if only is None else only:
            rows = slice(self.start[s], self.start[s + 1])
            # (what two sums joined in fp32 add, a few 2^-24, is far below the 2^-11 of a value that `room` has)
            want, want_lse, room, score_off = attention64(q[rows], self.k[s], self.v[s], scale, causal, 0)
            got = o[rows]
            assert np.isfinite(got).all(), s
            assert np.all(abs(got - want) <= room + HALF_ULP[self.dtype] * abs(want) + 2.0 ** -24), (s, self.keys[s], abs(got - want).max())
            off, near = off + np.sum((got - want) ** 2), near + np.sum(want ** 2)
            if lse is not None:
                g = lse.cpu().numpy()[rows]
                none = np.isinf(want_lse)
                assert np.all(g[none] == -np.inf)
                assert np.all(abs(g[~none] - want_lse[~none]) <= score_off[~none] + 2.0 ** -22 * (1 + abs(want_lse[~none])))
        # all together, as for attention over pages: the result's rounding and those of values, weights and scores to 11 bits
        assert np.sqrt(off) <= (1.0e-3 if self.dtype == "f16" else 3.0e-3) * np.sqrt(near) + 1e-12


@pytest.mark.parametrize("D,P,H,Hkv,dtype", [(32, 16, 1, 1, "f16"), (64, 16, 8, 2, "f16"), (96, 32, 6, 2, "bf16"), (128, 64, 32, 8, "f16"), (128, 128, 8, 8, "bf16"),
                                             (128, 16, 14, 2, "f16"), (64, 32, 16, 1, "f16"), (128, 64, 20, 1, "bf16"), (32, 64, 12, 4, "f16")])
@pytest.mark.parametrize("members", [2, 5, 33, 130])
def test_single_tokens(tc, ctx, D, P, H, Hkv, dtype, members):
    own = [1, 2, 15, 16, 17, 63, 64, 65, 130, 400]
    for n in (1, 16, 63, 200, 1111):
        c = Family(tc, [(n, [(own[i % len(own)], 1) for i in range(members)])], H, Hkv, D, P, dtype, seed=D + n)
        for start in (True, False):
            c.check(*c.run(tc, ctx, start=start))
        c.check(*c.run(tc, ctx, always=False))
    assert tc.take_device_error(ctx) == 0


GROUPS = [(300, [(20, 1), (1, 1), (130, 1)]), (0, [(50, 1)]), (77, [(9, 1)]), (500, [(10, 2), (40, 1), (8, 0), (90, 8)]), (64, [(30, 30), (1, 1)]), (129, [(200, 3)] * 20)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,Hkv,D,dtype", [(4, 2, 64, "f16"), (7, 7, 128, "bf16"), (8, 2, 128, "f16"), (4, 4, 96, "bf16"), (8, 1, 32, "f16")])
def test_groups_of_all_kinds(tc, ctx, H, Hkv, D, dtype, causal):
    """Groups of few rows and of many beside one another, of one sequence, without shared keys, with an idle slot; prompts beside single tokens."""
    c = Family(tc, GROUPS, H, Hkv, D, 32, dtype, seed=D)
    c.check(*c.run(tc, ctx, causal=causal), causal=causal)
    c.check(*c.run(tc, ctx, causal=causal, max_q=0, max_group_q=0), causal=causal)
    c.check(*c.run(tc, ctx, causal=causal, always=False), causal=causal)
    assert tc.take_device_error(ctx) == 0


@pytest.mark.parametrize("q,members", [(1, 6), (4, 6), (40, 6), (1, 40), (2, 33)])
def test_long_shared_keys(tc, ctx, q, members):
    c = Family(tc, [(9001, [(q + 3 * i, q) for i in range(members)])], 8, 2, 128, 64, seed=q)
    c.check(*c.run(tc, ctx))
    c.check(*c.run(tc, ctx, always=False))


@pytest.mark.parametrize("q", [1, 40, 150])
def test_shares_as_much_as_it_can(tc, ctx, q):
    """Shared lengths past a sequence's first query, below zero or of all keys count down to what is there before the first query; less may be named, too."""
    c = Family(tc, [(200, [(q, q), (q + 5, q)]), (90, [(q + 70, q), (q + 1, q)])], 4, 2, 64, 16, seed=q)
    for shared in ([200, 90], [200 + q, 91 + q], [2 ** 31 - 1, 2 ** 31 - 1], [7, 33], [0, -5]):
        if max(shared) > 1000 or shared[1] == 91 + q:
            # (the first keys of the second group's sequences are alike up to 90: so are its members' pages only as long)
            shared = [shared[0], 90]
        c.check(*c.run(tc, ctx, shared=shared))
    assert tc.take_device_error(ctx) == 0


@pytest.mark.parametrize("queries", [1, 3, 60])
def test_groups_that_leave_sequences_out(tc, ctx, queries):
    c = Family(tc, [(100, [(q, queries) for q in (70, 80, 90)]), (100, [(q, queries) for q in (65, 61)])], 4, 2, 64, 16, seed=8)
    for start, shared in (([0, 3, 5], [100, 100]), ([1, 3, 5], [100, 100]), ([0, 2, 2], [100, 100]), ([3, 5], [100]), ([0, 0, 0, 0, 5][:3], [100, 3]), ([5, 5], [100])):
        c.check(*c.run(tc, ctx, group_start=start, shared=shared))
    assert tc.take_device_error(ctx) == 0
    for start in ([-1, 3, 5], [0, 3, 6], [3, 1, 5]):                       # they do not rise within the sequences: told, and nothing out of place is touched
        o, _ = c.run(tc, ctx, group_start=start, shared=[16, 16])
        assert tc.take_device_error(ctx) == 2 and o.isfinite().all()


def test_more_queries_than_declared(tc, ctx):
    """A group with more queries than the call says shares nothing."""
    c = Family(tc, [(300, [(20, 1)] * 40), (200, [(5, 1)] * 3)], 4, 2, 64, 16, seed=1)
    for most in (1, 3, 39, 40):
        c.check(*c.run(tc, ctx, max_group_q=most))
    assert tc.take_device_error(ctx) == 0


@pytest.mark.parametrize("queries,max_q", [([300, 20, 260], 40), ([20, 700], 100), ([1] * 30 + [60], 1), ([100] * 4 + [140], 100)])
def test_more_queries_of_a_sequence_than_declared(tc, ctx, queries, max_q):
    """Either every row is right, or the error word says that rows may be missing."""
    c = Family(tc, [(200, [(q + 9, q) for q in queries]), (90, [(40, 1), (7, 1)])], 8, 2, 128, 64, seed=3)
    got = c.run(tc, ctx, max_q=max_q)
    if tc.take_device_error(ctx) == 0:
        c.check(*got)
    else:
        assert got[0].isfinite().all()
    c.check(*c.run(tc, ctx))
    assert tc.take_device_error(ctx) == 0


@pytest.mark.parametrize("q", [1, 50])
def test_rows_behind_the_last_sequence(tc, ctx, q):
    torch, _ = _torch()
    c = Family(tc, [(300, [(q + 9, q)] * 3), (0, [(1, 1)])], 4, 2, 64, 16, seed=q)
    rows = int(c.start[3])
    want, want_lse = c.run(tc, ctx)
    c.start[4] = rows                                                     # the last sequence has no queries any more: its row is behind
    o, lse = c.run(tc, ctx)
    assert (o[rows:] == 3).all() and (lse[rows:] == 3).all()
    c.check(o, lse, only=range(3))


@pytest.mark.parametrize("q", [1, 5, 60])
def test_what_is_not_seen_has_no_part(tc, ctx, q):
    """NaN and infinite scales behind sequences' ends and in pages of nobody change no bit; NaN in a shared key shows in every row of its group alone."""
    torch, _ = _torch()
    groups = [(150, [(q + 9, q), (q, q), (q + 40, q)]), (90, [(q + 3, q), (q + 30, q)])]
    a, b = (Family(tc, groups, 8, 2, 64, 16, seed=5, spare=s) for s in (0xFF, 0x00))
    want = a.run(tc, ctx)
    for x, y in zip(want, b.run(tc, ctx)):
        assert torch.equal(x, y)
    tile = a.pages.view(a.kv.n_pages, 2, 1, 1152)
    tile[int(a.table[0, 3]), :, :, 256 * 2 + 5 * 4:256 * 2 + 5 * 4 + 2] = 0xFF      # the scale of key 53, block 0
    o, lse = a.run(tc, ctx)
    rows = int(a.start[3])
    assert o[:rows].isnan().all() and lse[:rows].isnan().all()
    a.check(o, lse, only=(3, 4))
    # a value alone: its block, not the others
    b.pages.view(b.kv.n_pages, 2, 1, 1152)[int(b.table[0, 3]), :, :, 544 * 2:544 * 2 + 2] = 0xFF
    o, lse = b.run(tc, ctx)
    assert o[:rows, :, :32].isnan().all() and o[:rows, :, 32:].isfinite().all() and lse.isfinite().all() and o[rows:].isfinite().all()


@pytest.mark.parametrize("q", [1, 4, 70])
def test_large_and_small_values(tc, ctx, q):
    groups = [(200, [(q + 100, q), (q + 9, q)]), (33, [(q, q)] * 3)]
    for size, scale in ((300.0, 1e-4), (1e-3, 10.0), (2000.0, 1e-6)):
        c = Family(tc, groups, 8, 2, 128, 32, seed=11, size=size)
        c.check(*c.run(tc, ctx, scale=scale), scale=scale)
    c = Family(tc, groups, 8, 2, 128, 32, seed=12, size=20.0)
    o, lse = c.run(tc, ctx, scale=1.0)
    assert o.isfinite().all() and lse.isfinite().all()


@pytest.mark.parametrize("q", [1, 3, 50])
def test_strides_streams_and_repeats(tc, ctx, q):
    torch, _ = _torch()
    c = Family(tc, [(500, [(q + 60, q)] * 5), (40, [(q + 7, q)] * 2)], 8, 2, 64, 16, seed=2)
    want, want_lse = c.run(tc, ctx)
    for _ in range(4):
        o, lse = c.run(tc, ctx)
        assert torch.equal(o, want) and torch.equal(lse, want_lse)
    T, H, D = c.q.shape
    stream = torch.cuda.Stream()
    wide = torch.zeros(T, 2 * H * D, dtype=torch.float16, device="cuda")
    wide[:, :H * D] = c.q.view(T, -1)
    out = torch.zeros(H, T, D, dtype=torch.float16, device="cuda")
    c.run(tc, ctx, q=wide, q_strides=(2 * H * D, D), o=out, o_strides=(D, T * D), stream=stream, lse=False)
    assert torch.equal(out.transpose(0, 1), want)
    odd_q, odd_o = (torch.zeros(T * H * D + 1, dtype=torch.float16, device="cuda")[1:] for _ in range(2))
    odd_q.copy_(c.q.view(-1))
    c.run(tc, ctx, q=odd_q, o=odd_o, stream=stream)
    assert torch.equal(odd_o.view(T, H, D), want)


@pytest.mark.parametrize("q", [1, 4, 60])
def test_captured_in_a_graph(tc, ctx, q):
    """Replayed with other shared lengths and groups, beside calls on another stream and another graph of the same call."""
    torch, _ = _torch()
    c = Family(tc, [(700, [(q + 30, q)] * 6), (100, [(q + 1, q)] * 3)], 8, 2, 128, 16, seed=4)
    want = c.run(tc, ctx)
    ints = [_cuda(a) for a in (c.table, c.keys, c.start, c.group_start, c.shared)]
    desc = tc.attention_shared_desc(len(c.q), 9, c.table.shape[1], 8, 2, max_q=q, max_group_q=c.most(), always=True)
    outs = [(torch.zeros_like(c.q), torch.zeros(len(c.q), 8, device="cuda")) for _ in range(2)]

    def call(stream, o, lse):
        tc.raw_attention_shared(ctx, c.kv, desc, c.pages.data_ptr(), c.q.data_ptr(), *(x.data_ptr() for x in ints), o.data_ptr(), lse.data_ptr(), stream.cuda_stream)
    streams, graphs = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for stream, out in zip(streams, outs):
        call(stream, *out)
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            call(stream, *out)
        graphs.append(g)
    for shared in (c.shared, [0, 100], [650, 17], c.shared):
        ints[4].copy_(_cuda(shared))
        for o, lse in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
        beside = c.run(tc, ctx, stream=torch.cuda.Stream())
        assert torch.equal(beside[0], want[0])
        for o, lse in outs:
            c.check(o, lse)
            if shared is c.shared:
                assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    del graphs
    assert tc.take_device_error(ctx) == 0


@pytest.mark.parametrize("more", [0, 30])
def test_on_buffers(tc, ctx, more):
    c = Family(tc, [(90, [(5, 1), (9, 2)] + [(3, 1)] * more), (30, [(7, 1)])], 4, 2, 64, 16, seed=6)
    want, lse = c.run(tc, ctx)
    q, pages = ctx.buffer_from_array(c.q.cpu().numpy()), ctx.buffer_from_array(c.pages.cpu().numpy())
    ints = [ctx.buffer_from_array(np.array(a, np.int32)) for a in (c.table, c.keys, c.start, c.group_start, c.shared)]
    T = 4 + more
    o, s = ctx.buffer(c.q.numel() * 2), ctx.buffer(T * 4 * 4)
    before = tc.launch_count()
    tc.attention_shared(ctx, c.kv, tc.attention_shared_desc(T, 3 + more, c.table.shape[1], 4, 2, max_q=2, max_group_q=3 + more, always=True), pages, q, *ints, o, s)
    assert tc.launch_count() > before and "attention_shared" in tc.cuda_last_kernel_name() and tc.last_backend() == tc.TC_BACKEND_CUDA
    assert np.array_equal(o.to_numpy(c.q.shape, np.float16), want.cpu().numpy()) and np.array_equal(s.to_numpy((T, 4), np.float32), lse.cpu().numpy())


@pytest.mark.parametrize("q", [1, 50])
def test_pages_and_lengths_that_do_not_exist(tc, ctx, q):
    for table, keys in (((4, 0, 1 << 20), None), ((4, 1, -1), None), ((4, 3, -1), None), ((4, 3, 1 << 20), None), (None, (4, 16 * 100)), (None, (4, 2 ** 31 - 1))):
        c = Family(tc, [(100, [(q + 30, q)] * 3), (60, [(q + 7, q)] * 2)], 4, 2, 64, 16, seed=7)
        if table:
            c.table[table[0], table[1]] = table[2]
        if keys:
            c.table[4, :] = 0
            c.keys[keys[0]] = keys[1]
        o, lse = c.run(tc, ctx)
        told = tc.take_device_error(ctx)
        assert told == 2 or (told == 0 and table and 16 * table[1] < 48)      # (a page that has shared keys alone need not be looked for in this row)
        c.check(o, lse, only=range(3))
    c = Family(tc, [(100, [(q + 30, q)] * 3)], 4, 2, 64, 16, seed=7)
    c.keys[1] = -5                                                        # none of them shares anything then, and sequence 1 has no keys
    o, lse = c.run(tc, ctx)
    assert not o[c.start[1]:c.start[2]].any() and tc.take_device_error(ctx) == 0
    c.check(o, lse, only=(0, 2))


@pytest.mark.parametrize("q", [1, 4, 40])
def test_without_room(tc, ctx, q):
    """While the context has an error pending no room is handed out: every sequence reads its keys itself."""
    c = Family(tc, [(700, [(q + 30, q)] * 4)], 8, 2, 64, 16, seed=9)
    tc.set_device_error(ctx, 1)
    try:
        got = c.run(tc, ctx)
    finally:
        assert tc.take_device_error(ctx) == 1
    c.check(*got)


@pytest.mark.parametrize("n,q", [(257, 1), (600, 2)])
def test_more_sequences_than_a_launch_takes(tc, ctx, n, q):
    rng = np.random.default_rng(n)
    c = Family(tc, [(int(rng.integers(0, 120)), [(int(rng.integers(q, 40)), q) for _ in range(n // 4)]) for _ in range(5)], 4, 2, 64, 16, seed=n)
    c.check(*c.run(tc, ctx))
    many = Family(tc, [(20, [(3, 1), (9, 1)])] * (n // 2), 2, 1, 32, 16, seed=n)
    many.check(*many.run(tc, ctx))
    assert tc.take_device_error(ctx) == 0


def test_one_sequence(tc, ctx):
    c = Family(tc, [(90, [(5, 1)])], 4, 2, 64, 16, seed=6)
    c.check(*c.run(tc, ctx))


def test_refusals(tc, ctx):
    L, b = tc.lib(), ctx.buffer(1 << 16)
    h, kv, ok = b.handle, tc.kv_desc(4, 16, 2, 64), dict(tokens=4, n_seqs=4, max_pages=1, q_heads=4, n_groups=1)

    def status(kv=kv, q=h, start=h, groups=h, shared=h, **kw):
        return L.tcx_attention_shared(ctx.handle, ctypes.byref(kv), ctypes.byref(tc.attention_shared_desc(**{**ok, **kw})), h, q, h, h, start, groups, shared, h, None)
    assert L.tcx_attention_shared(None, *[None] * 11) == tc.TC_ERR_NOT_INITIALIZED
    for bad in (dict(q=None), dict(groups=None), dict(shared=None), dict(tokens=0), dict(n_seqs=0), dict(n_groups=0), dict(n_groups=5), dict(n_groups=-1), dict(max_group_q=-1),
                dict(max_pages=0), dict(q_heads=3), dict(max_q=-1), dict(tokens=5, start=None), dict(q_strides=(-1, 0)), dict(o_strides=(64, 0))):
        assert status(**bad) == tc.TC_ERR_INVALID_ARG, bad
    for bad in (dict(tokens=1 << 12, n_seqs=1 << 12), dict(max_pages=1 << 28), dict(kv=tc.kv_desc(4, 16, 2, 256)), dict(tokens=1 << 30)):
        assert status(**bad) == tc.TC_ERR_INVALID_SHAPE, bad
    assert status(dtype="f32") == tc.TC_ERR_UNSUPPORTED_DTYPE
    p, d = b.device_ptr(), tc.attention_shared_desc(**ok)
    for at, off in ((0, 8), (1, 1), (2, 2), (3, 1), (5, 1), (6, 2), (7, 1), (8, 2)):
        args = [p, p, p, p, None, p, p, p, None]
        args[at] = (args[at] or p) + off
        assert L.tcx_raw_attention_shared(ctx.handle, ctypes.byref(kv), ctypes.byref(d), *args, None) == tc.TC_ERR_INVALID_ARG
