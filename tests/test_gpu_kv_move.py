"""Pages and tokens of the 4-bit cache moved: byte for byte against the same moves in numpy, by the documented places."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


def _cuda(a, dtype=np.int32):
    return _torch().from_numpy(np.ascontiguousarray(np.asarray(a, dtype))).cuda()


def _bytes_of_a_token(nb, r):
    """Byte offsets within a tile of all that token r has there."""
    h, t, e = r // 8, r % 8 // 2, r % 2
    at = [r * 16 * nb + i for i in range(16 * nb)] + [256 * nb + r * 2 * nb + i for i in range(2 * nb)]
    for block in range(nb):
        for g in range(8):
            at += [288 * nb + ((((h * 8 + g) * 4 + t) * nb + block) * 2 + e) * 2 + i for i in range(2)]
        at += [544 * nb + (((h * 4 + t) * nb + block) * 2 + e) * 2 + i for i in range(2)]
    return at


class Cache:
    """Random bytes of `layers` layers, `gap` bytes between two of them."""

    def __init__(self, tc, n, P, Hkv, D, layers=1, gap=0, seed=0):
        rng = np.random.default_rng(seed)
        self.kv, self.n, self.P, self.Hkv, self.D, self.layers = tc.kv_desc(n, P, Hkv, D), n, P, Hkv, D, layers
        self.layer = n * tc.kv_page_bytes(self.kv)
        self.stride = self.layer + gap
        self.host = rng.integers(0, 256, self.stride * layers, dtype=np.uint8)
        self.dev = _torch().from_numpy(self.host).cuda()

    def view(self, host, layer):
        return host[layer * self.stride:layer * self.stride + self.layer].reshape(self.n, self.Hkv, self.P // 16, 18 * self.D)

    def got(self):
        _torch().cuda.synchronize()
        return self.dev.cpu().numpy()

    # -- plain forms
    def copied(self, src, dst, counts=None):
        out = self.host.copy()
        for layer in range(self.layers):
            old, new = self.view(self.host, layer), self.view(out, layer)
            for i, (a, b) in enumerate(zip(src, dst)):
                tiles = self.P // 16 if counts is None else -(-counts[i] // 16)
                if a >= 0 and tiles > 0:
                    new[b, :, :tiles] = old[a, :, :tiles]
        return out

    def compacted(self, table, to, lists, without=()):
        out = self.host.copy()
        for layer in range(self.layers):
            old, new = self.view(self.host, layer), self.view(out, layer)
            for s, keep in enumerate(lists):
                for j, place in enumerate(keep):
                    if (s, j) in without:
                        continue
                    d = to[s] + j
                    a, b = table[s][place // self.P], table[s][d // self.P]
                    new[b, :, d % self.P // 16, _bytes_of_a_token(self.D // 32, d % 16)] = old[a, :, place % self.P // 16, _bytes_of_a_token(self.D // 32, place % 16)]
        return out


def _copy(tc, ctx, c, src, dst, counts=None):
    t = [_cuda(a) for a in (src, dst) + (() if counts is None else (counts,))]      # (they live as long as the call)
    tc.raw_kv_copy(ctx, c.kv, tc.kv_copy_desc(len(src), c.layers, c.stride if c.stride != c.layer else 0), c.dev.data_ptr(), t[0].data_ptr(), t[1].data_ptr(),
                   0 if counts is None else t[2].data_ptr(), _torch().cuda.current_stream().cuda_stream)
    return c.got()


@pytest.mark.parametrize("n,P,Hkv,D,layers,gap", [(5, 16, 1, 32, 1, 0), (9, 64, 8, 128, 3, 0), (7, 32, 3, 96, 2, 4096), (4, 128, 2, 64, 5, 16), (3, 1024, 5, 32, 2, 0), (40, 16, 4, 128, 1, 0)])
def test_copies(tc, ctx, n, P, Hkv, D, layers, gap):
    rng = np.random.default_rng(n)
    for counts in (None, [0, 1, 15, 16, 17, P - 1, P]):
        c = Cache(tc, n, P, Hkv, D, layers, gap, seed=n)
        order = rng.permutation(n)
        pairs = n // 2
        src, dst = order[:pairs].tolist() + [-1, -7], order[pairs:2 * pairs].tolist() + [0, 2 ** 31 - 1]     # the last two are passed over
        num = None if counts is None else [min(counts[i % len(counts)], P) for i in range(len(src))]
        assert np.array_equal(_copy(tc, ctx, c, src, dst, num), c.copied(src, dst, num))
    assert tc.take_device_error(ctx) == 0


def test_a_page_onto_itself_and_from_one_to_many(tc, ctx):
    c = Cache(tc, 12, 16, 2, 64, 2, seed=1)
    src, dst = [3, 5, 5, 5, 0], [3, 1, 2, 11, 4]
    assert np.array_equal(_copy(tc, ctx, c, src, dst), c.copied(src, dst))


@pytest.mark.parametrize("src,dst,counts", [(6, 1, 16), (2 ** 31 - 1, 1, 16), (0, -1, 16), (0, 6, 16), (0, 1, 17)])
def test_copies_that_cannot_be(tc, ctx, src, dst, counts):
    """The pair is left out, the error word set; the others are copied."""
    c = Cache(tc, 6, 16, 2, 32, 2, seed=2)
    assert np.array_equal(_copy(tc, ctx, c, [2, src, 3], [4, dst, 5], [16, counts, 9]), c.copied([2, 3], [4, 5], [16, 9]))
    assert tc.take_device_error(ctx) == 2


def test_many_pairs_and_layers(tc, ctx):
    c = Cache(tc, 400, 16, 1, 32, 37, seed=3)
    order = np.random.default_rng(3).permutation(400)
    assert np.array_equal(_copy(tc, ctx, c, order[:200], order[200:]), c.copied(order[:200], order[200:]))


def _table(rng, lens, P, spare=2):
    n = [max(1, -(-k // P)) for k in lens]
    order = rng.permutation(sum(n) + spare)
    table, at = np.full((len(n), max(n)), -1, np.int32), 0
    for s, k in enumerate(n):
        table[s, :k] = order[at:at + k]
        at += k
    return table, sum(n) + spare


def _compact(tc, ctx, c, table, to, lists, stream=0):
    start = np.concatenate([[0], np.cumsum([len(k) for k in lists])])
    keep = [p for k in lists for p in k]
    t = [_cuda(a) for a in (table, to, start, keep)]
    _torch().cuda.synchronize()
    tc.raw_kv_compact(ctx, c.kv, tc.kv_compact_desc(len(keep), len(lists), table.shape[1], c.layers, c.stride if c.stride != c.layer else 0), c.dev.data_ptr(),
                      *(x.data_ptr() for x in t), stream)
    got = c.got()
    del t
    return got


@pytest.mark.parametrize("P,Hkv,D,layers,gap", [(16, 1, 32, 1, 0), (64, 8, 128, 2, 0), (32, 3, 96, 2, 64), (16, 2, 64, 5, 0), (128, 5, 128, 1, 0), (1024, 1, 64, 1, 0)])
def test_chosen_tokens_move_down(tc, ctx, P, Hkv, D, layers, gap):
    rng = np.random.default_rng(P + D)
    lens = [40, 1, 300, 17, 900, 33, 64]
    table, n = _table(rng, lens, P)
    for share in (0.1, 0.5, 0.95):
        to = [int(rng.integers(0, k)) for k in lens]
        # any rising list of places at or above the first one that the tokens go to: token j never goes up
        lists = [sorted(rng.choice(np.arange(a, k), size=int(np.ceil(share * (k - a))), replace=False).tolist()) for a, k in zip(to, lens)]
        lists[5] = []
        c = Cache(tc, n, P, Hkv, D, layers, gap, seed=P)
        assert np.array_equal(_compact(tc, ctx, c, table, to, lists), c.compacted(table, to, lists))
    assert tc.take_device_error(ctx) == 0


@pytest.mark.parametrize("by", [1, 2, 3, 16, 255, 256, 257, 1000])
@pytest.mark.parametrize("first", [0, 5])
def test_long_runs_over_themselves(tc, ctx, by, first):
    """2000 tokens a few places down: what one chunk is read from is where the one before is written."""
    rng = np.random.default_rng(by)
    table, n = _table(rng, [first + 2000 + by], 32)
    c = Cache(tc, n, 32, 2, 128, 1, seed=by)
    lists = [list(range(first + by, first + by + 2000))]
    assert np.array_equal(_compact(tc, ctx, c, table, [first], lists), c.compacted(table, [first], lists))


@pytest.mark.parametrize("P,Hkv,D,layers,gap", [(16, 1, 32, 3, 0), (64, 8, 128, 2, 0), (32, 3, 96, 2, 64), (16, 2, 64, 1, 0), (1024, 2, 96, 1, 0)])
def test_long_lists_of_several_sequences(tc, ctx, P, Hkv, D, layers, gap):
    """Of one round of places and of many, with gaps, and beside short and empty ones."""
    rng = np.random.default_rng(P + D)
    lens = [2500, 3, 900, 1400, 257]
    table, n = _table(rng, lens, P)
    for share, to in ((0.4, [0, 1, 7, 100, 0]), (0.97, [1, 0, 16, 9, 8]), (1.0, [2, 3, 896, 0, 1])):
        lists = [sorted(rng.choice(np.arange(a, k), size=int(np.ceil(share * (k - a))), replace=False).tolist()) for a, k in zip(to, lens)]
        c = Cache(tc, n, P, Hkv, D, layers, gap, seed=P)
        assert np.array_equal(_compact(tc, ctx, c, table, to, lists), c.compacted(table, to, lists))
    assert tc.take_device_error(ctx) == 0


def test_long_lists_with_moves_that_cannot_be(tc, ctx):
    rng = np.random.default_rng(8)
    table, n = _table(rng, [3000, 2000], 16)
    table[0, 40], table[1, 100] = n, -1                      # places 640 .. 655 of one, 1600 .. 1615 of the other are not there
    to = [5, 0]
    lists = [sorted(rng.choice(np.arange(a, k), size=1500, replace=False).tolist()) for a, k in zip(to, (3000, 2000))]
    for s, at, value in ((0, 300, -7), (0, 511, 1 << 30), (1, 256, 10), (1, 1000, lists[1][999])):
        lists[s][at] = value
    gone = ({*range(640, 656)}, {*range(1600, 1616)})
    out = set()
    for s, places in enumerate((table.shape[1] * 16, 2000)):
        for j, p in enumerate(lists[s]):
            if not to[s] + j <= p < places or (j and lists[s][j - 1] >= p) or p in gone[s] or to[s] + j in gone[s]:
                out.add((s, j))
    c = Cache(tc, n, 16, 2, 128, 2, seed=8)
    assert np.array_equal(_compact(tc, ctx, c, table, to, lists), c.compacted(table, to, lists, out))
    assert tc.take_device_error(ctx) == 2


def test_tokens_that_stay(tc, ctx):
    c = Cache(tc, 4, 16, 2, 128, 3, seed=9)
    table = np.array([[2, 0, 3]], np.int32)
    for to, keep in ((4, [4, 5, 6, 7]), (4, [4, 6, 7, 9]), (0, [0, 1, 30, 47]), (7, [7])):
        c.dev.copy_(_torch().from_numpy(c.host))
        assert np.array_equal(_compact(tc, ctx, c, table, [to], [keep]), c.compacted(table, [to], [keep]))


@pytest.mark.parametrize("bad,value", [(2, 48), (2, -1), (2, 2 ** 31 - 1), (2, 3), (1, 2)])
def test_moves_that_cannot_be(tc, ctx, bad, value):
    """A place that is not there, one that does not rise, one that would go up: that token is left out (and one behind a place that is too high, for
    the list does not rise there)."""
    c = Cache(tc, 6, 16, 2, 64, 2, seed=4)
    table = np.array([[2, 0, 3], [5, 1, 4]], np.int32)
    lists = [[8, 9, 20, 21], [7, 30]]
    lists[0][bad] = value
    # token 3 stands at place 21: not above its neighbour where that is 48 or more
    out = {(0, j) for j, p in enumerate(lists[0]) if p < 0 or p >= 48 or p < 3 + j or (j and lists[0][j - 1] >= p)}
    assert np.array_equal(_compact(tc, ctx, c, table, [3, 7], lists), c.compacted(table, [3, 7], lists, out))
    assert tc.take_device_error(ctx) == 2


def test_pages_that_do_not_exist(tc, ctx):
    c = Cache(tc, 4, 16, 1, 32, 1, seed=6)
    for table in ([[0, 4, 2]], [[0, -1, 2]]):
        table = np.array(table, np.int32)
        lists = [[14, 20, 21, 33]]
        # the second and third come from the page that is not there, the last would go to it
        assert np.array_equal(_compact(tc, ctx, c, table, [13], lists), c.compacted(table, [13], lists, {(0, 1), (0, 2), (0, 3)}))
        assert tc.take_device_error(ctx) == 2
        c.dev.copy_(_torch().from_numpy(c.host))


def test_on_buffers_streams_and_in_graphs(tc, ctx):
    torch = _torch()
    c = Cache(tc, 6, 16, 2, 64, 2, seed=5)
    want = c.copied([0, 1], [4, 5], [16, 3])
    pages = ctx.buffer_from_array(c.host)
    before = tc.launch_count()
    tc.kv_copy(ctx, c.kv, tc.kv_copy_desc(2, 2), pages, *(ctx.buffer_from_array(np.array(a, np.int32)) for a in ([0, 1], [4, 5], [16, 3])))
    assert tc.launch_count() == before + 1 and "kv_copy" in tc.cuda_last_kernel_name()
    assert np.array_equal(pages.to_numpy(c.host.shape, np.uint8), want)
    table, lists = np.array([[2, 0, 3], [5, 1, 4]], np.int32), [[9, 20, 21], [7, 30]]
    want = c.compacted(table, [3, 7], lists)
    pages = ctx.buffer_from_array(c.host)
    tc.kv_compact(ctx, c.kv, tc.kv_compact_desc(5, 2, 3, 2), pages, *(ctx.buffer_from_array(np.array(a, np.int32)) for a in (table, [3, 7], [0, 3, 5], [9, 20, 21, 7, 30])))
    assert np.array_equal(pages.to_numpy(c.host.shape, np.uint8), want)
    # captured: the lists are read when the graph runs
    ints = [_cuda(a) for a in (table, [3, 7], [0, 3, 5], [9, 20, 21, 7, 30], [0, 1], [4, 5])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        tc.raw_kv_compact(ctx, c.kv, tc.kv_compact_desc(5, 2, 3, 2), c.dev.data_ptr(), *(x.data_ptr() for x in ints[:4]), side.cuda_stream)
    for lists in (lists, [[8, 9, 40], [30, 31]]):
        ints[3].copy_(_cuda([p for k in lists for p in k]))
        c.dev.copy_(torch.from_numpy(c.host))
        torch.cuda.synchronize()
        g.replay()
        assert np.array_equal(c.got(), c.compacted(table, [3, 7], lists))
    del g
    assert tc.take_device_error(ctx) == 0


def test_pages_behind_four_gigabytes(tc, ctx):
    torch = _torch()
    kv = tc.kv_desc(80000, 64, 8, 128)                                   # 5.9 GB
    page = tc.kv_page_bytes(kv)
    dev = torch.empty(80000 * page, dtype=torch.uint8, device="cuda")
    low, high = dev[:2 * page], dev[79998 * page:]
    low.random_(0, 256)
    high.zero_()
    ints = [_cuda(a) for a in ([0, 1], [79998, 79999], [[79998, 79999]], [0], [0, 1], [100])]
    tc.raw_kv_copy(ctx, kv, tc.kv_copy_desc(2), dev.data_ptr(), ints[0].data_ptr(), ints[1].data_ptr())
    assert torch.equal(low, high)
    tc.raw_kv_compact(ctx, kv, tc.kv_compact_desc(1, 1, 2), dev.data_ptr(), *(t.data_ptr() for t in ints[2:]))
    torch.cuda.synchronize()
    h = high.view(2, 8, 4, 2304)
    assert torch.equal(h[0, :, 0, _bytes_of_a_token(4, 0)], h[1, :, 2, _bytes_of_a_token(4, 4)])
    assert torch.equal(high[page:], low[page:]) and tc.take_device_error(ctx) == 0


def test_refusals(tc, ctx):
    L, h, kv = tc.lib(), ctx.buffer(1 << 16).handle, tc.kv_desc(4, 16, 2, 64)

    def copy(kv=kv, pages=h, src=h, dst=h, **kw):
        return L.tcx_kv_copy(ctx.handle, ctypes.byref(kv), ctypes.byref(tc.kv_copy_desc(**{**dict(pairs=1, layers=1), **kw})), pages, src, dst, None)

    def compact(kv=kv, keep=h, to=h, start=h, **kw):
        return L.tcx_kv_compact(ctx.handle, ctypes.byref(kv), ctypes.byref(tc.kv_compact_desc(**{**dict(tokens=1, n_seqs=1, max_pages=1), **kw})), h, h, to, start, keep)
    layer = 4 * tc.kv_page_bytes(kv)
    for bad in (dict(pairs=0), dict(pairs=-1), dict(layers=0), dict(layers=2, layer_stride=layer - 16), dict(layer_stride=8), dict(layer_stride=-16), dict(src=None), dict(dst=None),
                dict(pages=None), dict(kv=tc.kv_desc(0, 16, 2, 64))):
        assert copy(**bad) == tc.TC_ERR_INVALID_ARG, bad
    for bad in (dict(tokens=0), dict(n_seqs=0), dict(max_pages=0), dict(layers=0), dict(layer_stride=24), dict(keep=None), dict(to=None), dict(start=None)):
        assert compact(**bad) == tc.TC_ERR_INVALID_ARG, bad
    for call in (copy, compact):
        for bad in (dict(layers=1 << 20), dict(kv=tc.kv_desc(4, 24, 2, 64)), dict(kv=tc.kv_desc(2 ** 31 - 1, 1024, 1, 32)), dict(kv=tc.kv_desc(4, 16, 2, 48))):
            assert call(**bad) == tc.TC_ERR_INVALID_SHAPE, bad
    assert copy(pairs=1 << 20) == tc.TC_ERR_INVALID_SHAPE and compact(n_seqs=1 << 20) == tc.TC_ERR_INVALID_SHAPE      # buffers that are too small
    p = ctx.buffer(1 << 16).device_ptr()
    for at, off in ((0, 8), (1, 2), (2, 1), (3, 2)):
        args = [p, p, p, p]
        args[at] += off
        assert L.tcx_raw_kv_copy(ctx.handle, ctypes.byref(kv), ctypes.byref(tc.kv_copy_desc(1)), *args, None) == tc.TC_ERR_INVALID_ARG
    for at, off in ((0, 8), (1, 2), (2, 1), (3, 2), (4, 1)):
        args = [p] * 5
        args[at] += off
        assert L.tcx_raw_kv_compact(ctx.handle, ctypes.byref(kv), ctypes.byref(tc.kv_compact_desc(1, 1, 1)), *args, None) == tc.TC_ERR_INVALID_ARG
