"""Bounds of blocks, the choice of blocks and attention over what is chosen: bounds, scores and choices bit for bit, attention against 64 bits."""
import ctypes

import numpy as np
import pytest

from paged_reference import attention64, numbers, pack, quantise

pytestmark = pytest.mark.gpu
HALF_ULP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
F = np.float32


def _torch():
    import torch
    return torch, {"f16": torch.float16, "bf16": torch.bfloat16}


def _cuda(a, dtype=np.int32):
    return _torch()[0].from_numpy(np.ascontiguousarray(np.asarray(a, dtype))).cuda()


# ---- plain forms, every fp32 step rounded by itself
def bounds_of(k, finite=True):
    """k [Hkv, tokens, D] (what the codes stand for: exact in fp32): hi, lo int8 [Hkv, D], step fp32 [Hkv]."""
    k = k.astype(F)
    hi, lo = k.max(axis=1), k.min(axis=1)
    step = (np.maximum(abs(hi), abs(lo)).max(axis=1) / F(127)).astype(F)
    by = np.where(step > 0, step, F(1))[:, None]
    some = (step > 0)[:, None]
    up = np.where(some, np.clip(np.ceil((hi / by).astype(F)), -127, 127), 0).astype(np.int8)
    down = np.where(some, np.clip(np.floor((lo / by).astype(F)), -127, 127), 0).astype(np.int8)
    return up, down, step


def scores_of(q, hi, lo, step):
    """q [heads, D] of one K/V head (fp32), hi and lo [blocks, D], step [blocks]."""
    most = abs(q).max()
    if not np.isfinite(most):
        q, most = np.zeros_like(q), F(0)
    qs = F(most / F(127))
    code = np.clip(np.rint((q / qs).astype(F)), -127, 127).astype(np.int64) if qs > 0 else np.zeros(q.shape, np.int64)
    total = np.maximum(code[None] * hi[:, None].astype(np.int64), code[None] * lo[:, None].astype(np.int64)).sum(axis=(1, 2))
    with np.errstate(invalid="ignore"):
        return ((total.astype(F) * step).astype(F) * (qs if qs > 0 else F(0))).astype(F)


def choose(scores, first, last, most):
    n = len(scores)
    rank = np.where(np.isnan(scores), np.inf, scores.astype(np.float64))
    forced = [i for i in range(n) if i < first or i >= n - last]
    rest = sorted((i for i in range(n) if i not in set(forced)), key=lambda i: (-rank[i], i))
    return sorted((forced + rest)[:most] if n > most else range(n))


class Cache:
    """Sequences of random keys; every page's bounds are worked out by the library."""

    def __init__(self, tc, lens, H, Hkv, D, P, dtype="f16", seed=0, spare=0xFF, max_pages=None, alike=False):
        torch, types = _torch()
        rng = np.random.default_rng(seed)
        self.lens, self.H, self.Hkv, self.D, self.P, self.dtype = lens, H, Hkv, D, P, dtype
        n = [-(-k // P) for k in lens]
        total = sum(n) + 2
        order, at = rng.permutation(total), 0
        self.table = np.full((len(lens), max_pages or max(1, max(n))), -1, np.int32)
        codes = [np.full((total, Hkv, P, D), spare & 15, np.uint8) for _ in range(2)]
        scales = [np.full((total, Hkv, P, D // 32), np.array([spare * 257], np.uint16).view(np.float16)[0], np.float16) for _ in range(2)]
        self.k, self.v = [], []
        for s, k in enumerate(lens):
            own = order[at:at + n[s]]
            at += n[s]
            self.table[s, :n[s]] = own
            for w, to in enumerate((self.k, self.v)):
                x = rng.standard_normal((Hkv, k, D)).astype(F)
                if alike and w == 0:
                    x = np.tile(rng.standard_normal((Hkv, 1, D)).astype(F), (1, k, 1))      # every block has the same score
                c, d = quantise(x)
                to.append(numbers(c, d))
                for i in range(n[s]):
                    j = slice(i * P, min(k, (i + 1) * P))
                    codes[w][own[i], :, :j.stop - j.start] = c[:, j]
                    scales[w][own[i], :, :j.stop - j.start] = d[:, j]
        self.pages = torch.from_numpy(pack(codes[0], scales[0], codes[1], scales[1])).cuda()
        self.kv = tc.kv_desc(total, P, Hkv, D)
        self.record = tc.kv_bounds_bytes(self.kv)
        self.bounds = torch.full((total, Hkv, self.record), 0xAB, dtype=torch.uint8, device="cuda")
        self.q = torch.from_numpy(rng.standard_normal((len(lens), H, D)).astype(F)).cuda().to(types[dtype])

    def update(self, tc, ctx, first=None, lens=None, max_new=0, stream=0):
        ints = [_cuda([0] * len(self.lens) if first is None else first), _cuda(self.lens if lens is None else lens), _cuda(self.table)]
        _torch()[0].cuda.synchronize()
        tc.raw_kv_bounds(ctx, self.kv, tc.kv_bounds_desc(len(self.lens), self.table.shape[1], max_new), self.pages.data_ptr(), self.bounds.data_ptr(), *(t.data_ptr() for t in ints), stream)
        _torch()[0].cuda.synchronize()
        return self.bounds.cpu().numpy()

    def records(self, s, upto=None):
        """Of sequence s's blocks, in order: hi, lo [blocks, Hkv, D], step [blocks, Hkv]."""
        k = self.k[s][:, :upto]
        got = [bounds_of(k[:, i:i + self.P]) for i in range(0, k.shape[1], self.P)]
        return [np.stack([g[j] for g in got]) if got else np.zeros((0,)) for j in range(3)]

    def want(self, s, upto=None):
        hi, lo, step = self.records(s, upto)
        out = np.zeros((len(step), self.Hkv, self.record), np.uint8)
        if len(step):
            out[:, :, :self.D], out[:, :, self.D:2 * self.D] = hi.view(np.uint8), lo.view(np.uint8)
            out[:, :, 2 * self.D:2 * self.D + 4] = np.ascontiguousarray(step[..., None]).view(np.uint8)
        return out

    def select(self, tc, ctx, blocks, first=0, last=0, positions=None, sequences=None, q=None, q_strides=(0, 0), stream=None):
        torch, _ = _torch()
        T = len(self.q) if positions is None else len(positions)
        ints = [_cuda([k - 1 for k in self.lens] if positions is None else positions), None if sequences is None else _cuda(sequences), _cuda(self.table)]
        scores = torch.full((T, self.Hkv, self.table.shape[1]), 7.0, device="cuda")
        picked, lens = torch.full((T, self.Hkv, blocks), 77, dtype=torch.int32, device="cuda"), torch.full((T,), 77, dtype=torch.int32, device="cuda")
        desc = tc.kv_select_desc(T, len(self.lens), self.table.shape[1], self.H, blocks, first, last, self.dtype, q_strides=q_strides)
        torch.cuda.synchronize()
        tc.raw_kv_select(ctx, self.kv, desc, self.bounds.data_ptr(), (self.q if q is None else q).data_ptr(), ints[0].data_ptr(), 0 if sequences is None else ints[1].data_ptr(),
                         ints[2].data_ptr(), scores.data_ptr(), picked.data_ptr(), lens.data_ptr(), (stream or torch.cuda.current_stream()).cuda_stream)
        torch.cuda.synchronize()
        return scores.cpu().numpy(), picked.cpu().numpy(), lens.cpu().numpy()

    def check(self, got, blocks, first, last, positions=None, sequences=None):
        scores, picked, lens = got
        q, rep = self.q.float().cpu().numpy(), self.H // self.Hkv
        for t, position in enumerate([k - 1 for k in self.lens] if positions is None else positions):
            s = t if sequences is None else sequences[t]
            if position < 0:
                assert lens[t] == 0 and (picked[t] == -1).all() and (scores[t] == 7).all()
                continue
            n = position // self.P + 1
            # (bounds know nothing of a token's place: a block's are of all its keys)
            hi, lo, step = (x[:n] for x in self.records(s))
            for h in range(self.Hkv):
                want = scores_of(q[t, h * rep:(h + 1) * rep], hi[:, h], lo[:, h], step[:, h])
                assert np.array_equal(scores[t, h, :n], want) and (scores[t, h, n:] == 7).all()
                take = choose(want, first, max(1, last), blocks)
                assert picked[t, h].tolist() == self.table[s, take].tolist() + [-1] * (blocks - len(take)), (t, h)
            assert lens[t] == (min(n, blocks) - 1) * self.P + position % self.P + 1


@pytest.mark.parametrize("Hkv,D,P", [(1, 32, 16), (8, 128, 64), (3, 96, 32), (2, 64, 128), (9, 128, 16), (2, 32, 1024)])
def test_bounds(tc, ctx, Hkv, D, P):
    lens = [1, 0, P - 1, P, P + 1, 3 * P, 5 * P + 7]
    c = Cache(tc, lens, Hkv, Hkv, D, P, seed=D)
    c.pages[int(c.table[0, 0]), 0, 0, :256 * (D // 32)] = 0x88                     # a block of zeros
    c.k[0][0] = 0
    for max_new in (0, 1, max(lens)):
        c.bounds.fill_(0xAB)
        got = c.update(tc, ctx, max_new=max_new)
        touched = np.zeros(c.kv.n_pages, bool)
        for s, k in enumerate(lens):
            n = -(-k // P)
            assert np.array_equal(got[c.table[s, :n]], c.want(s)), s
            touched[c.table[s, :n]] = True
        assert (got[~touched] == 0xAB).all()
    assert tc.take_device_error(ctx) == 0


def test_bounds_of_a_few_new_keys(tc, ctx):
    """Blocks without a new key are left as they are; one that has some is worked out from all of its keys up to the length."""
    c = Cache(tc, [100, 64, 17, 5], 4, 2, 64, 16, seed=1)
    first, lens = [95, 64, 16, 0], [100, 64, 17, 0]
    got = c.update(tc, ctx, first, lens, max_new=5)
    for s, blocks in enumerate(([5, 6], [], [1], [])):
        for i in range(-(-c.lens[s] // 16)):
            assert np.array_equal(got[c.table[s, i]], c.want(s)[i]) if i in blocks else (got[c.table[s, i]] == 0xAB).all()
    # with fewer of the keys: those behind the length have no part
    got = c.update(tc, ctx, [80, 0, 0, 0], [90, 20, 0, 3], max_new=20)
    assert np.array_equal(got[c.table[0, 5]], c.want(0, 90)[5]) and np.array_equal(got[c.table[1, :2]], c.want(1, 20)) and np.array_equal(got[c.table[3, 0]], c.want(3, 3)[0])


def test_bounds_of_what_is_not_finite(tc, ctx):
    c = Cache(tc, [48], 1, 2, 64, 16, seed=2)
    tile = c.pages.view(c.kv.n_pages, 2, 1, 1152)
    for i, bits in ((0, 0x7C00), (1, 0x7E00)):
        tile[int(c.table[0, i]), 1, :, 256 * 2 + 3 * 4 + 2:256 * 2 + 3 * 4 + 4] = _torch()[0].from_numpy(np.array([bits], np.uint16).view(np.uint8)).cuda()
    got = c.update(tc, ctx)[c.table[0]]
    want = c.want(0)
    assert np.array_equal(got[:, 0], want[:, 0]) and np.array_equal(got[2], want[2])
    for i in (0, 1):
        assert not got[i, 1, :128].any() and np.isnan(got[i, 1, 128:132].view(F)[0]) and not got[i, 1, 132:].any()


def test_bounds_of_pages_that_do_not_exist(tc, ctx):
    c = Cache(tc, [40, 20], 1, 1, 32, 16, seed=3)
    c.table[0, 1], keep = c.kv.n_pages, c.table[0].copy()
    got = c.update(tc, ctx)
    assert tc.take_device_error(ctx) == 2
    assert np.array_equal(got[c.table[1, :2]], c.want(1)) and np.array_equal(got[keep[[0, 2]]], c.want(0)[[0, 2]])
    c.update(tc, ctx, lens=[2 ** 31 - 1, 20])                             # cut to what the row of the table holds
    assert tc.take_device_error(ctx) == 2


@pytest.mark.parametrize("D,P,H,Hkv,dtype", [(32, 16, 1, 1, "f16"), (64, 16, 8, 2, "f16"), (96, 32, 6, 2, "bf16"), (128, 64, 32, 8, "f16"), (128, 16, 14, 2, "bf16"), (64, 128, 64, 1, "bf16"),
                                             (32, 16, 256, 1, "f16")])
def test_choice(tc, ctx, D, P, H, Hkv, dtype):
    lens = [1, 0, P, P + 1, 7 * P, 8 * P, 9 * P + 3, 20 * P - 1]
    c = Cache(tc, lens, H, Hkv, D, P, dtype, seed=H)
    c.update(tc, ctx)
    for blocks, first, last in ((1, 0, 0), (2, 1, 1), (8, 1, 2), (8, 3, 5), (8, 0, 8), (9, 2, 1), (100, 1, 1)):
        c.check(c.select(tc, ctx, blocks, first, last), blocks, first, last)
    assert tc.take_device_error(ctx) == 0


@pytest.mark.parametrize("n,blocks", [(300, 64), (2100, 100), (8193, 33), (9000, 513)])
def test_choice_of_many(tc, ctx, n, blocks):
    c = Cache(tc, [16 * n - 3, 40], 2, 1, 32, 16, seed=n)
    c.update(tc, ctx)
    c.check(c.select(tc, ctx, blocks, 1, 3), blocks, 1, 3)


@pytest.mark.parametrize("n,blocks", [(40, 8), (700, 300), (8500, 30)])
def test_equal_scores(tc, ctx, n, blocks):
    """All blocks are alike: the earlier ones are taken."""
    c = Cache(tc, [16 * n], 2, 1, 32, 16, seed=n, alike=True)
    c.update(tc, ctx)
    got = c.select(tc, ctx, blocks, 0, 2)
    c.check(got, blocks, 0, 2)
    assert got[1][0, 0].tolist() == c.table[0, list(range(blocks - 2)) + [n - 2, n - 1]].tolist()
    c.q.zero_()
    got = c.select(tc, ctx, blocks, 2, 1)
    c.check(got, blocks, 2, 1)
    assert not got[0].any()


def test_nan_and_infinities(tc, ctx):
    """A block with a NaN comes before all others; queries with something not finite leave no scores, but that NaN."""
    c = Cache(tc, [320], 2, 1, 32, 16, seed=4)
    c.update(tc, ctx)
    c.bounds.view(_torch()[0].float32)[int(c.table[0, 9]), 0, 16] = float("nan")
    scores, picked, _ = c.select(tc, ctx, 2, 0, 1)
    assert np.isnan(scores[0, 0, 9]) and np.isfinite(np.delete(scores[0, 0], 9)).all() and picked[0, 0].tolist() == c.table[0, [9, 19]].tolist()
    for value in (float("inf"), float("nan"), -float("inf")):
        c.q[0, 1, 5] = value
        scores, picked, _ = c.select(tc, ctx, 4, 0, 1)
        assert np.isnan(scores[0, 0, 9]) and not np.delete(scores[0, 0], 9).any() and picked[0, 0].tolist() == c.table[0, [0, 1, 9, 19]].tolist()


def test_tokens_of_sequences_and_strides(tc, ctx):
    """Several tokens of a sequence, in no order, one passed over; queries inside wider rows, at odd addresses, on another stream."""
    torch, types = _torch()
    c = Cache(tc, [200, 90, 130], 8, 2, 64, 16, seed=5, max_pages=40)
    c.update(tc, ctx)
    positions, sequences = [199, 10, -1, 64, 129, 63, 0], [0, 0, 2, 2, 2, 1, 1]
    c.q = torch.randn(7, 8, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(5)).half()
    want = c.select(tc, ctx, 4, 1, 1, positions, sequences)
    c.check(want, 4, 1, 1, positions, sequences)
    wide = torch.zeros(7, 3 * 8 * 64 + 1, dtype=torch.float16, device="cuda")
    rows = wide.view(-1)[1:][:7 * (3 * 512 + 1) - 1]
    view = torch.as_strided(rows, (7, 8, 64), (1537, 130, 1))
    view.copy_(c.q)
    got = c.select(tc, ctx, 4, 1, 1, positions, sequences, q=view, q_strides=(1537, 130), stream=torch.cuda.Stream())
    for a, b in zip(got, want):
        assert np.array_equal(a, b)
    assert tc.take_device_error(ctx) == 0


def test_places_that_do_not_exist(tc, ctx):
    c = Cache(tc, [60, 33], 2, 1, 32, 16, seed=6)
    c.update(tc, ctx)
    good = c.select(tc, ctx, 2, 0, 1)
    for positions, sequences in (([59, 64], [0, 1]), ([59, 10], [0, 2]), ([59, 10], [0, -1]), ([59, 2 ** 31 - 1], [0, 1])):
        scores, picked, lens = c.select(tc, ctx, 2, 0, 1, positions, sequences)
        assert tc.take_device_error(ctx) == 2 and lens[1] == 0 and (picked[1] == -1).all() and (scores[1] == 7).all()
        assert np.array_equal(picked[0], good[1][0]) and lens[0] == good[2][0]
    page = int(c.table[0, 1])
    for bad in (-1, c.kv.n_pages):
        c.table[0, 1] = bad
        scores, picked, _ = c.select(tc, ctx, 2, 0, 1)
        assert tc.take_device_error(ctx) == 2 and scores[0, 0, 1] == -np.inf and bad not in picked[0, 0].tolist() and np.array_equal(picked[1], good[1][1])
    c.table[0, 1] = page


# ---- attention over what is chosen
def attend(c, tc, ctx, picked, lens, q=None, scale=0.0, q_strides=(0, 0), o=None, o_strides=(0, 0), stream=None):
    torch, _ = _torch()
    q = c.q if q is None else q
    T = len(lens)
    o, lse = torch.full((T, c.H, c.D), 3.0, dtype=c.q.dtype, device="cuda") if o is None else o, torch.full((T, c.H), 3.0, device="cuda")
    lists, n = _cuda(picked), _cuda(lens)
    torch.cuda.synchronize()
    tc.raw_attention_blocks(ctx, c.kv, tc.attention_blocks_desc(T, picked.shape[2], c.H, c.dtype, scale, q_strides, o_strides), c.pages.data_ptr(), q.data_ptr(), lists.data_ptr(),
                            n.data_ptr(), o.data_ptr(), lse.data_ptr(), (stream or torch.cuda.current_stream()).cuda_stream)
    torch.cuda.synchronize()
    return o, lse


def check_attention(c, o, lse, blocks_of, lens):
    """blocks_of[t][h]: the blocks of sequence t, rising."""
    o, q, rep = o.float().cpu().numpy().astype(np.float64), c.q.float().cpu().numpy().astype(np.float64), c.H // c.Hkv
    off = near = 0.0
    for t, n in enumerate(lens):
        for h in range(c.Hkv):
            at = np.concatenate([np.arange(i * c.P, min((i + 1) * c.P, c.lens[t])) for i in blocks_of[t][h]] + [np.zeros(0, int)]).astype(int)[:n]
            want, want_lse, room, score_off = attention64(q[t:t + 1, h * rep:(h + 1) * rep], c.k[t][h:h + 1, at], c.v[t][h:h + 1, at], c.D ** -0.5, False, 0)
            got = o[t:t + 1, h * rep:(h + 1) * rep]
            assert np.all(abs(got - want) <= room + HALF_ULP[c.dtype] * abs(want) + 2.0 ** -24), (t, h)
            g, none = lse[t:t + 1, h * rep:(h + 1) * rep].cpu().numpy(), np.isinf(want_lse)
            assert np.all(g[none] == -np.inf) and np.all(abs(g[~none] - want_lse[~none]) <= score_off[~none] + 2.0 ** -22 * (1 + abs(want_lse[~none])))
            off, near = off + np.sum((got - want) ** 2), near + np.sum(want ** 2)
    assert np.sqrt(off) <= (1.0e-3 if c.dtype == "f16" else 3.0e-3) * np.sqrt(near) + 1e-12


@pytest.mark.parametrize("D,P,H,Hkv,dtype", [(32, 16, 1, 1, "f16"), (64, 16, 8, 2, "f16"), (96, 32, 6, 2, "bf16"), (128, 64, 32, 8, "f16"), (128, 16, 14, 2, "bf16"), (64, 32, 16, 1, "f16"),
                                             (64, 16, 66, 2, "bf16"), (128, 128, 64, 8, "f16")])
def test_attention_over_the_choice(tc, ctx, D, P, H, Hkv, dtype):
    """Bounds, choice and attention one after the other: what was chosen, and nothing else, is attended to."""
    lens = [1, 0, P, P + 1, 7 * P, 8 * P, 9 * P + 3, 20 * P - 1]
    c = Cache(tc, lens, H, Hkv, D, P, dtype, seed=H + D)
    c.update(tc, ctx)
    for blocks in (1, 3, 8, 50):
        _, picked, n = c.select(tc, ctx, blocks, 1 if blocks > 1 else 0, 1)
        where = [{int(p): i for i, p in enumerate(c.table[t]) if p >= 0} for t in range(len(lens))]
        blocks_of = [[[where[t][p] for p in picked[t, h] if p >= 0] for h in range(Hkv)] for t in range(len(lens))]
        check_attention(c, *attend(c, tc, ctx, picked, n), blocks_of, n)
    assert tc.take_device_error(ctx) == 0


def test_all_blocks_are_the_whole(tc, ctx):
    """With room for every block the results are those of attention over the pages, to the last bits of sums in another order."""
    torch, _ = _torch()
    c = Cache(tc, [700, 33, 0, 1400], 8, 2, 128, 64, seed=7)
    c.update(tc, ctx)
    _, picked, n = c.select(tc, ctx, 40, 1, 1)
    o, lse = attend(c, tc, ctx, picked, n)
    full, full_lse = torch.zeros_like(c.q), torch.zeros(4, 8, device="cuda")
    ints = [_cuda(c.table), _cuda(c.lens)]
    tc.raw_attention_paged(ctx, c.kv, tc.attention_paged_desc(4, 4, c.table.shape[1], 8, max_q=1), c.pages.data_ptr(), c.q.data_ptr(), ints[0].data_ptr(), ints[1].data_ptr(), 0,
                           full.data_ptr(), full_lse.data_ptr())
    torch.cuda.synchronize()
    assert n.tolist() == c.lens
    assert torch.equal(o, full) and torch.equal(lse, full_lse)            # (the same units of work: the same order too)


def test_many_tokens_strides_and_repeats(tc, ctx):
    torch, _ = _torch()
    rng = np.random.default_rng(8)
    T, blocks = 600, 5
    c = Cache(tc, [80] * T, 4, 2, 64, 16, seed=8)
    blocks_of = [[sorted(rng.choice(5, size=k, replace=False).tolist()) for _ in range(2)] for k in rng.integers(1, 6, T)]
    picked = np.full((T, 2, blocks), -1, np.int32)
    lens = np.array([len(b[0]) * 16 - int(rng.integers(0, 16)) for b in blocks_of], np.int32)
    lens[5] = 0
    for t in range(T):
        for h in range(2):
            picked[t, h, :len(blocks_of[t][h])] = c.table[t, blocks_of[t][h]]
    want = attend(c, tc, ctx, picked, lens)
    check_attention(c, *want, blocks_of, lens)
    wide, out = torch.zeros(T, 600, dtype=torch.float16, device="cuda"), torch.zeros(4, T, 64, dtype=torch.float16, device="cuda")
    wide[:, :256] = c.q.view(T, -1)
    for _ in range(3):
        _, lse = attend(c, tc, ctx, picked, lens, q=wide, q_strides=(600, 64), o=out, o_strides=(64, 64 * T), stream=torch.cuda.Stream())
        assert torch.equal(out.transpose(0, 1), want[0]) and torch.equal(lse, want[1])
    assert tc.take_device_error(ctx) == 0


def test_lists_that_are_wrong(tc, ctx):
    """A page that is not there is passed over, a length past the list cut to it; the error word is set, the other tokens are right."""
    c = Cache(tc, [64, 64, 64], 4, 2, 64, 16, seed=9)
    picked = np.stack([np.tile(c.table[t, :3], (2, 1)) for t in range(3)])
    blocks_of = [[[0, 1, 2]] * 2] * 3
    for page, n in ((c.kv.n_pages, 48), (-1, 48), (2 ** 31 - 1, 48), (None, 49), (None, 2 ** 31 - 1)):
        lists, lens = picked.copy(), np.array([48, n, 30], np.int32)
        if page is not None:
            lists[1, 1, 0] = page
        o, lse = attend(c, tc, ctx, lists, lens)
        assert tc.take_device_error(ctx) == 2 and o.isfinite().all()
        c3 = Cache(tc, [64, 64, 64], 4, 2, 64, 16, seed=9)
        keep = [0, 2]
        c3.lens, c3.k, c3.v, c3.q = [64, 64], [c.k[i] for i in keep], [c.v[i] for i in keep], c.q[keep]
        check_attention(c3, o[keep], lse[keep], [blocks_of[i] for i in keep], lens[keep])
    assert not attend(c, tc, ctx, picked, np.array([48, -3, 5], np.int32))[0][1].any() and tc.take_device_error(ctx) == 0


def test_without_room(tc, ctx):
    c = Cache(tc, [3000, 700], 8, 2, 64, 16, seed=10)
    n = [-(-k // 16) for k in c.lens]
    picked = np.stack([np.tile(np.concatenate([c.table[t, :n[t]], -np.ones(n[0] - n[t], np.int32)]), (2, 1)) for t in range(2)])
    tc.set_device_error(ctx, 1)
    try:
        got = attend(c, tc, ctx, picked, np.array(c.lens, np.int32))
    finally:
        assert tc.take_device_error(ctx) == 1
    check_attention(c, *got, [[list(range(n[t]))] * 2 for t in range(2)], c.lens)


def test_on_buffers_and_in_graphs(tc, ctx):
    torch, _ = _torch()
    c = Cache(tc, [200, 90, 130], 8, 2, 64, 16, seed=11)
    bounds = c.update(tc, ctx)
    scores, picked, n = c.select(tc, ctx, 4, 1, 1)
    o, lse = attend(c, tc, ctx, picked, n)
    pages, q = ctx.buffer_from_array(c.pages.cpu().numpy()), ctx.buffer_from_array(c.q.cpu().numpy())
    bb = ctx.buffer_from_array(np.full(bounds.shape, 0xAB, np.uint8))
    zero, lens, table, pos = (ctx.buffer_from_array(np.array(a, np.int32)) for a in ([0, 0, 0], c.lens, c.table, [k - 1 for k in c.lens]))
    sc, pk, ln = ctx.buffer_from_array(np.full(scores.shape, 7.0, F)), ctx.buffer(picked.nbytes), ctx.buffer(n.nbytes)
    before = tc.launch_count()
    tc.kv_bounds(ctx, c.kv, tc.kv_bounds_desc(3, c.table.shape[1]), pages, bb, zero, lens, table)
    assert "kv_bounds" in tc.cuda_last_kernel_name() and np.array_equal(bb.to_numpy(bounds.shape, np.uint8), bounds)
    tc.kv_select(ctx, c.kv, tc.kv_select_desc(3, 3, c.table.shape[1], 8, 4, 1, 1), bb, q, pos, None, table, sc, pk, ln)
    assert "kv_select" in tc.cuda_last_kernel_name() and tc.launch_count() == before + 3
    assert np.array_equal(sc.to_numpy(scores.shape, F), scores) and np.array_equal(pk.to_numpy(picked.shape, np.int32), picked) and np.array_equal(ln.to_numpy(n.shape, np.int32), n)
    bo, bl = ctx.buffer(c.q.numel() * 2), ctx.buffer(3 * 8 * 4)
    tc.attention_blocks(ctx, c.kv, tc.attention_blocks_desc(3, 4, 8), pages, q, pk, ln, bo, bl)
    assert "attention_blocks" in tc.cuda_last_kernel_name()
    assert np.array_equal(bo.to_numpy(c.q.shape, np.float16), o.cpu().numpy()) and np.array_equal(bl.to_numpy((3, 8), F), lse.cpu().numpy())
    # the three in one graph, replayed with other queries and places
    ints = [_cuda([0, 0, 0]), _cuda(c.lens), _cuda(c.table), _cuda([k - 1 for k in c.lens])]
    ts, tp, tl = torch.zeros(3, 2, c.table.shape[1], device="cuda"), torch.zeros(3, 2, 4, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    to, tlse = torch.zeros_like(c.q), torch.zeros(3, 8, device="cuda")

    def call(st):
        tc.raw_kv_bounds(ctx, c.kv, tc.kv_bounds_desc(3, c.table.shape[1]), c.pages.data_ptr(), c.bounds.data_ptr(), ints[0].data_ptr(), ints[1].data_ptr(), ints[2].data_ptr(), st)
        tc.raw_kv_select(ctx, c.kv, tc.kv_select_desc(3, 3, c.table.shape[1], 8, 4, 1, 1), c.bounds.data_ptr(), c.q.data_ptr(), ints[3].data_ptr(), 0, ints[2].data_ptr(), ts.data_ptr(),
                         tp.data_ptr(), tl.data_ptr(), st)
        tc.raw_attention_blocks(ctx, c.kv, tc.attention_blocks_desc(3, 4, 8), c.pages.data_ptr(), c.q.data_ptr(), tp.data_ptr(), tl.data_ptr(), to.data_ptr(), tlse.data_ptr(), st)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    call(side.cuda_stream)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        call(side.cuda_stream)
    old = c.q.clone()
    for turn in range(3):
        c.q.copy_(old if turn != 1 else old.flip(0))
        c.bounds.fill_(0xAB)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        if turn != 1:
            assert np.array_equal(tp.cpu().numpy(), picked) and torch.equal(to, o) and torch.equal(tlse, lse)
        else:
            assert not torch.equal(to, o)
    del g
    assert tc.take_device_error(ctx) == 0


def test_refusals(tc, ctx):
    L, b = tc.lib(), ctx.buffer(1 << 16)
    h, kv = b.handle, tc.kv_desc(4, 16, 2, 64)
    ref = ctypes.byref

    def bounds(kv=kv, pages=h, out=h, first=h, **kw):
        return L.tcx_kv_bounds(ctx.handle, ref(kv), ref(tc.kv_bounds_desc(**{**dict(n_seqs=1, max_pages=1), **kw})), pages, out, first, h, h)

    def select(kv=kv, q=h, scores=h, sequences=None, **kw):
        return L.tcx_kv_select(ctx.handle, ref(kv), ref(tc.kv_select_desc(**{**dict(tokens=1, n_seqs=1, max_pages=1, q_heads=2, max_blocks=2), **kw})), h, q, h, sequences, h, scores, h, h)

    def blocks(kv=kv, q=h, lists=h, **kw):
        return L.tcx_attention_blocks(ctx.handle, ref(kv), ref(tc.attention_blocks_desc(**{**dict(tokens=1, max_blocks=1, q_heads=2), **kw})), h, q, lists, h, h, None)
    for call, n in ((L.tcx_kv_bounds, 7), (L.tcx_kv_select, 10), (L.tcx_attention_blocks, 8)):
        assert call(None, *[None] * n) == tc.TC_ERR_NOT_INITIALIZED
    A, S = tc.TC_ERR_INVALID_ARG, tc.TC_ERR_INVALID_SHAPE
    for bad in (dict(n_seqs=0), dict(max_pages=0), dict(max_new=-1), dict(pages=None), dict(out=None), dict(first=None)):
        assert bounds(**bad) == A, bad
    for bad in (dict(tokens=0), dict(n_seqs=0), dict(max_pages=0), dict(q_heads=0), dict(q_heads=3), dict(max_blocks=0), dict(first_blocks=-1), dict(last_blocks=-1),
                dict(first_blocks=2), dict(first_blocks=1, last_blocks=2), dict(last_blocks=3), dict(q=None), dict(scores=None), dict(q_strides=(-1, 0))):
        assert select(**bad) == A, bad
    for bad in (dict(tokens=2), dict(q_heads=2 * 257), dict(max_pages=1 << 27), dict(max_blocks=1 << 27), dict(tokens=1 << 30, n_seqs=1 << 30)):
        assert select(**bad) == S, bad
    for bad in (dict(tokens=0), dict(max_blocks=0), dict(q_heads=0), dict(q_heads=5), dict(q=None), dict(lists=None), dict(o_strides=(64, 0), tokens=2), dict(q_strides=(0, -1))):
        assert blocks(**bad) == A, bad
    for bad in (dict(max_blocks=1 << 27), dict(tokens=1 << 30), dict(tokens=1 << 12)):
        assert blocks(**bad) == S, bad
    assert bounds(n_seqs=1 << 15) == S and bounds(max_pages=1 << 27) == S
    for call in (bounds, select, blocks):
        assert call(kv=tc.kv_desc(4, 16, 2, 256)) == S and call(kv=tc.kv_desc(4, 20, 2, 64)) == S and call(kv=tc.kv_desc(0, 16, 2, 64)) == A
    assert select(dtype="f32") == tc.TC_ERR_UNSUPPORTED_DTYPE and blocks(dtype="f32") == tc.TC_ERR_UNSUPPORTED_DTYPE
    p = b.device_ptr()
    for fn, d, n, odd in ((L.tcx_raw_kv_bounds, tc.kv_bounds_desc(1, 1), 5, {0: 8, 1: 8, 2: 2, 3: 1, 4: 2}),
                          (L.tcx_raw_kv_select, tc.kv_select_desc(1, 1, 1, 2, 2), 8, {0: 8, 1: 1, 2: 2, 3: 2, 4: 1, 5: 2, 6: 2, 7: 1}),
                          (L.tcx_raw_attention_blocks, tc.attention_blocks_desc(1, 1, 2), 6, {0: 8, 1: 1, 2: 2, 3: 1, 4: 1, 5: 2})):
        for at, off in odd.items():
            args = [p] * n
            args[at] += off
            assert fn(ctx.handle, ref(kv), ref(d), *args, None) == A, (fn, at)
