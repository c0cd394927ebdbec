"""Layers over a cache whose pages sequences have together: forked, added to, kept in part, attended to by blocks."""
import numpy as np
import pytest

from test_gpu_paged_decoder import APART, _apart

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def shape():
    from tensorcore_b200 import decode as D
    return D.tiny_shape()


def _decoder(tc, ctx, shape, **kw):
    from tensorcore_b200 import paged
    return paged.PagedDecoder(ctx, shape, **{**dict(slots=4, n_pages=48, page_tokens=16, max_pages=12), **kw})


def _rows_of(tc, ctx, d, layer, slot, places):
    """Keys and values of the cache at places of a slot, as fp32 numbers."""
    import torch
    ints = torch.from_numpy(np.concatenate([places, [slot] * len(places), d.book.table.reshape(-1)]).astype(np.int32)).cuda()
    out = torch.zeros(2, len(places), d.kv.kv_heads, d.kv.head_dim, device="cuda")
    slots, most = d.book.table.shape
    tc.raw_kv_read(ctx, d.kv, tc.kv_read_desc(len(places), slots, most, dtype="f32"), d.pages[layer].data_ptr(), out[0].data_ptr(), out[1].data_ptr(), ints.data_ptr(),
                   ints[len(places):].data_ptr(), ints[2 * len(places):].data_ptr(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("prompt", [90, 96])
def test_forks_go_on_like_sequences_of_their_own(tc, ctx, shape, prompt):
    import torch
    from tensorcore_b200 import paged
    x = paged.rows(prompt, shape.d_model, 1)
    more = [paged.rows(20, shape.d_model, 10 + s) for s in range(4)]
    alone, forked = _decoder(tc, ctx, shape), _decoder(tc, ctx, shape)
    for s in range(3):
        alone.step(x, [prompt if s == i else 0 for i in range(4)])
    forked.step(x, [prompt, 0, 0, 0])
    forked.fork(0, 2)
    forked.fork(2, 1)
    assert forked.book.free_pages() > alone.book.free_pages()
    a, b = 0, 0
    for counts in ([1, 1, 1, 0], [0, 2, 1, 0], [3, 1, 0, 0], [1, 1, 1, 0], [5, 0, 9, 0]):
        y = torch.cat([more[s][a:a + n] for s, n in enumerate(counts)])
        want, got = alone.step(y, counts), forked.step(y, counts)
        assert torch.isfinite(got).all() and _apart(got, want, y) <= APART
        a += max(counts)
    assert (forked.book.groups()[1] > 0).any() and forked.book.lengths.tolist() == alone.book.lengths.tolist()
    for s in range(3):                                       # what was shared is as it was, in every layer
        for layer in range(shape.n_layers):
            got, want = (_rows_of(tc, ctx, d, layer, s, np.arange(prompt)) for d in (forked, alone))
            # (first layer: of the same rows; their projections' last fp16 places differ from run to run, which can turn a code over)
            assert ((got - want).norm() / want.norm()).item() <= 4 * APART
        assert torch.equal(_rows_of(tc, ctx, forked, 0, s, np.arange(prompt)), _rows_of(tc, ctx, forked, 0, 0, np.arange(prompt)))
    forked.release(0)
    forked.release(1)
    forked.release(2)
    assert forked.book.free_pages() == 48 and tc.take_device_error(ctx) == 0


def test_many_samples_of_one_prompt(tc, ctx, shape):
    """So many that their shared keys are read once."""
    import torch
    from tensorcore_b200 import paged
    n, prompt = 80, 1500
    kw = dict(slots=n, n_pages=2 * n + 100, page_tokens=16, max_pages=100)
    d = _decoder(tc, ctx, shape, **kw)
    x = paged.rows(prompt, shape.d_model, 2)
    d.step(x, [prompt] + [0] * (n - 1))
    for s in range(1, n):
        d.fork(0, s)
    y = paged.rows(n, shape.d_model, 3)
    got = d.step(y, [1] * n)
    one = _decoder(tc, ctx, shape, slots=1, n_pages=100, max_pages=100)
    for s in (0, 1, 40, 79):
        one.release(0)
        one.step(x, [prompt])
        assert _apart(got[s:s + 1], one.step(y[s:s + 1], [1]), y[s:s + 1]) <= APART
    assert d.book.free_pages() == 2 * n + 100 - (prompt // 16) - n and tc.take_device_error(ctx) == 0


def test_what_is_kept_is_as_it_was(tc, ctx, shape):
    import torch
    from tensorcore_b200 import paged
    d = _decoder(tc, ctx, shape, blocks=4)
    d.step(paged.rows(150, shape.d_model, 4), [100, 50, 0, 0])
    places = np.array([4, 5, 9, 30, 31, 32, 47, 48, 63, 64, 80, 99])
    before = [_rows_of(tc, ctx, d, l, 0, places) for l in range(shape.n_layers)]
    other = _rows_of(tc, ctx, d, 0, 1, np.arange(50))
    free = d.book.free_pages()
    d.keep(0, 4, places)
    assert d.book.lengths[0] == 16 and d.book.free_pages() == free + 6
    for l in range(shape.n_layers):
        assert torch.equal(_rows_of(tc, ctx, d, l, 0, 4 + np.arange(len(places))), before[l])
    assert torch.equal(_rows_of(tc, ctx, d, 0, 1, np.arange(50)), other)
    k = before[0][0]                                         # its bounds have been worked out again
    head = _rows_of(tc, ctx, d, 0, 0, np.arange(16))[0]
    step = head.abs().amax(dim=(0, 2)) / torch.full((head.shape[1],), 127.0, device="cuda")
    got = d.bounds[0, int(d.book.table[0, 0])].view(torch.float32)[:, 2 * d.head_dim // 4]
    assert torch.equal(got, step)
    y = d.step(paged.rows(2, shape.d_model, 5), [1, 1, 0, 0])
    assert torch.isfinite(y).all() and d.book.lengths.tolist() == [17, 51, 0, 0] and k.shape[0] == 12
    assert tc.take_device_error(ctx) == 0


def test_bounds_of_a_page_that_another_has_more_of(tc, ctx, shape):
    import torch
    from tensorcore_b200 import paged
    d = _decoder(tc, ctx, shape, blocks=4)
    d.step(paged.rows(60, shape.d_model, 8), [60, 0, 0, 0])
    d.fork(0, 1)
    before = d.bounds.clone()
    d.keep(1, 50, [])                                        # the page of places 48 .. 63, whose first sequence has 60
    assert d.book.lengths.tolist() == [60, 50, 0, 0] and torch.equal(d.bounds, before)
    d.release(0)                                             # now it is the second one's alone
    d.keep(1, 49, [49])
    assert not torch.equal(d.bounds, before)
    head = _rows_of(tc, ctx, d, 0, 1, np.arange(48, 50))[0]
    step = head.abs().amax(dim=(0, 2)) / torch.full((head.shape[1],), 127.0, device="cuda")
    assert torch.equal(d.bounds[0, int(d.book.table[1, 3])].view(torch.float32)[:, 2 * d.head_dim // 4], step)
    assert tc.take_device_error(ctx) == 0


def test_blocks(tc, ctx, shape):
    """With room for all blocks the layers add what they add without a choice; with few, something near it, from prompts on and over forks."""
    import torch
    from tensorcore_b200 import paged
    x, more = paged.rows(130, shape.d_model, 6), paged.rows(12, shape.d_model, 7)
    full, wide, few = (_decoder(tc, ctx, shape, blocks=b) for b in (0, 12, 3))
    for d in (full, wide, few):
        d.step(x, [90, 40, 0, 0])
        d.fork(0, 2)
    for t in range(4):
        y = more[3 * t:3 * t + 3]
        want = full.step(y, [1, 1, 1, 0])
        assert _apart(wide.step(y, [1, 1, 1, 0]), want, y) <= APART
        got = few.step(y, [1, 1, 1, 0])
        assert torch.isfinite(got).all() and not torch.equal(got, want)
    assert tc.take_device_error(ctx) == 0


def test_the_command_with_samples(capsys):
    from tensorcore_b200 import paged
    assert paged.main(["--layers", "1", "--slots", "2", "--prompt", "60", "--tokens", "4", "--samples", "3"]) == 0
    out = capsys.readouterr().out
    assert "device error 0" in out and "3 samples" in out
