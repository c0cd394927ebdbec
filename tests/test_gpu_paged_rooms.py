"""Attention over pages beside attention over plain K and V on the same stream: what the one leaves in its scratch is nothing that the other
takes for sums handed over."""
import ctypes

import numpy as np
import pytest

from test_gpu_attention_paged import Case

pytestmark = pytest.mark.gpu

# Dense decode shapes whose handed-over sums take 1.4 to 1.9 MB: more than 148 CTAs of the paged kernel hand over (1.2 MB at most), so a
# room that held anything else behind those would show.
DENSE = [(4, 4, 32, 8, 4096), (4, 3, 32, 8, 4096), (6, 1, 256, 16, 2338)]
D = 128


class Dense:
    def __init__(self, tc, B, Sq, H, Hkv, Sk):
        import torch
        g = torch.Generator(device="cuda").manual_seed(B + Sq)
        self.q, self.k, self.v = (torch.randn(B, h, s, D, device="cuda", generator=g).half() for h, s in ((H, Sq), (Hkv, Sk), (Hkv, Sk)))
        self.shape, self.o = (B, H, Sq, Sk), torch.zeros_like(self.q)
        self.lse = torch.zeros(B, H, Sq, device="cuda")
        self.desc = tc.TCAttentionDesc(B, H, Sq, Sk, D, tc.TC_DTYPE_F16, tc.TC_DTYPE_F32, 0.0, False, True, Hkv, 0, None)

    def call(self, tc, ctx, stream):
        rc = tc.lib().tcx_raw_attention_forward(ctx.handle, ctypes.byref(self.desc), *(ctypes.c_void_p(t.data_ptr()) for t in (self.q, self.k, self.v, self.o, self.lse)),
                                                ctypes.c_void_p(stream))
        assert rc == 0

    def take(self):
        import torch
        torch.cuda.synchronize()
        got = self.o.clone(), self.lse.clone()
        self.o.fill_(3.0)
        self.lse.fill_(3.0)
        torch.cuda.synchronize()
        return got


class Paged:
    """A ragged batch: sequences whose keys many warps share, so that each CTA's warps leave pieces."""

    def __init__(self, tc, queries):
        import torch
        self.c = c = Case(tc, [3000, 1, 2048, 700, 0, 3500, 64, 1999], [queries] * 8, 32, 8, D, 64, seed=queries)
        cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
        self.table, self.lens, self.start = cuda(c.table), cuda(np.array(c.keys, np.int32)), cuda(c.start)
        self.o, self.lse = torch.zeros_like(c.q), torch.zeros(len(c.q), 32, device="cuda")
        self.desc = tc.attention_paged_desc(len(c.q), 8, c.table.shape[1], 32, max_q=queries)

    def call(self, tc, ctx, stream):
        tc.raw_attention_paged(ctx, self.c.kv, self.desc, self.c.pages.data_ptr(), self.c.q.data_ptr(), self.table.data_ptr(), self.lens.data_ptr(), self.start.data_ptr(),
                               self.o.data_ptr(), self.lse.data_ptr(), stream)


def _same(a, b):
    import torch
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("queries", [1, 4])
@pytest.mark.parametrize("shape", DENSE)
def test_dense_attention_after_paged(tc, ctx, shape, queries):
    """In turn on one stream, eagerly and in a captured graph: the bits that each gives alone."""
    import torch
    d, p = Dense(tc, *shape), Paged(tc, queries)
    torch.cuda.synchronize()
    d.call(tc, ctx, torch.cuda.Stream().cuda_stream)
    want = d.take()
    p.call(tc, ctx, torch.cuda.Stream().cuda_stream)
    torch.cuda.synchronize()
    paged = p.o.clone(), p.lse.clone()
    st = torch.cuda.Stream()
    for _ in range(4):
        p.call(tc, ctx, st.cuda_stream)
        d.call(tc, ctx, st.cuda_stream)
        assert _same(d.take(), want) and _same((p.o, p.lse), paged)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        for _ in range(2):
            p.call(tc, ctx, st.cuda_stream)
            d.call(tc, ctx, st.cuda_stream)
    for _ in range(3):
        graph.replay()
        assert _same(d.take(), want) and _same((p.o, p.lse), paged)
    del graph
    assert tc.take_device_error(ctx) == 0


def test_on_buffers(tc, ctx):
    """The synchronous forms, which share a stream of the context."""
    d, p = Dense(tc, *DENSE[0]), Paged(tc, 1)
    B, H, Sq, Sk = d.shape
    q, k, v = (ctx.buffer_from_array(t.cpu().numpy()) for t in (d.q, d.k, d.v))
    o = ctx.buffer(d.q.numel() * 2)
    c = p.c
    pq, pages = ctx.buffer_from_array(c.q.cpu().numpy()), ctx.buffer_from_array(c.pages.cpu().numpy())
    t, l, b = (ctx.buffer_from_array(np.array(a, np.int32)) for a in (c.table, c.keys, c.start))
    po = ctx.buffer(c.q.numel() * 2)
    d.call(tc, ctx, 0)
    want = d.take()[0].cpu().numpy()
    for _ in range(3):
        tc.attention_paged(ctx, c.kv, p.desc, pages, pq, t, l, b, po)
        tc.attention_forward(ctx, q, k, v, o, B, H, Sq, Sk, D, causal=False, kv_heads=8)
        assert np.array_equal(o.to_numpy(want.shape, np.float16), want)
    assert tc.take_device_error(ctx) == 0


def test_scratch_of_a_closed_stream(tc, ctx):
    """A stream that is opened later takes over the scratch of one that was closed."""
    import torch
    d, p = Dense(tc, *DENSE[0]), Paged(tc, 1)
    torch.cuda.synchronize()
    d.call(tc, ctx, torch.cuda.Stream().cuda_stream)
    want = d.take()
    for _ in range(3):
        with tc.Stream(ctx) as s:
            p.call(tc, ctx, s.cuda_handle())
            torch.cuda.synchronize()
        with tc.Stream(ctx) as s:
            for _ in range(2):
                d.call(tc, ctx, s.cuda_handle())
                assert _same(d.take(), want)
    assert tc.take_device_error(ctx) == 0
