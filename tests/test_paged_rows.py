"""Rows that a step over the paged cache is given: on the GPU, of the step's shape, in any strides."""
import numpy as np
import pytest

from tensorcore_b200 import decode, paged


def test_rows_that_are_not_on_the_gpu_are_refused():
    """Before anything is planned: an address on the host never reaches a kernel."""
    import torch
    d = object.__new__(paged.PagedDecoder)
    d.torch, d.shape, d.book = torch, decode.tiny_shape(), paged.PageBook(4, 16, 1, 4)
    for x in (torch.zeros(3, d.shape.d_model).half(), torch.zeros(3, d.shape.d_model), torch.zeros(2, d.shape.d_model).half()):
        with pytest.raises(ValueError):
            d.step(x, [3])
    assert d.book.lengths.tolist() == [0] and d.book.free_pages() == 4


@pytest.mark.gpu
def test_rows_of_a_wider_matrix(tc, ctx):
    import torch
    shape = decode.tiny_shape()
    d = paged.PagedDecoder(ctx, shape, slots=1, n_pages=4, page_tokens=16)
    x = paged.rows(20, shape.d_model, 1)
    want = d.step(x, [20])
    wide, columns = torch.full((20, 2 * shape.d_model), 7.0, device="cuda").half(), x.t().contiguous().t()
    wide[:, :shape.d_model] = x
    for same in (wide[:, :shape.d_model], columns):
        d.release(0)
        # (a projection's last fp16 places differ from run to run)
        assert ((d.step(same, [20]) - want).float().norm() / (want - x).float().norm()).item() <= 3.0e-2
    assert tc.take_device_error(ctx) == 0
