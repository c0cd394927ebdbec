"""Layers over the paged cache: prompts at once, in pieces and token by token, beside other sequences, in slots used again."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

# Between two ways of taking the same tokens a projection's row differs by roundings to fp16 (2^-11 each way), which turn a code of the
# cache over with a probability of about 2^-11 times (a row's elements in units of a code's step, up to 8): at random a
# change of sqrt(2^-11 * 4) = 4% of a step, a sixth of an element's typical size away at most, so 1% of a key or value.  Two layers, each with the
# same again from its input: 3% of what the layers add, at random over a row's elements.
APART = 3.0e-2


def _apart(got, want, x):
    return ((got - want).float().norm() / (want - x).float().norm()).item()


@pytest.fixture(scope="module")
def shape():
    from tensorcore_b200 import decode as D
    return D.tiny_shape()


@pytest.fixture()
def decoder(tc, ctx, shape):
    from tensorcore_b200 import paged
    return paged.PagedDecoder(ctx, shape, slots=3, n_pages=24, page_tokens=16, max_pages=10, scaling="by_wavelength", factor=4.0, original_context=40.0)


def test_at_once_in_pieces_and_one_by_one(tc, ctx, shape, decoder):
    import torch
    from tensorcore_b200 import paged
    x = [paged.rows(n, shape.d_model, i) for i, n in enumerate((90, 41, 7))]
    at_once = decoder.step(torch.cat(x), [90, 41, 7])
    parts = at_once.split([90, 41, 7])
    for s in range(3):
        decoder.release(s)
    # sequence 0 in pieces beside 1 token by token; 2 waits, then comes at once
    got, a, b = [[], [], []], 0, 0
    for piece in (1, 50, 9, 30):
        y = decoder.step(torch.cat([x[0][a:a + piece], x[1][b:b + 1]]), [piece, 1, 0])
        got[0].append(y[:piece])
        got[1].append(y[piece:])
        a, b = a + piece, b + 1
    for t in range(b, 41):
        n = 7 if t == 20 else 0
        y = decoder.step(torch.cat([x[1][t:t + 1], x[2][:n]]), [0, 1, n])
        got[1].append(y[:1])
        got[2].append(y[1:])
    for s in range(3):
        y = torch.cat(got[s])
        assert torch.isfinite(y).all()
        assert _apart(y, parts[s], x[s]) <= APART
    assert decoder.book.lengths.tolist() == [90, 41, 7]
    assert tc.take_device_error(ctx) == 0


def test_slots_are_used_again(tc, ctx, shape, decoder):
    """What a page held before, and what other sequences hold, has no part in a sequence (projections' last fp16 places differ from run to run)."""
    from tensorcore_b200 import paged
    x = paged.rows(33, shape.d_model, 5)
    first = decoder.step(x, [0, 33, 0])
    decoder.release(1)
    decoder.step(paged.rows(150, shape.d_model, 6), [100, 0, 50])
    decoder.pages[:, decoder.book._free] = 0xFF                          # free pages: NaN scales
    decoder.release(0)
    decoder.release(2)
    assert _apart(decoder.step(x, [0, 33, 0]), first, x) <= APART
    with pytest.raises(paged.OutOfPages):
        decoder.step(paged.rows(161, shape.d_model, 7), [161, 0, 0])
    with pytest.raises(ValueError):
        decoder.step(x, [32, 0, 0])
    assert decoder.book.lengths.tolist() == [0, 33, 0]
    assert tc.take_device_error(ctx) == 0


def test_the_command(capsys):
    from tensorcore_b200 import paged
    assert paged.main(["--layers", "1", "--slots", "2", "--prompt", "60", "--tokens", "3"]) == 0
    assert "device error 0" in capsys.readouterr().out
