"""Rules on logits where the kernel and what joins a row's slices change: vocabularies around one slice of 2048 tokens,
rows of more than 64 slices, of which a lane of the join takes several, and choices beside values that are not finite."""
import numpy as np
import pytest

from test_gpu_choose import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 130])
@pytest.mark.parametrize("vocab", [2045, 2047, 2048, 2049, 2050, 2051, 4096])
def test_around_one_slice(ctx, vocab, rows):
    Case(ctx, vocab + rows, vocab, [1] * rows, past=100, bias=20, allowed=True).run()


@pytest.mark.parametrize("vocab", [64 * 2048, 64 * 2048 + 1, 130 * 2048 + 5])
def test_more_than_64_slices(ctx, vocab):
    """The largest in each part of the row, and twice, in slices that one lane takes and that several do: the lowest token counts."""
    places = [(vocab - 1,), (5, 64 * 2048 - 1), (3000, vocab - 1), (65 * 2048, 2048) if vocab > 66 * 2048 else (2048,),
              (129 * 2048 + 7, 65 * 2048 + 7) if vocab > 130 * 2048 else (63 * 2048 + 7,), (vocab - 2, vocab - 1)]
    c = Case(ctx, vocab, vocab, [1] * len(places))
    for r, at in enumerate(places):
        c.x[r, list(at)] = 40.0
    c.run()
    assert list(c.cb.download(np.int32)) == [min(at) for at in places]


def test_choices_beside_infinities(ctx):
    """A row of -inf behind its first tokens, some of them NaN: what is chosen is the largest allowed one that is left, and where
    only -inf is allowed the lowest of those."""
    c = Case(ctx, 12, 2000, [1] * 4, allowed=True)
    c.x[:, 5:] = -np.inf
    c.x[:, :5] = [np.nan, 2.0, 3.0, np.nan, 1.0]
    c.allowed[:] = True
    c.allowed[1, 2] = False
    c.allowed[2, :9] = False
    c.allowed[3] = False
    c.allowed[3, [0, 3]] = True
    c.run()
    assert list(c.cb.download(np.int32)) == [2, 1, 9, -1]
