"""Where the operators between the projections could lose bits, against 64-bit forms."""
import pytest

from test_gpu_kv8_attention import Case

pytestmark = pytest.mark.gpu


def page_scales(c, exponent):
    """Gives page p of each sequence the value scale 2^exponent(p)."""
    for s in range(len(c.b.lens)):
        for p in range(c.b.stride):
            if c.b.table[s, p] >= 0:
                c.vs[c.b.table[s, p]] = 2.0 ** exponent(p)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("ratio", [30, 70])
@pytest.mark.parametrize("every,first", [(3, 0), (3, 1), (3, 2), (9, 2), (9, 8)])
@pytest.mark.parametrize("d,P,hq,hkv,lens,rows,window", [
    # 16 columns at a time: a later row's page in the tile of an earlier one; pages before a window
    (64, 16, 2, 1, [52, 37], [18, 10], 0), (128, 16, 4, 2, [150, 77], [8, 6], 20), (256, 16, 2, 1, [150, 90], [40, 7], 12),
    (128, 32, 2, 1, [210, 100], [30, 9], 40), (64, 64, 2, 2, [420, 260], [30, 25], 70), (256, 64, 4, 2, [300], [60], 33),
    (64, 16, 4, 2, [1700, 90], [24, 5], 25), (128, 32, 2, 1, [2100, 700], [40, 40], 36), (64, 16, 2, 2, [300, 287], [16, 13], 116),
    (128, 16, 3, 3, [1300, 1287], [15, 13], 122),
    # 128 columns at a time, in one piece and in several
    (64, 16, 4, 2, [150, 77], [90, 40], 0), (128, 16, 4, 2, [170, 150], [130, 33], 20), (256, 16, 8, 1, [180], [150], 18),
    (128, 32, 2, 1, [300, 130], [200, 130], 40), (128, 64, 2, 1, [400, 130], [300, 130], 70), (64, 16, 2, 1, [1500], [400], 24)])
def test_scales_of_hidden_values(ctx, d, P, hq, hkv, lens, rows, window, every, first, ratio, half):
    """Some pages have values 2^ratio times the others'.  A row that sees none of them is held to the bound of its own
    values, whatever rows it shares a tile with."""
    c = Case(ctx, d + P + ratio, lens, rows, P, d, hq, hkv)
    page_scales(c, lambda p: ratio - 5 if p % every == first else p % 4 - 6)
    c.check(c.run(half, window), half, window)
