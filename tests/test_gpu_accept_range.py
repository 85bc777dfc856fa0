"""Acceptance of drafts at the ends of its range: values next to fp32's largest,
and pages that are missing in front of ones that are there."""
import pytest

from test_accept_schedule import near_the_largest
from test_gpu_accept import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("scales", [[120], [118, 119, 120], [-100, 0, 120]])
@pytest.mark.parametrize("d,P", [(64, 16), (64, 64), (128, 32), (256, 16)])
def test_values_past_fp32(ctx, d, P, scales, whole):
    c = near_the_largest(70 + d, P, d, scales, whole)
    c.ctx = ctx
    c.check(c.run(), c.expect())


@pytest.mark.parametrize("d,P,heads", [(64, 16, 2), (128, 16, 1), (256, 32, 2), (64, 64, 1)])
def test_pages_around_gaps(ctx, d, P, heads):
    """Every other page of the drafts' places has none in the pool."""
    for odd in (0, 1):
        c = Case(ctx, d + P + odd, [11 * P - 3, 6 * P], [9 * P, 5 * P], P, d, heads, 1.0, chain=True)
        for s, n in enumerate(c.b.rows):
            at = c.b.start[s]
            line = [0] + [r for r in range(2, n)]
            for a, r in zip(line, line[1:]):
                c.parent[at + r], c.chosen[at + a] = a, c.token[at + r]
            c.parent[at + 1] = -1
            c.b.table[s, 1 + odd::2] = -1
        exp = c.expect()
        assert list(exp[1][1]) == [9 * P - 1, 5 * P - 1]
        c.check(c.run(), exp)
