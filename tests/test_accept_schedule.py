"""The acceptance kernel's source on the CPU (accept_schedule.cpp), its waves in
every order: what it leaves must not depend on which wave is faster.  No GPU."""
import ctypes as C
import itertools
import subprocess
from pathlib import Path

import numpy as np
import pytest

from edgerunner_amd.build import CSRC, ROOT
from test_gpu_accept import Case


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = tmp_path_factory.mktemp("accept") / "libaccept.so"
    subprocess.run(["g++", "-O1", "-fPIC", "-shared", "-std=c++17", "-I", str(ROOT / "include"), "-I", str(CSRC),
                    str(Path(__file__).with_name("accept_schedule.cpp")), "-o", str(out)], check=True)
    return C.CDLL(str(out))


def accept(lib, c, order):
    """(cache, outputs) as Case.state gives them."""
    b, S = c.b, len(c.b.lens)
    cache = [a.copy() for a in c.before]
    out = [np.full(n, -77, np.int32) for n in (b.total, S, S, S)]
    arrays = [*cache, np.ascontiguousarray(b.table), np.array(b.lens, np.int32), b.start, c.parent, c.token, c.chosen, *out]
    pages, heads, P, d = c.before[0].shape
    sizes = (pages, heads, P.bit_length() - 1, d, S, b.stride, b.total, max(1, max(b.rows)), max(b.lens))
    status = lib.accept_in_order((C.c_void_p * len(arrays))(*(a.ctypes.data for a in arrays)), (C.c_uint32 * len(sizes))(*sizes),
                                 (C.c_int * 4)(*order))
    assert status == 0
    return cache, out


ORDERS = list(itertools.permutations(range(4)))


@pytest.mark.parametrize("d,P,heads,lens,rows", [(64, 16, 2, [70, 33, 0, 5], [25, 8, 0, 5]), (128, 32, 1, [150, 40], [70, 9]),
                                                 (256, 64, 1, [130, 66], [60, 66])])
def test_orders(lib, d, P, heads, lens, rows):
    c = Case(None, d + P, lens, rows, P, d, heads, 1.0, behind=2)
    for order in (ORDERS[0], ORDERS[-1], ORDERS[9]):
        c.check(accept(lib, c, order), c.expect())


@pytest.mark.parametrize("gaps", [(4,), (3, 5), (3, 4, 5), (2, 3)])
def test_orders_over_missing_pages(lib, gaps):
    """Pages without a place in the pool among those that kept tokens come to: the ones in front of a gap and behind it share nothing."""
    for seed in range(3):
        c = Case(None, 50 + seed, [130], [110], 16, 64, 1, 1.0, apart=6)
        c.parent[2:110] = np.arange(1, 109)  # all but the row behind the first are kept, each a place lower than it was
        c.parent[1:3] = 0
        c.chosen[:109], c.token[1] = c.token[1:], 2000
        c.chosen[0] = c.token[2]
        for p in gaps:
            c.b.table[0, p] = -1
        exp = c.expect()
        assert exp[1][1][0] == 109
        for order in ORDERS:
            c.check(accept(lib, c, order), exp)


def near_the_largest(seed, P, d, scales, whole=False):
    """Kept drafts whose codes, 208 to 448, stand for values past fp32's largest under some of the pages' scales."""
    c = Case(None, seed, [3 * P + 5], [2 * P + 9], P, d, 1, 1.0)
    n = c.b.rows[0]
    for i in (0, 2):
        big = c.rng.integers(0x75, 0x7f, c.before[i].shape).astype(np.uint8) | (c.rng.integers(0, 2, c.before[i].shape) << 7).astype(np.uint8)
        c.before[i] = big if whole else np.where(c.rng.random(big.shape) < 0.1, big, c.before[i])
        c.before[i + 1][:] = np.float32(2.0) ** c.rng.choice(scales, c.before[i + 1].shape).astype(np.float32)
    c.parent[2:n] = np.arange(1, n - 1)
    c.parent[1:3] = 0
    c.chosen[:n - 1], c.token[1] = c.token[1:n], 2000
    c.chosen[0] = c.token[2]
    return c


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("scales", [[120], [118, 119, 120], [-100, 0, 120]])
def test_values_past_fp32(lib, scales, whole):
    """A finite code under a scale of up to 2^120 moves as what it stands for, although fp32 does not hold that."""
    for seed, P in ((70, 16), (71, 32)):
        c = near_the_largest(seed, P, 64, scales, whole)
        exp = c.expect()
        # the append's rule asks for no larger scale than the codes come from, so none of them is lost
        assert max(float(exp[0][i].max()) for i in (1, 3)) <= 2.0 ** max(scales)
        c.check(accept(lib, c, ORDERS[0]), exp)
