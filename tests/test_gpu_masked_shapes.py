"""Attention under masks where the work is cut up otherwise (two blocks of columns a wave, shares across units), where values'
scales lie far apart, and in a pool of more than 2^32 code bytes."""
import ctypes as C

import numpy as np
import pytest

from edgerunner_amd import HeadRows, KV8AcceptKernel, KV8Cache
from test_gpu_accept import Case as AcceptCase
from test_gpu_masked_attention import Case

pytestmark = pytest.mark.gpu


def many(long, few, n=31):
    """One long sequence and many short ones: as many steps as the longest of each would have decide how many columns a wave has."""
    return [long] + [20 + 7 * i % 90 for i in range(n)], [few] + [1 + i % min(few, 19) for i in range(n)]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("d,P,hq,hkv,long,few,masks,window,sinks", [
    # 32 columns a wave; shares of one unit
    (64, 16, 16, 8, 8200, 17, "tree", 0, 0), (64, 32, 8, 8, 8300, 31, "any", 0, 0), (64, 64, 8, 8, 8200, 33, "tree", 900, 5),
    (128, 16, 16, 8, 8200, 20, "any", 3000, 70), (128, 32, 8, 8, 8200, 17, None, 5000, 4), (128, 64, 16, 8, 8300, 16, "tree", 0, 0),
    # and across units
    (64, 16, 16, 8, 12000, 64, "tree", 0, 0), (128, 16, 8, 8, 12100, 128, None, 9000, 65), (128, 64, 16, 8, 12000, 61, "any", 0, 0),
    (64, 64, 24, 8, 14000, 40, "tree", 11000, 130)])
def test_two_blocks_a_wave(ctx, d, P, hq, hkv, long, few, masks, window, sinks, half):
    c = Case(ctx, d + P + few, *many(long, few), P, d, hq, hkv, masks, behind=1)
    c.check(c.run(half, window, sinks), half, window, sinks)


@pytest.mark.parametrize("d,P,hq,hkv,lens,rows,masks", [
    (256, 64, 8, 2, [4000, 2000, 70, 900, 1], [60, 64, 9, 33, 1], "tree"), (256, 16, 16, 4, [2300, 1500, 900, 63], [60, 64, 2, 63], None),
    (64, 64, 8, 8, [40000, 9000, 777], [3, 4, 1], "any")])
def test_shared_across_units(ctx, d, P, hq, hkv, lens, rows, masks):
    c = Case(ctx, d + P, lens, rows, P, d, hq, hkv, masks)
    c.check(c.run())


@pytest.mark.parametrize("d,P,hq,hkv,most,masks,window,sinks", [
    (64, 16, 8, 4, 1900, "tree", 0, 0), (128, 32, 8, 8, 1500, None, 700, 70), (64, 64, 16, 8, 2048, "any", 0, 0),
    (128, 16, 8, 4, 1100, "tree", 200, 1), (128, 64, 4, 4, 5000, None, 900, 4), (64, 32, 24, 4, 2500, "tree", 0, 0)])
def test_a_workgroup_a_unit(ctx, d, P, hq, hkv, most, masks, window, sinks):
    """Many units of middling length, or of long caches under a window, each one workgroup's: no workspace where none is long."""
    rng = np.random.default_rng(most)
    lens = [most, 0, 1] + [int(x) for x in rng.integers(1, min(most, 1200), 37)]
    rows = [min(m, int(x)) for m, x in zip(lens, rng.integers(0, 7, 40))]
    c = Case(ctx, d + P, lens, rows, P, d, hq, hkv, masks)
    c.check(c.run(window=window, sinks=sinks), window=window, sinks=sinks)
    if most <= 2500:
        assert c.kern.lib.er_hip_kv8_attention_masked_workspace(ctx.handle, c.cache.ref, c.b.upload(ctx).ref, hq,
                                                                C.byref(n := C.c_uint64(1))) == 0 and n.value == 0


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("ratio", [30, 70])
@pytest.mark.parametrize("every,first", [(3, 0), (3, 2), (9, 8)])
@pytest.mark.parametrize("d,P,hq,hkv,lens,rows,masks,window,sinks", [
    (64, 16, 2, 1, [52, 37], [18, 10], "any", 0, 0), (128, 16, 4, 2, [150, 77], [8, 6], "tree", 20, 3),
    (256, 16, 2, 1, [150, 90], [40, 7], "any", 12, 20), (128, 32, 2, 1, [210, 100], [30, 9], None, 40, 5),
    (64, 64, 2, 2, [420, 260], [30, 25], "tree", 70, 70), (64, 16, 4, 2, [1700, 90], [24, 5], "any", 25, 2),
    (64, 16, 4, 2, [150, 77], [90, 40], "any", 0, 0), (128, 16, 4, 2, [170, 150], [130, 33], "tree", 20, 18),
    (64, 16, 2, 1, [1500], [400], "tree", 24, 33), (128, 16, 8, 8, *many(8200, 18), "any", 30, 17)])
def test_scales_of_hidden_values(ctx, d, P, hq, hkv, lens, rows, masks, window, sinks, every, first, ratio, half):
    """Some pages have values 2^ratio times the others'.  A row that sees none of them is held to the bound of its own values,
    whatever rows it shares a tile with."""
    c = Case(ctx, d + P + ratio, lens, rows, P, d, hq, hkv, masks)
    for s in range(len(lens)):
        for p in range(c.b.stride):
            if c.b.table[s, p] >= 0:
                c.vs[c.b.table[s, p]] = 2.0 ** (ratio - 5 if p % every == first else p % 4 - 6)
    c.check(c.run(half, window, sinks), half, window, sinks)


class Far:
    """The pages of a small case's one sequence as the last ones of a large pool."""

    def __init__(self, ctx, table, arrays):
        heads, P, d = arrays[0].shape[1:]
        self.pages = pages = (1 << 32) // (P * d * heads) + 40
        self.bufs = [ctx.alloc(n) for n in (pages * heads * P * d, 4 * pages * heads) * 2]
        self.cache = KV8Cache(self.bufs[0], self.bufs[2], self.bufs[1], self.bufs[3], pages, heads, P, d)
        self.far = [pages - 1 - 6 * i % 13 for i in range(len(table))]
        self.sizes = [heads * P * d, 4 * heads] * 2
        for to, src in zip(self.far, table):
            for b, a, size in zip(self.bufs, arrays, self.sizes):
                b.upload(np.ascontiguousarray(a[src]), to * size)

    def download(self, arrays):
        return [[b.download(a.dtype, size // a.dtype.itemsize, to * size).reshape(a.shape[1:]) for to in self.far]
                for b, a, size in zip(self.bufs, arrays, self.sizes)]

    def free(self):
        for b in self.bufs:
            b.free()


@pytest.mark.parametrize("rows,masks", [(1, None), (30, "tree"), (100, "any")])
def test_attention_beyond_32_bits(ctx, rows, masks):
    c = Case(ctx, 18, [150], [rows], 64, 256, 4, 2, masks)
    c.upload()
    far = Far(ctx, c.b.table[0], (c.kc, c.ks, c.vc, c.vs))
    batch = c.b.upload(ctx)
    c.b.bufs[0].upload(np.array(far.far, np.int32))
    ob = ctx.upload(np.full(c.q.shape, 7, np.float32))
    c.cache = far.cache
    c.encode(HeadRows(ob, 4, 4 * 256), c.scratch(batch), batch, False, 60, 3)
    ctx.synchronize()
    c.raw, c.fill = ob.download(np.float32).reshape(c.q.shape), np.float32(7)
    c.check(c.raw.astype(np.float64), window=60, sinks=3)
    far.free()


def test_acceptance_beyond_32_bits(ctx):
    c = AcceptCase(ctx, 19, [150], [64], 64, 256, 2, luck=1.0)
    c.upload()
    far = Far(ctx, c.b.table[0], c.before)
    batch = c.b.upload(ctx)
    c.b.bufs[0].upload(np.array(far.far, np.int32))
    KV8AcceptKernel(ctx).encode(None, far.cache, batch, c.drafts, c.tree[2], *c.out)
    ctx.synchronize()
    exp = c.expect()
    got = [a.copy() for a in c.before]
    for a, pages in zip(got, far.download(c.before)):
        a[c.b.table[0]] = pages
    c.check((got, [x.download(np.int32) for x in c.out]), exp)
    far.free()


def test_two_streams_with_their_own_workspaces(ctx):
    """Two calls under way at once, of one cache and of two kernels' kinds."""
    a = Case(ctx, 20, *many(8200, 20), 16, 64, 16, 8, "tree")
    b = Case(ctx, 21, [5000, 900], [90, 100], 64, 64, 8, 2, "any")
    streams = [ctx.stream(), ctx.stream()]
    work = []
    for c in (a, b):
        c.upload()
        batch = c.b.upload(ctx)
        out = ctx.upload(np.full((c.b.total, c.hq * 64), 7, np.float32))
        work.append((HeadRows(out, c.hq, c.hq * 64), c.scratch(batch), batch, out))
    ctx.synchronize()
    for _ in range(3):
        for c, w, st in zip((a, b), work, streams):
            c.encode(w[0], w[1], w[2], False, 0, 0, st)
    for st in streams:
        st.synchronize()
    for c, w in zip((a, b), work):
        c.raw, c.fill = w[3].download(np.float32).reshape(c.b.total, c.hq, 64), np.float32(7)
        c.check(c.raw.astype(np.float64))
    for st in streams:
        st.destroy()
