"""Where the operators between the projections could lose bits: value scales of
tokens that a row does not see, weights far below a row's largest, rotation
angles, head norms of very large and very small heads, values near fp32's
largest.  All against 64-bit forms."""
import numpy as np
import pytest

import kv8_ref as R
from edgerunner_amd import HeadRows, KV8AttentionKernel, KV8Batch, KV8Cache, QKNormRopeKernel, Rope
from test_gpu_kv8_append import Case as AppendCase, freqs, turn_tol
from test_gpu_kv8_attention import LONE, Case

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


@pytest.mark.parametrize("down", [20, 22])
@pytest.mark.parametrize("d,P,hq,hkv,lens,rows", [
    (64, 16, 4, 2, [400, 300], [1, 1]), (128, 32, 4, 2, [500], [5]), (256, 64, 2, 1, [700, 90], [3, 2]),
    (64, 16, 4, 2, [400, 300], [70, 30]), (128, 64, 4, 1, [600], [100]), (256, 32, 2, 1, [350], [200])])
def test_codes_below_the_largest_scale(ctx, d, P, hq, hkv, lens, rows, down):
    """A block of values whose scale is 2^-22 of the largest that a row sees keeps its codes whole, subnormal ones too: the pages
    of the large scale have values in element 0 alone, so the other elements are held to the small ones' own bound."""
    c = Case(ctx, d + down, lens, rows, P, d, hq, hkv)
    page_scales(c, lambda p: 10 if p % 4 == 1 else 10 - down)
    for s in range(len(lens)):
        for p in range(c.b.stride):
            page = c.b.table[s, p]
            if page >= 0 and p % 4 == 1:
                c.vc[page, ..., 1:] = 0
            elif page >= 0:  # the smallest codes, whose last bit is the one at stake
                keep = (c.vc[page] & 0x7f) == 0x7f
                c.vc[page] = np.where(keep, c.vc[page], c.vc[page] & 0x87)
    c.check(c.run())


# Weights are held as two fp16 terms of up to 2^15 for the largest of a row and 2^13 at the least, so one of 2^-33 of the
# largest is 2^-20 there at the least, off by at most half of fp16's smallest step, 2^-25
@pytest.mark.parametrize("seqs,rows", [(512, 1), (800, 80)])
def test_long_tail_of_small_weights(ctx, seqs, rows):
    """Four tokens with a score 33 powers of two above those of 2^18 others, whose values make up the whole output."""
    d, P, n = 64, 64, 1 << 18
    kc, vc = np.zeros((2, 1, P, d), np.uint8), np.full((2, 1, P, d), 0x38, np.uint8)  # 0x38: 1
    kc[..., 0] = 0xb8  # -1
    for t in (0, 32):
        kc[0, 0, t], vc[0, 0, t] = 0, 0
    table = np.ones((seqs, n // P), np.int32)
    table[:, :2] = 0
    total = seqs * rows
    q = np.zeros((total, d), np.float32)
    q[:, 0] = 33
    ones = np.ones((2, 1), np.float32)
    cache = KV8Cache(*[ctx.upload(a) for a in (kc, vc, ones, ones)], 2, 1, P, d)
    batch = KV8Batch(ctx.upload(table), ctx.upload(np.full(seqs, n, np.int32)),
                     ctx.upload(np.arange(seqs + 1, dtype=np.int32) * rows), seqs, n // P, total, rows, n)
    kern = KV8AttentionKernel(ctx)
    ws = ctx.alloc(max(16, kern.workspaceBytes(cache, batch, 1)))
    ob = ctx.alloc(4 * q.size)
    kern.encode(None, cache, batch, HeadRows(ctx.upload(q), 1, d), HeadRows(ob, 1, d), float(np.log(2.0)), workspace=ws)
    ctx.synchronize()
    got = ob.download(np.float32).reshape(seqs, rows, d)
    tail = (n - rows + np.arange(rows) + 1 - 4) * 2.0 ** -33
    exp = (tail / (4 + tail))[None, :, None]
    # beside the terms: 33 * 2^-23 of the exponent, and sums of fp32
    assert np.all(np.abs(got - exp) <= exp * (2.0 ** -5 + 2.0 ** -8))


@pytest.mark.parametrize("pairs", [False, True])
def test_rotation_angles(ctx, pairs):
    """cos and sin of far positions as the rotation uses them.  The angle, at most a quarter turn's half, is rounded once from
    64 bits (2^-25, times 0.71 for a cosine and 0.76 for a sine of that size); the series adds 2.7e-8 and 1.9e-8 to it, and
    the result is rounded once (2^-25): at most 8.1e-8."""
    d, rows = 128, 20000
    rng = np.random.default_rng(3)
    x = np.zeros((rows, d), np.float32)
    a = np.arange(0, d, 2) if pairs else np.arange(d // 2)
    x[:, a] = 1
    pos = rng.integers(0, 1 << 20, rows).astype(np.int32)
    f = freqs(d)
    xb = ctx.upload(x)
    h = HeadRows(xb, 1, d)
    QKNormRopeKernel(ctx).encode(None, h, None, h, None, ctx.upload(pos), rows, d, Rope(ctx.upload(f), d, pairs))
    ctx.synchronize()
    got = xb.download(np.float32).reshape(rows, d)
    exp = R.norm_rope(x[:, None], pos, f, d, pairs)[:, 0]
    assert np.abs(got - exp).max() <= 8.1e-8


@pytest.mark.parametrize("d,power,eps", [(64, 70, 1e-6), (128, 120, 1e-6), (256, 100, 1e-5), (64, -80, 0.0), (128, -120, 0.0),
                                         (256, -40, 1e-30), (128, -141, 0.0)])
def test_norms_of_large_and_small_heads(ctx, d, power, eps):
    """Heads whose squares pass fp32's range at either end are normed as the others, alone and on the way of an append."""
    rng = np.random.default_rng(d + abs(power))
    rows, hq, hk = 7, 5, 3
    x = rng.standard_normal((rows, hq + hk, d)).astype(np.float32)
    x[::2, ::2] = np.clip(x[::2, ::2], -3, 3) * np.float32(2.0 ** max(power, -126)) * np.float32(2.0 ** min(power + 126, 0))
    pos, w, f = rng.integers(0, 9000, rows).astype(np.int32), (rng.random(d) + 0.5).astype(np.float32), freqs(d)
    xb, wb, fb, pb = ctx.upload(x), ctx.upload(w), ctx.upload(f), ctx.upload(pos)
    width = (hq + hk) * d
    q, k = HeadRows(xb, hq, width), HeadRows(xb.view(4 * hq * d), hk, width)
    QKNormRopeKernel(ctx).encode(None, q, k, q, k, pb, rows, d, Rope(fb, d), wb, wb, eps)
    ctx.synchronize()
    got = xb.download(np.float32).reshape(x.shape)
    assert np.all(np.abs(got - R.norm_rope(x, pos, f, d, False, w, eps)) <= turn_tol(x, d, False, w, eps))
    c = AppendCase(ctx, rng, [rows], [rows], 16, d, hk, norm=True, hq=hq)
    c.q, c.w = x[:, :hq].copy(), w
    c.run(eps=eps)
    got = c.io[3].download(np.float32).reshape(c.q.shape)
    exp = R.norm_rope(c.q, np.arange(rows), c.f, d, False, w, eps)
    assert np.all(np.abs(got - exp) <= turn_tol(c.q, d, False, w, eps))


@pytest.mark.parametrize("lens,rows,hq,hkv", [([1], [1], 2, 1), ([40, 3], [1, 1], 4, 2), ([2000], [3], 2, 1), ([90], [70], 2, 1),
                                              ([1500], [80], 2, 1), ([50000], [1], 1, 1)])
def test_values_near_the_largest(ctx, lens, rows, hq, hkv):
    """Values of up to 240 * 2^120, next to fp32's largest: a mean of them is no larger, however many there are."""
    c = Case(ctx, 21, lens, rows, 32, 64, hq, hkv)
    nan = (c.vc & 0x7f) == 0x7f
    c.vc = np.where(nan, c.vc, 0x70 + (c.vc & 7)).astype(np.uint8)  # 128 .. 240
    c.vs[:] = np.where(np.isnan(c.vs), c.vs, 2.0 ** 120)
    if lens == [1]:
        got = c.run()
        exp = R.VALUES[c.vc[c.b.table[0, 0], 0, 0]] * 2.0 ** 120
        assert np.all(np.abs(got[0] - exp) <= LONE * exp)
    c.check(c.run())
