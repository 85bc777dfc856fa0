"""The operators between the projections run as a program runs them: Q8_0 q/k/v
projections, append with the queries riding along, attention, and the output
projection, for ragged prompts and then for decode steps replayed from one
recorded graph while the sequences grow.  Each stage is held against a 64-bit
form of what the stage before it left on the device."""
import numpy as np
import pytest

import edgerunner_amd.synth as synth
import kv8_ref as R
from conftest import rel_l2
from edgerunner_amd import (Capture, FusedQ8Kernel, GEMVKernel, HeadRows, KV8AppendKernel, KV8AttentionKernel, KV8Batch,
                            KV8Cache, QuantGEMMKernel, Rope)
from oracle import ref

pytestmark = pytest.mark.gpu

HID, HQ, HKV, D, P, EPS = 256, 4, 2, 64, 16, 1e-6


def weights(seed, rows, cols):
    W = synth.q8_0(synth.seed(70, seed), rows, cols, dscale=0.01)
    return W, ref.dequant("q8_0", W).astype(np.float64).reshape(rows, cols)


class Layer:
    def __init__(self, ctx):
        self.ctx = ctx
        self.W = {n: weights(i, r, c) for i, (n, r, c) in enumerate(
            (("q", HQ * D, HID), ("k", HKV * D, HID), ("v", HKV * D, HID), ("o", HID, HQ * D)))}
        self.w = {n: ctx.upload(W) for n, (W, _) in self.W.items()}
        rng = np.random.default_rng(3)
        self.norm, self.qw, self.kw = [(rng.random(n) + 0.5).astype(np.float32) for n in (HID, D, D)]
        self.freq = (10000.0 ** (-np.arange(0, D, 2) / D)).astype(np.float32)
        self.nb, self.qwb, self.kwb, self.fb = [ctx.upload(a) for a in (self.norm, self.qw, self.kw, self.freq)]
        self.rope = Rope(self.fb, D)
        self.fused, self.gemv, self.gemm = FusedQ8Kernel(ctx), GEMVKernel(ctx), QuantGEMMKernel(ctx)
        self.append, self.attend = KV8AppendKernel(ctx), KV8AttentionKernel(ctx)
        self.cache = KV8Cache.alloc(ctx, 40, HKV, P, D)

    def buffers(self, T, half):
        a = self.ctx.alloc
        return {"x": a(4 * T * HID), "q": a(4 * T * HQ * D), "k": a(4 * T * HKV * D), "v": a((2 if half else 4) * T * HKV * D),
                "a": a((2 if T > 16 else 4) * T * HQ * D), "y": a(4 * T * HID)}

    def encode(self, st, b, batch, T, half, ws):
        qkv = self.fused.encodeFusedQKV if half else self.fused.encodeFusedQKVTurbo
        qkv(st, self.w["q"], self.w["k"], self.w["v"], b["x"], b["q"], b["k"], b["v"], self.nb, HQ * D, HKV * D, HID, T, EPS)
        q = HeadRows(b["q"], HQ, HQ * D)
        self.append.encode(st, self.cache, batch, HeadRows(b["k"], HKV, HKV * D), HeadRows(b["v"], HKV, HKV * D), self.rope,
                           kNorm=self.kwb, q=q, qOut=q, qNorm=self.qwb, eps=EPS, vHalf=half)
        prompt = T > 16
        self.attend.encode(st, self.cache, batch, q, HeadRows(b["a"], HQ, HQ * D), D ** -0.5, workspace=ws, outBF16=prompt)
        if prompt:  # the prefill GEMM takes the attention's bf16 rows as they are
            self.gemm.encodeQ8_0(st, self.w["o"], b["a"], b["y"], T, HID, HQ * D)
        else:
            self.gemv.encodeBatchedQ8_0Weights(st, self.w["o"], b["a"], b["y"], T, HID, HQ * D)
        return q

    def snapshot(self):
        c = self.cache
        shape = (40, HKV, P, D)
        k, v, ks, vs = c.buffers
        return (k.download(np.uint8).reshape(shape), ks.download(np.float32).reshape(shape[:2]),
                v.download(np.uint8).reshape(shape), vs.download(np.float32).reshape(shape[:2]))

    def check(self, x, b, R_batch, T, half, before):
        n = x.astype(np.float64)
        n = n / np.sqrt((n * n).mean(1, keepdims=True) + EPS) * self.norm
        k = b["k"].download(np.float32).reshape(T, HKV, D)
        v = b["v"].download(np.float16 if half else np.float32).reshape(T, HKV, D)
        assert rel_l2(k.reshape(T, -1), n @ self.W["k"][1].T) < 1e-5
        assert rel_l2(v.reshape(T, -1).astype(np.float64), n @ self.W["v"][1].T) < (1e-3 if half else 1e-5)
        pos = np.concatenate([np.arange(m - r, m) for r, m in zip(R_batch.rows, R_batch.lens)])
        q = b["q"].download(np.float32).reshape(T, HQ, D)
        # the queries were turned in place, so they are held against the projection's 64-bit form
        eq = R.norm_rope((n @ self.W["q"][1].T).reshape(T, HQ, D), pos, self.freq, D, False, self.qw, EPS)
        assert rel_l2(q, eq) < 1e-5
        after = self.snapshot()
        ek = R.append(before[0], before[1], R_batch, R.norm_rope(k, pos, self.freq, D, False, self.kw, EPS))
        ev = R.append(before[2], before[3], R_batch, v.astype(np.float64))
        for got, exp in zip(after, (*ek, *ev)):
            assert np.array_equal(got, exp, equal_nan=True)
        prompt = T > 16
        raw = b["a"].download(np.uint16 if prompt else np.float32).reshape(T, HQ, D)
        a = R.bf16_to_f32(raw) if prompt else raw
        exp, tol = R.attend(*after, R_batch, q, D ** -0.5, 0, prompt)
        assert np.all(np.abs(a - exp) <= tol)
        y = b["y"].download(np.float32).reshape(T, HID)
        assert rel_l2(y, a.reshape(T, -1).astype(np.float64) @ self.W["o"][1].T) < (5e-3 if prompt else 1e-5)


def test_prompts_then_replayed_decode_steps(ctx):
    rng = np.random.default_rng(1)
    layer = Layer(ctx)
    pages = rng.permutation(40)
    table = np.full((3, 12), -1, np.int32)
    table[0, :12], table[2, :12] = pages[:12], pages[12:24]  # sequence 1 is an unused slot
    tb = ctx.upload(table)

    def described(lens, rows):
        b = R.Batch(rng, [0] * 3, [0] * 3, P)
        b.table, b.lens, b.rows, b.stride = table, lens, rows, 12
        b.start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        b.total = int(b.start[-1])
        return b

    lens, rows = [23, 0, 61], [23, 0, 61]
    T = sum(rows)
    d = described(lens, rows)
    batch = KV8Batch(tb, ctx.upload(np.array(lens, np.int32)), ctx.upload(d.start), 3, 12, T, max(rows), max(lens))
    b = layer.buffers(T, False)
    x = synth.normal_f32(synth.seed(71, 1), T * HID).reshape(T, HID)
    b["x"].upload(x)
    ws = ctx.alloc(max(16, layer.attend.workspaceBytes(layer.cache, batch, HQ)))
    for buf in layer.cache.buffers:  # a pool that no one has used reads as anything: zeros here, for the comparison
        buf.upload(np.zeros(buf.length, np.uint8))
    before = layer.snapshot()
    layer.encode(None, b, batch, T, False, ws)
    ctx.synchronize()
    layer.check(x, b, d, T, False, before)

    # decode: two rows, lengths kept on the device, one graph for every step
    lb = ctx.upload(np.array(lens, np.int32))
    start = ctx.upload(np.array([0, 1, 1, 2], np.int32))
    step = KV8Batch(tb, lb, start, 3, 12, 2, 1, 12 * P)
    db = layer.buffers(2, True)
    ws2 = ctx.alloc(max(16, layer.attend.workspaceBytes(layer.cache, step, HQ)))
    st = ctx.stream()
    with Capture(ctx, st) as cap:
        layer.encode(st, db, step, 2, True, ws2)
    for i in range(4):
        lens = [lens[0] + 1, 0, lens[2] + 1]
        lb.upload(np.array(lens, np.int32))
        x = synth.normal_f32(synth.seed(71, 2 + i), 2 * HID).reshape(2, HID)
        db["x"].upload(x)
        before = layer.snapshot()
        cap.graph.launch(st)
        st.synchronize()
        layer.check(x, db, described(lens, [1, 0, 1]), 2, True, before)
    cap.graph.destroy()
    st.destroy()
