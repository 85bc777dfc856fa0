"""A step that checks trees of drafted tokens run as a program runs it, recorded
once and replayed: norms and rotations at the drafts' positions, append,
attention over the tree, output projection, LM head, rules on the logits with
the choice, acceptance.  Each stage is held against a 64-bit form of what the
stage before it left on the device, and the walks go on from the cache that
the last ones left."""
import numpy as np
import pytest

import draft_ref as D
import edgerunner_amd.synth as synth
import kv8_ref as R
from conftest import rel_l2
from edgerunner_amd import (Capture, Drafts, FusedQ8Kernel, GEMVKernel, HeadRows, KV8AcceptKernel, KV8AppendKernel,
                            KV8AttentionKernel, KV8Batch, KV8Cache, LogitChoiceKernel, LogitRules, QKNormRopeKernel, Rope)
from oracle import ref

pytestmark = pytest.mark.gpu

HID, HQ, HKV, W, P, V, EPS, PAGES = 256, 4, 2, 64, 16, 512, 1e-6, 40


def weights(ctx, seed, rows, cols):
    q = synth.q8_0(synth.seed(75, seed), rows, cols, dscale=0.01)
    return ctx.upload(q), ref.dequant("q8_0", q).astype(np.float64).reshape(rows, cols)


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_replayed_tree_steps(ctx, window, sinks):
    rng = np.random.default_rng(5)
    (wq, mq), (wk, mk), (wv, mv), (wo, mo), (wh, mh) = [weights(ctx, i, r, c) for i, (r, c) in enumerate(
        ((HQ * W, HID), (HKV * W, HID), (HKV * W, HID), (HID, HQ * W), (V, HID)))]
    norm, freq = (rng.random(HID) + 0.5).astype(np.float32), (10000.0 ** (-np.arange(0, W, 2) / W)).astype(np.float32)
    nb, fb = ctx.upload(norm), ctx.upload(freq)
    up, rows, S = ctx.upload, [9, 0, 20], 3
    T, most, words = sum(rows), 20, 1
    start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    table = np.full((S, 12), -1, np.int32)
    order = rng.permutation(PAGES)
    table[0], table[2] = order[:12], order[12:24]  # sequence 1 is an unused slot
    cache = KV8Cache.alloc(ctx, PAGES, HKV, P, W)
    for b in cache.buffers:
        b.upload(np.zeros(b.length, np.uint8))
    lens = [30, 0, 61]  # of tokens before the step; their codes are whatever the first test step finds: zeros with a scale
    for i in (2, 3):
        cache.buffers[i].upload(np.full(PAGES * HKV, 2.0 ** -6, np.float32))
    for i in (0, 1):
        cache.buffers[i].upload((rng.integers(0, 256, PAGES * HKV * P * W).astype(np.uint8) & 0xbf))
    tb, lb, sb = up(table), up(np.zeros(S, np.int32)), up(start)
    batch = KV8Batch(tb, lb, sb, S, 12, T, most, 12 * P)
    f32 = {n: ctx.alloc(4 * T * w) for n, w in (("x", HID), ("q", HQ * W), ("k", HKV * W), ("v", HKV * W), ("a", HQ * W), ("y", HID),
                                                 ("l", V), ("p", V))}
    i32 = {n: up(np.zeros(k, np.int32)) for n, k in (("pos", T), ("parent", T), ("token", T), ("chosen", T), ("path", T), ("count", S),
                                                     ("next", S), ("left", S), ("past", S * 64), ("past_len", S))}
    seen, allowed, penalty = up(np.zeros(T, np.uint32)), up(np.zeros((T, V // 32), np.uint32)), up(np.tile(
        np.array([1.2, 0.3, 0.1], np.float32), (S, 1)))
    drafts = Drafts(seen, words, position=i32["pos"], parent=i32["parent"], token=i32["token"])
    rules = LogitRules(sb, S, most, penalty=penalty, history=i32["past"], historyLen=i32["past_len"], historyStride=64,
                       allowed=allowed, allowedStride=V // 32)
    q, k, v = HeadRows(f32["q"], HQ, HQ * W), HeadRows(f32["k"], HKV, HKV * W), HeadRows(f32["v"], HKV, HKV * W)
    a = HeadRows(f32["a"], HQ, HQ * W)
    attend, choose = KV8AttentionKernel(ctx), LogitChoiceKernel(ctx)
    ws, ws2 = ctx.alloc(max(16, attend.workspaceBytes(cache, batch, HQ))), ctx.alloc(choose.workspaceBytes(T, V))
    gemv = GEMVKernel(ctx)
    st = ctx.stream()
    with Capture(ctx, st) as cap:
        FusedQ8Kernel(ctx).encodeFusedQKVTurbo(st, wq, wk, wv, f32["x"], f32["q"], f32["k"], f32["v"], nb, HQ * W, HKV * W, HID, T, EPS)
        QKNormRopeKernel(ctx).encode(st, q, k, q, k, i32["pos"], T, W, Rope(fb, W))
        KV8AppendKernel(ctx).encode(st, cache, batch, k, v, Rope(None, 0))
        attend.encode(st, cache, batch, q, a, W ** -0.5, window=window, workspace=ws, sinks=sinks, drafts=drafts)
        gemv.encodeBatchedQ8_0Weights(st, wo, f32["a"], f32["y"], T, HID, HQ * W)
        gemv.encodeBatchedQ8_0Weights(st, wh, f32["y"], f32["l"], T, V, HID)
        choose.encode(st, f32["l"], T, V, rules, drafts=drafts, out=f32["p"], chosen=i32["chosen"], workspace=ws2)
        KV8AcceptKernel(ctx).encode(st, cache, batch, drafts, i32["chosen"], i32["path"], i32["count"], i32["next"], i32["left"])

    def snapshot():
        shape = (PAGES, HKV, P, W)
        kc, vc, ks, vs = cache.buffers
        return (kc.download(np.uint8).reshape(shape), ks.download(np.float32).reshape(shape[:2]),
                vc.download(np.uint8).reshape(shape), vs.download(np.float32).reshape(shape[:2]))

    def host(n, width):
        return f32[n].download(np.float32).reshape(T, width)
    kept = moved = 0
    history = [[int(t) for t in rng.integers(0, V, 10)] for _ in range(S)]
    token = rng.integers(0, V, T).astype(np.int32)
    trees = [D.tree(rng, n)[0] if n else np.zeros(0, np.int32) for n in rows]
    able = rng.random((T, V)) < 0.5
    able[5] = False
    for step in range(4):
        b = R.Batch(rng, [0] * S, [0] * S, P)
        b.table, b.stride, b.pages, b.start, b.rows, b.total = table, 12, PAGES, start, rows, T
        b.lens = [m + n for m, n in zip(lens, rows)]
        parent, pos, mask, bits = np.zeros(T, np.int32), np.zeros(T, np.int32), np.zeros(T, np.uint32), []
        for s, n in enumerate(rows):
            at = slice(start[s], start[s] + n)
            parent[at] = trees[s]
            bits.append(D.lines(parent[at]))
            pos[at] = lens[s] + bits[s].sum(1) - 1
            mask[at] = D.words(bits[s], words)[:, 0] if n else []
        # the same rows as in the step before, so that some of the drafts are what the model chooses there
        x = synth.normal_f32(synth.seed(76, 1), T * HID).reshape(T, HID)
        past = np.zeros((S, 64), np.int32)
        for s in range(S):
            past[s, :len(history[s])] = history[s]
        for n, w in (("pos", pos), ("parent", parent), ("token", token), ("past", past),
                     ("past_len", np.array([len(h) for h in history], np.int32))):
            i32[n].upload(w)
        f32["x"].upload(x), seen.upload(mask), allowed.upload(D.words(able)), lb.upload(np.array(b.lens, np.int32))
        before = snapshot()
        ctx.synchronize()
        cap.graph.launch(st)
        st.synchronize()
        n64 = x.astype(np.float64)
        n64 = n64 / np.sqrt((n64 * n64).mean(1, keepdims=True) + EPS) * norm
        hq, hk, hv = host("q", HQ * W), host("k", HKV * W), host("v", HKV * W)
        assert rel_l2(hq, R.norm_rope((n64 @ mq.T).reshape(T, HQ, W), pos, freq, W, False).reshape(T, -1)) < 1e-5
        assert rel_l2(hk, R.norm_rope((n64 @ mk.T).reshape(T, HKV, W), pos, freq, W, False).reshape(T, -1)) < 1e-5
        assert rel_l2(hv, n64 @ mv.T) < 1e-5
        kc, ks = R.append(before[0], before[1], b, hk.reshape(T, HKV, W).astype(np.float64))
        vc, vs = R.append(before[2], before[3], b, hv.reshape(T, HKV, W).astype(np.float64))
        see = [D.visible(m, n, window, sinks, bits[s], pos[start[s]:start[s] + n]) for s, (n, m) in enumerate(zip(rows, b.lens))]
        exp, tol = D.attend(kc, ks, vc, vs, b, hq.reshape(T, HQ, W), W ** -0.5, see)
        ha = host("a", HQ * W)
        assert np.all(np.abs(ha.reshape(T, HQ, W) - exp) <= tol)
        assert rel_l2(host("y", HID), ha.astype(np.float64) @ mo.T) < 1e-5
        assert rel_l2(host("l", V), host("y", HID).astype(np.float64) @ mh.T) < 1e-5
        logits, chosen = host("l", V), i32["chosen"].download(np.int32)
        paths = []
        for s, n in enumerate(rows):
            for i in range(n):
                r = start[s] + i
                context = history[s] + [token[start[s] + j] for j in np.flatnonzero(bits[s][i])]
                y, pick = D.choose(logits[r], context, (1.2, 0.3, 0.1), (), able[r])
                assert pick == chosen[r]
                fin = np.isfinite(y)
                assert np.all(np.abs(host("p", V)[r][fin] - y[fin]) <= D.U24 * 1.001 * np.abs(y[fin]) + 1e-12)
            at = slice(start[s], start[s] + n)
            paths.append(D.walk(parent[at], token[at], chosen[at]) if n else ([], -1))
        want = D.accept(kc, ks, b, [p for p, _ in paths]) + D.accept(vc, vs, b, [p for p, _ in paths])
        assert all(np.array_equal(g, w) for g, w in zip(snapshot(), want))
        assert list(i32["count"].download(np.int32)) == [len(p) for p, _ in paths]
        assert list(i32["next"].download(np.int32)) == [t for _, t in paths]
        left = list(i32["left"].download(np.int32))
        assert left == [m + len(p) for m, (p, _) in zip(lens, paths)]
        kept += sum(len(p) - 1 for p, _ in paths if p)
        moved += sum(p[-1] != len(p) - 1 for p, _ in paths if p)
        for s, (p, t) in enumerate(paths):
            history[s] += [int(token[start[s] + j]) for j in p]
        lens = [int(m) for m in left]
        # drafts of the next step: mostly what was chosen in this one at the row in front of them
        trees = [D.tree(rng, n)[0] if n else np.zeros(0, np.int32) for n in rows]
        for s, n in enumerate(rows):
            for i in range(1, n):
                token[start[s] + i] = chosen[start[s] + trees[s][i]] if rng.random() < 0.8 else rng.integers(0, V)
    cap.graph.destroy()
    st.destroy()
    assert kept > 0 and moved > 0
