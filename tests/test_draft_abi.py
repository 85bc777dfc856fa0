"""Refusals of the operators on drafts and logits, decided from sizes, lengths
and pointers before a device is touched (null context, placeholder pointers
that are never read), and what their host launches, with a context and a
runtime that only record it (draft_host_stub.cpp): no GPU."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

from edgerunner_amd import _ffi
from edgerunner_amd.build import CSRC, ROCM, ROOT

F32, F16, BF16 = 0, 1, 30
NO_CTX, ARG, VEC, MAT, ENC, NOLIB = 8, 8, 5, 4, 3, 1
NULL = _ffi.er_buffer(None, 0)
MOST = (1 << 24) - 1  # workgroups whose threads 32 bits count


def buf(n, ptr=0x100000):
    return _ffi.er_buffer(ptr, n)


def rows(heads, n, ptr, d=64, width=4):
    return _ffi.er_head_rows(buf(n * heads * d * width, ptr), heads, heads * d)


def cache(pages=8, heads=2, P=16, d=64, short=None):
    n, s = pages * heads * P * d, 4 * pages * heads
    c = _ffi.er_kv8_cache(buf(n, 1 << 50), buf(n, 2 << 50), buf(s, 3 << 50), buf(s, 4 << 50), pages, heads, P, d)
    if short:
        getattr(c, short).length -= 1
    return c


def batch(seqs=2, n=6, most=4, tokens=100, P=16):
    stride = -(-tokens // P)
    return _ffi.er_kv8_batch(buf(4 * seqs * stride, 1 << 40), buf(4 * seqs, 2 << 40), buf(4 * seqs + 4, 3 << 40), seqs, stride, n,
                             most, tokens)


def drafts(n=6, words=1, **over):
    d = _ffi.er_drafts(buf(4 * n * words, 11 << 40), buf(4 * n, 12 << 40), buf(4 * n, 13 << 40), buf(4 * n, 14 << 40), words)
    for k, v in over.items():
        setattr(d, k, v)
    return d


def ref(x):
    return C.byref(x) if x is not None else None


def last():
    return _ffi.last_error()


def attend(c=None, b=None, q=None, o=None, ot=F32, scale=0.125, window=0, sinks=4, d=None, ws=NULL, lib=None, ctx=None, n=6):
    q = rows(4, n, 5 << 50) if q is None else q
    o = rows(4, n, 6 << 50) if o is None else o
    return (lib or _ffi.load()).er_hip_kv8_attention_masked(ctx, None, ref(cache() if c is None else c),
                                                            ref(batch() if b is None else b), ref(q), ref(o), ot, scale, window,
                                                            sinks, ref(d), ws)


def accept(c=None, b=None, d="some", lib=None, ctx=None, n=6, seqs=2, **over):
    d = drafts(n) if d == "some" else d
    a = {"chosen": buf(4 * n, 21 << 40), "path": buf(4 * n, 22 << 40), "count": buf(4 * seqs, 23 << 40),
         "next": buf(4 * seqs, 24 << 40), "kv_len": buf(4 * seqs, 25 << 40)} | over
    return (lib or _ffi.load()).er_hip_kv8_accept(ctx, None, ref(cache() if c is None else c), ref(batch() if b is None else b),
                                                  ref(d), *a.values())


def rules(seqs=2, most=4, past=50, entries=5, words=32, n=6, **over):
    r = _ffi.er_logit_rules(buf(4 * seqs + 4, 31 << 40), buf(12 * seqs, 32 << 40), buf(4 * seqs * past, 33 << 40),
                            buf(4 * seqs, 34 << 40), buf(4 * seqs * entries, 35 << 40), buf(4 * seqs * entries, 36 << 40),
                            buf(4 * seqs, 37 << 40), buf(4 * n * words, 38 << 40), seqs, most, past, entries, words)
    for k, v in over.items():
        setattr(r, k, v)
    return r


def choose(n=6, vocab=1000, stride=None, r="some", d=None, lib=None, ctx=None, **over):
    r = rules(n=n) if r == "some" else r
    span = 4 * n * (stride or vocab)
    a = {"out": buf(span, 42 << 40), "chosen": buf(4 * n, 43 << 40), "workspace": buf(8 * n * -(-vocab // 1024), 44 << 40)} | over
    x = a.pop("logits", buf(span, 41 << 40))
    return (lib or _ffi.load()).er_hip_choose_logits(ctx, None, x, n, vocab, vocab if stride is None else stride, ref(r), ref(d),
                                                     *a.values())


# ---------------------------------------------------------------- refusals

def reaches_the_context(status):
    return status == NO_CTX and "null er_hip_ctx" in last()


def test_valid_calls_reach_the_context():
    assert reaches_the_context(attend()) and reaches_the_context(attend(d=drafts())) and reaches_the_context(accept())
    assert reaches_the_context(attend(d=drafts(position=NULL, parent=NULL, token=NULL)))
    assert reaches_the_context(accept(d=drafts(seen=NULL, position=NULL, seen_words=0)))
    none = _ffi.er_kv8_batch(NULL, NULL, NULL, 0, 0, 3, 1, 0)
    assert reaches_the_context(attend(b=none)) and reaches_the_context(accept(b=none))
    assert reaches_the_context(choose()) and reaches_the_context(choose(r=None)) and reaches_the_context(choose(d=drafts()))
    assert reaches_the_context(choose(out=NULL)) and reaches_the_context(choose(chosen=NULL, workspace=NULL))
    x = buf(4 * 6 * 1000, 41 << 40)
    assert reaches_the_context(choose(logits=x, out=x))
    assert reaches_the_context(choose(r=rules(row_start=NULL, sequences=0, max_rows=0, penalty=buf(72, 1 << 40), bias=NULL, history=NULL)))
    empty = _ffi.er_logit_rules()
    assert reaches_the_context(choose(r=empty))


@pytest.mark.parametrize("call", [attend, accept])
def test_cache_and_batch_refusals(call):
    assert call(c=cache(d=96)) == VEC and call(c=cache(P=8)) == VEC and call(c=cache(heads=0)) == VEC
    for part in ("k", "v", "k_scale", "v_scale"):
        assert call(c=cache(short=part)) == MAT, part
    assert call(b=batch(most=0)) == VEC and call(b=batch(most=7)) == VEC and call(b=batch(tokens=1 << 30)) == VEC
    for part in ("page_table", "kv_len", "row_start"):
        b = batch()
        getattr(b, part).length -= 1
        assert call(b=b) == ENC and "too small" in last(), part


def test_attention_refusals():
    assert attend(ot=F16) == ARG and attend(scale=float("nan")) == ARG
    assert attend(q=rows(3, 6, 5 << 50), o=rows(3, 6, 6 << 50)) == VEC and attend(o=rows(4, 6, 5 << 50)) == ARG
    assert attend(o=rows(4, 6, 6 << 50, width=2)) == ENC and reaches_the_context(attend(o=rows(4, 6, 6 << 50, width=2), ot=BF16))
    # masks: too few words, too short, unaligned, more drafts than a tree has
    assert attend(d=drafts(words=0)) == VEC and "mask words" in last()
    assert attend(b=batch(n=40, most=33), d=drafts(40), n=40) == VEC
    assert reaches_the_context(attend(b=batch(n=40, most=33), d=drafts(40, 2), n=40))
    assert attend(d=drafts(seen=buf(23))) == ENC and attend(d=drafts(seen=buf(24, 0x1002))) == ARG and attend(d=drafts(seen=NULL)) == ENC
    assert attend(b=batch(n=1025, most=1025), d=drafts(1025, 33), n=1025) == VEC and "1024" in last()
    assert reaches_the_context(attend(b=batch(n=1025, most=1025), n=1025))  # causal rows are not drafts
    # positions are read under a window alone
    assert attend(d=drafts(position=NULL), window=5) == ENC and attend(d=drafts(position=buf(23)), window=5) == ENC
    assert reaches_the_context(attend(d=drafts(position=NULL)))


def test_lines_of_steps_that_32_bits_do_not_count():
    """Sequences of 513 tokens: 9 steps and 16 that rounding may add, of two heads, in 16 blocks of columns."""
    fit, d, ws = ((1 << 32) - 1) // (25 * 2 * 16), 256, C.c_uint64()
    f = _ffi.load().er_hip_kv8_attention_masked_workspace
    # 257 columns are the wide kernel's, which does not count them, and 512 tokens no shares
    for n, tokens, group, status in ((fit, 513, 256, NO_CTX), (fit + 1, 513, 256, VEC), (fit + 1, 513, 240, NO_CTX),
                                     (fit + 1, 513, 257, NO_CTX), (fit + 1, 512, 256, NO_CTX)):
        c, b = cache(100, 2, 64, d), batch(n, n, 1, tokens, 64)
        q, o = (_ffi.er_head_rows(buf(n * 2 * group * d * 4, x << 50), 2 * group, 2 * group * d) for x in (5, 6))
        assert attend(c, b, q, o, n=n) == status, (n, tokens, group)
        assert f(None, ref(c), ref(b), 2 * group, C.byref(ws)) == status, (n, tokens, group)


def test_accept_refusals():
    assert accept(d=None) == ARG and "null drafts" in last()
    assert accept(b=batch(n=1025, most=1025), d=drafts(1025), n=1025) == VEC and "1024" in last()
    for part in ("parent", "token"):
        assert accept(d=drafts(**{part: buf(23)})) == ENC and accept(d=drafts(**{part: buf(24, 0x1002)})) == ARG, part
    for part, n in (("chosen", 24), ("path", 24), ("count", 8), ("next", 8), ("kv_len", 8)):
        assert accept(**{part: buf(n - 1, 50 << 40)}) == ENC, part
        assert accept(**{part: _ffi.er_buffer(None, n)}) == ARG, part
    for part, n in (("path", 24), ("count", 8), ("next", 8), ("kv_len", 8)):
        for where in (2 << 40, (2 << 40) + 4, 3 << 40, 1 << 40, 13 << 40, 14 << 40, 21 << 40, 1 << 50, (2 << 50) + 4, 3 << 50, 4 << 50):
            assert accept(**{part: buf(n, where)}) == ARG and "overlap" in last(), (part, hex(where))
    assert accept(count=buf(8, 24 << 40)) == ARG and accept(path=buf(24, (25 << 40) - 20)) == ARG


def test_choose_refusals():
    assert choose(vocab=0) == VEC and choose(stride=999) == VEC and choose(n=1 << 30, r=None) == VEC
    assert choose(out=NULL, chosen=NULL) == ARG and "neither" in last()
    assert choose(logits=buf(23999, 41 << 40)) == ENC and choose(out=buf(23999, 42 << 40)) == ENC
    assert choose(logits=buf(24000, (41 << 40) + 2)) == ARG
    assert choose(chosen=buf(23, 43 << 40)) == ENC and choose(workspace=buf(47, 44 << 40)) == ENC
    assert choose(r=rules(max_rows=0)) == VEC and choose(r=rules(max_rows=7)) == VEC
    for part in ("row_start", "penalty", "history", "history_len", "bias", "bias_token", "bias_len", "allowed"):
        r = rules()
        getattr(r, part).length -= 1
        assert choose(r=r) == ENC, part
    assert choose(r=rules(allowed_stride=31)) == VEC and reaches_the_context(choose(r=rules(words=40, allowed=buf(4 * (5 * 40 + 32), 38 << 40))))
    assert choose(r=rules(history_stride=1 << 30)) == VEC and choose(r=rules(history_len=NULL)) == ENC
    assert choose(d=drafts(words=0)) == VEC and choose(d=drafts(token=buf(23))) == ENC
    for where in (31, 32, 33, 34, 35, 36, 37, 38, 43, 44):
        assert choose(out=buf(24000, where << 40)) == ARG and "overlap" in last(), where
    assert choose(out=buf(24000, (41 << 40) + 4)) == ARG and choose(chosen=buf(24, 41 << 40)) == ARG
    x = buf(24000, 41 << 40)
    assert choose(logits=x, out=x, chosen=buf(24, (41 << 40) + 40)) == ARG
    assert choose(d=drafts(), chosen=buf(24, 11 << 40)) == ARG and choose(d=drafts(), chosen=buf(24, 14 << 40)) == ARG


def test_workspace_query():
    n = C.c_uint64(7)
    f = _ffi.load().er_hip_choose_logits_workspace
    assert f(None, 6, 0, C.byref(n)) == VEC and n.value == 0
    assert f(None, 6, 1000, C.byref(n)) == NO_CTX and f(None, 6, 1000, None) == ARG
    n = C.c_uint64(7)
    f = _ffi.load().er_hip_kv8_attention_masked_workspace
    assert f(None, ref(cache()), ref(batch()), 3, C.byref(n)) == VEC and n.value == 0
    assert f(None, ref(cache(d=96)), ref(batch()), 4, C.byref(n)) == VEC and f(None, ref(cache()), None, 4, C.byref(n)) == ARG
    assert f(None, ref(cache()), ref(batch()), 4, C.byref(n)) == NO_CTX and f(None, ref(cache()), ref(batch()), 4, None) == ARG


# ---------------------------------------------------------------- launches

@pytest.fixture(scope="module")
def host(tmp_path_factory):
    out = tmp_path_factory.mktemp("draft") / "libdrafthost.so"
    stub = Path(__file__).with_name("draft_host_stub.cpp")
    subprocess.run(["g++", "-O1", "-fPIC", "-shared", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I", str(ROCM / "include"),
                    "-I", str(ROOT / "include"), "-I", str(CSRC), str(CSRC / "er_draft.cpp"), str(stub), "-o", str(out)], check=True)
    lib = C.CDLL(str(out))
    for name in ("er_hip_kv8_attention_masked", "er_hip_kv8_accept", "er_hip_choose_logits", "er_hip_choose_logits_workspace",
                 "er_hip_kv8_attention_masked_workspace"):
        f = getattr(lib, name)
        f.restype, f.argtypes = _ffi.SIGNATURES[name]
    lib.stub_create.restype = C.c_void_p
    lib.stub_destroy.argtypes = [C.c_void_p]
    lib.stub_error.restype = C.c_char_p
    return lib


@pytest.fixture
def ctx(host):
    c = host.stub_create(256, 1)
    launches(host)
    yield c
    host.stub_destroy(c)


def launches(host):
    a = (C.c_uint * 4)()
    n = host.stub_launches(a)
    return [(a[2 * i], a[2 * i + 1]) for i in range(min(n, 2))]


def test_ordinary_calls_launch(host, ctx):
    on = {"lib": host, "ctx": ctx}
    assert attend(**on) == 0 and [g for g, _ in launches(host)] == [2 * 2]
    big = buf(1 << 34, 7 << 50)
    assert attend(b=batch(tokens=4000), ws=big, **on) == 0 and [g for g, _ in launches(host)] == [512, 6 * 4]
    # a window that covers few tokens of a long cache: fewer pieces, and sinks add theirs
    long = batch(1, 200, 200, 100000, 64)
    args = dict(c=cache(2000, 2, 64), b=long, q=rows(4, 200, 5 << 50), o=rows(4, 200, 6 << 50), ws=big, n=200, **on)
    grids = []
    for window, sinks in ((0, 0), (1000, 0), (1000, 500)):
        assert attend(window=window, sinks=sinks, **args) == 0
        grids.append(launches(host)[0][0])
    assert grids[1] < grids[2] < grids[0]
    assert accept(**on) == 0 and [g for g, _ in launches(host)] == [2 * 2 * 2]


def test_more_units_than_workgroups_are_shared(host, ctx):
    """Units of middling length are a workgroup's each as long as a launch counts them."""
    on = {"lib": host, "ctx": ctx, "n": 600000}
    for n, grid in ((500000, 500000 * 8 * 4), (600000, 512)):
        c, b = cache(100, 8), batch(n, 600000, 16, 1000)
        q, o = rows(64, 600000, 5 << 50), rows(64, 600000, 6 << 50)
        assert attend(c, b, q, o, ws=buf(1 << 40, 7 << 50), **on) == 0, host.stub_error()
        assert launches(host)[0][0] == grid


def test_workspace_holds_the_parts_of_every_call(host, ctx):
    """What the query says is enough for each window, sinks and masks of such a batch, and one byte less is refused
    where the call that needs all of it is made."""
    n = C.c_uint64()
    f = host.er_hip_kv8_attention_masked_workspace
    for heads, most, tokens, P, need in ((4, 4, 512, 16, False), (4, 4, 4000, 16, True), (64, 20, 40000, 64, True), (64, 4, 900, 32, True)):
        c, b = cache(4000, 2, P), batch(3, 40, most, tokens, P)
        assert f(ctx, ref(c), ref(b), heads, C.byref(n)) == 0 and (n.value > 0) == need
        refused = 0
        for short in (0, 1):
            for window, sinks, d in ((0, 0, None), (700, 0, None), (700, 100, drafts(40)), (0, 0, drafts(40)), (1 << 31, 1 << 31, None)):
                ws = buf(n.value - short, 7 << 50) if need else NULL
                st = attend(c, b, rows(heads, 40, 5 << 50), rows(heads, 40, 6 << 50), window=window, sinks=sinks, d=d, ws=ws,
                            lib=host, ctx=ctx, n=40)
                assert st == (ENC if st and short and need else 0), (heads, window, sinks, host.stub_error())
                refused += st != 0
        assert (refused > 0) == need
    launches(host)


def test_small_calls_do_nothing(host, ctx):
    on = {"lib": host, "ctx": ctx}
    none = _ffi.er_kv8_batch(NULL, NULL, NULL, 0, 0, 3, 1, 0)
    assert attend(b=none, **on) == 0 and accept(b=none, **on) == 0 and choose(n=0, r=None, **on) == 0
    assert choose(r=rules(sequences=0), **on) == 0
    assert launches(host) == []


def test_calls_that_a_launch_does_not_count(host, ctx):
    on = {"lib": host, "ctx": ctx}
    n = 1 << 22
    b = batch(n, n, 1, 16)
    assert accept(cache(heads=3), b, drafts(n), n=n, seqs=n, **on) == ENC and b"workgroups" in host.stub_error()
    assert choose(n=n, vocab=20000, r=None, **on) == ENC and b"workgroups" in host.stub_error()
    assert launches(host) == []


def test_kernels_that_did_not_load_are_not_launched(host):
    ctx = host.stub_create(256, 0)
    launches(host)
    for call in (attend, accept, choose):
        assert call(lib=host, ctx=ctx) == NOLIB and b"did not load" in host.stub_error() and launches(host) == []
    host.stub_destroy(ctx)
