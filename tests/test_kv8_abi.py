"""Refusals of the operators between the projections: decided from sizes,
lengths and pointers before a device is touched (null context, placeholder
pointers that are never read), so they run without a GPU."""
import ctypes as C

import pytest

from edgerunner_amd import _ffi

F32, F16, BF16 = 0, 1, 30
OK_BUT_NO_CTX, ARG, VEC, MAT, ENC = 8, 8, 5, 4, 3
NULL = _ffi.er_buffer(None, 0)


def buf(n, ptr=0x100000):
    return _ffi.er_buffer(ptr, n)


def rows(heads, stride, n, d=64, ptr=0x10000000, width=4):
    return _ffi.er_head_rows(buf(((n - 1) * stride + heads * d) * width, ptr), heads, stride)


def rope(rot=64, inter=0, length=None):
    return _ffi.er_rope(buf(rot * 2 if length is None else length), rot, inter)


def last():
    return _ffi.last_error()


# ---------------------------------------------------------------- qk_norm_rope

def call_rope(q=None, k="same", qo=None, ko="same", pos=None, qn=NULL, kn=NULL, r=None, n=3, d=64):
    q = rows(4, 256, 3, ptr=0x10000000) if q is None else q
    qo = rows(4, 256, 3, ptr=0x20000000) if qo is None else qo
    k = rows(2, 128, 3, ptr=0x30000000) if k == "same" else k
    ko = rows(2, 128, 3, ptr=0x40000000) if ko == "same" else ko
    ref = lambda x: C.byref(x) if x is not None else None  # noqa: E731
    return _ffi.load().er_hip_qk_norm_rope(None, None, ref(q), ref(k), ref(qo), ref(ko), buf(12) if pos is None else pos,
                                           qn, kn, ref(rope() if r is None else r), n, d, 1e-6)


def test_rope_valid_calls_reach_the_context():
    assert call_rope() == OK_BUT_NO_CTX and "null er_hip_ctx" in last()
    assert call_rope(k=None, ko=None) == OK_BUT_NO_CTX and "null er_hip_ctx" in last()
    same = rows(4, 256, 3)
    assert call_rope(q=same, qo=same) == OK_BUT_NO_CTX and "null er_hip_ctx" in last()
    # q and k as columns of one projection's rows, normed in place
    q, k = rows(4, 384, 3, ptr=0x10000000), rows(2, 384, 3, ptr=0x10000000 + 4 * 256)
    assert call_rope(q=q, k=k, qo=q, ko=k) == OK_BUT_NO_CTX and "null er_hip_ctx" in last()
    # no rotation needs neither frequencies nor positions
    assert call_rope(r=_ffi.er_rope(NULL, 0, 0), pos=NULL) == OK_BUT_NO_CTX and "null er_hip_ctx" in last()


def test_rope_refusals():
    assert call_rope(d=96) == VEC and "head_dim 96" in last()
    assert call_rope(r=rope(60)) == VEC and call_rope(r=rope(72)) == VEC
    assert call_rope(r=rope(64, length=127)) == ENC and "inv_freq" in last()
    assert call_rope(r=_ffi.er_rope(buf(128, 0x1002), 64, 0)) == ARG and "aligned" in last()
    assert call_rope(k=None) == ARG and "together" in last()
    assert call_rope(pos=buf(11)) == ENC and "positions" in last()
    assert call_rope(qn=buf(255)) == ENC and call_rope(kn=buf(255)) == ENC
    assert call_rope(q=rows(4, 255, 3)) == VEC and "stride" in last()
    assert call_rope(q=rows(0, 256, 3)) == VEC
    q = rows(4, 256, 3)
    q.data.length -= 1
    assert call_rope(q=q) == ENC and "too small" in last()
    assert call_rope(qo=rows(3, 256, 3, ptr=0x20000000)) == VEC
    assert call_rope(q=rows(4, 256, 3, ptr=0x10000002)) == ARG
    assert call_rope(n=1 << 30) == VEC


@pytest.mark.parametrize("shift", [4, 4 * 64, 4 * 255])
def test_rope_refuses_overlapping_outputs(shift):
    assert call_rope(q=rows(4, 256, 3, ptr=0x10000000), qo=rows(4, 256, 3, ptr=0x10000000 + shift)) == ARG
    assert "overlap" in last()
    assert call_rope(q=rows(4, 256, 3, ptr=0x10000000 + shift), qo=rows(4, 256, 3, ptr=0x10000000)) == ARG
    # k written into q's rows, between its heads' end and the next row: 384 wide rows hold 4 + 2 heads, not 4 + 3
    assert call_rope(qo=rows(4, 384, 3, ptr=0x20000000), ko=rows(2, 384, 3, ptr=0x20000000 + 4 * 256 + 4)) == ARG


# ---------------------------------------------------------------- cache and batch

def cache(pages=8, heads=2, P=16, d=64, short=None):
    n, s = pages * heads * P * d, 4 * pages * heads
    c = _ffi.er_kv8_cache(buf(n, 0x50000000), buf(n, 0x60000000), buf(s, 0x70000000), buf(s, 0x71000000), pages, heads, P, d)
    if short:
        getattr(c, short).length -= 1
    return c


def batch(seqs=2, stride=3, rows_=3, max_rows=2, max_len=40):
    return _ffi.er_kv8_batch(buf(4 * seqs * stride), buf(4 * seqs), buf(4 * seqs + 4), seqs, stride, rows_, max_rows, max_len)


def call_append(c=None, b=None, k=None, v=None, vt=F32, q=None, qo=None, kn=NULL, qn=NULL, r=None):
    k = rows(2, 128, 3, ptr=0x10000000) if k is None else k
    v = rows(2, 128, 3, ptr=0x20000000) if v is None else v
    ref = lambda x: C.byref(x) if x is not None else None  # noqa: E731
    return _ffi.load().er_hip_kv8_append(None, None, ref(cache() if c is None else c), ref(batch() if b is None else b), ref(k),
                                         ref(v), vt, ref(q), ref(qo), kn, qn, ref(rope() if r is None else r), 1e-6)


def call_attend(c=None, b=None, q=None, o=None, ot=F32, scale=0.125, window=0, ws=NULL):
    q = rows(4, 256, 3, ptr=0x10000000) if q is None else q
    o = rows(4, 256, 3, ptr=0x20000000) if o is None else o
    return _ffi.load().er_hip_kv8_attention(None, None, C.byref(cache() if c is None else c),
                                            C.byref(batch() if b is None else b), C.byref(q), C.byref(o), ot, scale, window, ws)


def test_cache_valid_calls_reach_the_context():
    for call in (call_append, call_attend):
        assert call() == OK_BUT_NO_CTX and "null er_hip_ctx" in last()
        assert call(b=batch(rows_=0, max_rows=0)) == OK_BUT_NO_CTX and "null er_hip_ctx" in last()
        assert call(b=_ffi.er_kv8_batch(NULL, NULL, NULL, 0, 0, 3, 1, 0)) == OK_BUT_NO_CTX and "null er_hip_ctx" in last()
    q = rows(4, 256, 3, ptr=0x30000000)
    assert call_append(q=q, qo=q) == OK_BUT_NO_CTX and "null er_hip_ctx" in last()


@pytest.mark.parametrize("call", [call_append, call_attend])
def test_cache_and_batch_refusals(call):
    assert call(c=cache(d=96)) == VEC and call(c=cache(P=8)) == VEC and call(c=cache(P=128)) == VEC
    assert call(c=cache(heads=0)) == VEC and call(c=cache(pages=0)) == MAT
    for part in ("k", "v", "k_scale", "v_scale"):
        assert call(c=cache(short=part)) == MAT and "too small" in last(), part
    c = cache()
    c.k.data = 0x50000008
    assert call(c=c) == ARG and "16-byte" in last()
    c = cache()
    c.v.data = None
    assert call(c=c) == ARG and "null" in last()
    assert call(b=batch(max_rows=0)) == VEC and call(b=batch(max_rows=4)) == VEC
    assert call(b=batch(max_len=1 << 30)) == VEC
    for part in ("page_table", "kv_len", "row_start"):
        b = batch()
        getattr(b, part).length -= 1
        assert call(b=b) == ENC and "too small" in last(), part
        b = batch()
        getattr(b, part).data = 0x1002
        assert call(b=b) == ARG, part


def test_cache_sizes_pass_32_bits():
    """A pool of over 2^32 bytes is measured in 64 bits: one byte short is refused, the whole reaches the context."""
    assert call_attend(c=cache(pages=1 << 20, heads=2, P=64, d=64)) == OK_BUT_NO_CTX
    assert call_attend(c=cache(pages=1 << 20, heads=2, P=64, d=64, short="v")) == MAT
    assert call_attend(c=cache(pages=0x7fffffff, heads=65536, P=64, d=256)) == VEC  # 4 query heads over 65536


def test_append_refusals():
    assert call_append(vt=BF16) == ARG and "v_type" in last()
    assert call_append(k=rows(3, 192, 3)) == VEC and call_append(v=rows(1, 64, 3)) == VEC
    short = rows(2, 128, 3, ptr=0x20000000)
    short.data.length //= 2
    assert call_append(v=short) == ENC
    assert call_append(v=rows(2, 128, 3, ptr=0x20000000, width=2), vt=F16) == OK_BUT_NO_CTX
    assert call_append(q=rows(4, 256, 3, ptr=0x30000000)) == ARG and "together" in last()
    q = rows(4, 256, 3, ptr=0x30000000)
    assert call_append(q=q, qo=rows(4, 256, 3, ptr=0x30000004)) == ARG and "overlap" in last()
    assert call_append(q=q, qo=rows(4, 256, 3, ptr=0x10000000)) == ARG and "overlap" in last()
    assert call_append(q=q, qo=rows(4, 256, 3, ptr=0x20000000)) == ARG and "overlap" in last()
    assert call_append(kn=buf(255)) == ENC and call_append(r=rope(12)) == VEC


def test_attention_refusals():
    assert call_attend(ot=F16) == ARG and "out_type" in last()
    assert call_attend(scale=float("nan")) == ARG and call_attend(scale=float("inf")) == ARG
    assert call_attend(q=rows(3, 192, 3), o=rows(3, 192, 3, ptr=0x20000000)) == VEC
    assert call_attend(q=rows(2, 256, 3)) == VEC and "differ" in last()
    assert call_attend(o=rows(4, 256, 3, ptr=0x10000000)) == ARG and "overlap" in last()
    assert call_attend(c=cache(heads=1), q=rows(1025, 1025 * 64, 3), o=rows(1025, 1025 * 64, 3, ptr=0x20000000)) == VEC
    half = rows(4, 256, 3, ptr=0x20000000, width=2)
    assert call_attend(o=half) == ENC
    assert call_attend(o=half, ot=BF16) == OK_BUT_NO_CTX and "null er_hip_ctx" in last()


def test_attention_refuses_what_32_bits_cannot_count():
    wide = 1024 * 64
    many = rows(1024, wide, 1 << 22)
    b = batch(rows_=1 << 22, max_rows=1 << 22)
    assert call_attend(c=cache(heads=1), b=b, q=many, o=rows(1024, wide, 1 << 22, ptr=1 << 60)) == VEC and "31 bits" in last()
    n = 1 << 20
    b = _ffi.er_kv8_batch(buf(4 * n * (1 << 18)), buf(4 * n), buf(4 * n + 4), n, 1 << 18, 3, 2, 1 << 22)
    assert call_attend(b=b) == VEC and "31 bits" in last()
    b.max_kv_len = 1 << 10
    assert call_attend(b=b) == OK_BUT_NO_CTX and "null er_hip_ctx" in last()


def test_workspace_query():
    n = C.c_uint64(7)
    f = _ffi.load().er_hip_kv8_attention_workspace
    assert f(None, C.byref(cache()), C.byref(batch()), 4, C.byref(n)) == OK_BUT_NO_CTX and n.value == 0
    assert f(None, C.byref(cache()), C.byref(batch()), 3, C.byref(n)) == VEC
    assert f(None, C.byref(cache()), C.byref(batch()), 4, None) == ARG
