"""What the host of the operators between the projections launches, with a
context and a runtime that only record it (kv8_host_stub.cpp): no GPU."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

from edgerunner_amd import _ffi
from edgerunner_amd.build import CSRC, ROCM, ROOT

F32, NOLIB, ENC = 0, 1, 3
NULL = _ffi.er_buffer(None, 0)
MOST = (1 << 24) - 1  # workgroups whose threads 32 bits count
STUB = Path(__file__).with_name("kv8_host_stub.cpp")


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    out = tmp_path_factory.mktemp("kv8") / "libkv8host.so"
    subprocess.run(["g++", "-O1", "-fPIC", "-shared", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I", str(ROCM / "include"),
                    "-I", str(ROOT / "include"), "-I", str(CSRC), str(CSRC / "er_kv8.cpp"), str(STUB), "-o", str(out)], check=True)
    lib = C.CDLL(str(out))
    for name in ("er_hip_qk_norm_rope", "er_hip_kv8_append", "er_hip_kv8_attention", "er_hip_kv8_attention_workspace"):
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
    a, b = C.c_uint(), C.c_uint()
    n = host.stub_launches(C.byref(a), C.byref(b))
    return [a.value, b.value][:n]


def rows(heads, n, ptr, d=64):
    return _ffi.er_head_rows(_ffi.er_buffer(ptr, n * heads * d * 4), heads, heads * d)


def cache(heads, pages=64, P=64, d=64):
    codes, scales = pages * heads * P * d, 4 * pages * heads
    return _ffi.er_kv8_cache(_ffi.er_buffer(1 << 50, codes), _ffi.er_buffer(2 << 50, codes), _ffi.er_buffer(3 << 50, scales),
                             _ffi.er_buffer(4 << 50, scales), pages, heads, P, d)


def batch(seqs, n, most, tokens, P=64):
    stride = -(-tokens // P)
    return _ffi.er_kv8_batch(_ffi.er_buffer(1 << 40, 4 * seqs * stride), _ffi.er_buffer(2 << 40, 4 * seqs),
                             _ffi.er_buffer(3 << 40, 4 * seqs + 4), seqs, stride, n, most, tokens)


def norm_rope(host, ctx, n):
    q, o = rows(1, n, 1 << 40), rows(1, n, 2 << 40)
    return host.er_hip_qk_norm_rope(ctx, None, C.byref(q), None, C.byref(o), None, NULL, NULL, NULL, C.byref(_ffi.er_rope(NULL, 0, 0)),
                                    n, 64, 1e-6)


def append(host, ctx, heads, b, n, queries=0):
    k, v = rows(heads, n, 5 << 50), rows(heads, n, 6 << 50)
    q, o = rows(max(queries, 1), n, 7 << 50), rows(max(queries, 1), n, 8 << 50)
    qs = (C.byref(q), C.byref(o)) if queries else (None, None)
    return host.er_hip_kv8_append(ctx, None, C.byref(cache(heads)), C.byref(b), C.byref(k), C.byref(v), F32, *qs, NULL, NULL,
                                  C.byref(_ffi.er_rope(NULL, 0, 0)), 1e-6)


def attend(host, ctx, heads, group, b, n, window=0):
    q, o = rows(heads * group, n, 5 << 50), rows(heads * group, n, 6 << 50)
    c, need = cache(heads), C.c_uint64()
    st = host.er_hip_kv8_attention_workspace(ctx, C.byref(c), C.byref(b), heads * group, C.byref(need))
    assert st == 0
    return host.er_hip_kv8_attention(ctx, None, C.byref(c), C.byref(b), C.byref(q), C.byref(o), F32, 0.125, window,
                                     _ffi.er_buffer(7 << 50, need.value))


def test_ordinary_calls_launch(host, ctx):
    assert norm_rope(host, ctx, 4096) == 0 and launches(host) == [1024]
    assert append(host, ctx, 8, batch(64, 64, 1, 2048), 64, 32) == 0 and len(launches(host)) == 1
    assert attend(host, ctx, 8, 4, batch(64, 64, 1, 512), 64) == 0 and launches(host) == [512]
    assert attend(host, ctx, 8, 4, batch(64, 64, 1, 8192), 64) == 0 and launches(host) == [512, 64 * 32]
    assert attend(host, ctx, 8, 4, batch(1, 4096, 4096, 4096), 4096) == 0 and launches(host) == [2 * 8 * 128, 4096]


def refused(host, status):
    return status == ENC and b"workgroups" in host.stub_error() and launches(host) == []


def test_rows_that_a_launch_does_not_count(host, ctx):
    assert norm_rope(host, ctx, 4 * MOST) == 0 and launches(host) == [MOST]
    assert refused(host, norm_rope(host, ctx, 4 * MOST + 1))
    assert refused(host, norm_rope(host, ctx, 1 << 28))


def test_appends_that_a_launch_does_not_count(host, ctx):
    n = 1 << 20
    assert append(host, ctx, 7, batch(n, n, 1, 64), n) == 0 and launches(host) == [14 * n]
    assert refused(host, append(host, ctx, 8, batch(n, n, 1, 64), n))
    n = 1 << 22  # the queries' workgroups count too
    assert append(host, ctx, 1, batch(n, n, 1, 64), n, 1) == 0 and launches(host) == [2 * n + n // 4]
    assert refused(host, append(host, ctx, 2, batch(n, n, 1, 64), n, 1))


def test_attention_that_a_launch_does_not_count(host, ctx):
    """Both launches of a call are checked before the first is queued."""
    n = 1 << 20
    assert refused(host, attend(host, ctx, 16, 1, batch(n, n, 1, 512), n))  # a workgroup a sequence and head
    assert refused(host, attend(host, ctx, 2, 16, batch(n, n, 1, 640), n))  # the join: a workgroup a row and query head
    assert attend(host, ctx, 2, 4, batch(n, n, 1, 640), n) == 0 and launches(host) == [512, 8 * n]
    assert refused(host, attend(host, ctx, 16, 1, batch(n, 128 * n, 128, 128), 128 * n))  # 128 columns a workgroup


def test_kernels_that_did_not_load_are_not_launched(host):
    """A context without the cache's kernels stays usable for the rest; the operators that need them say so."""
    ctx = host.stub_create(256, 0)
    launches(host)
    b = batch(2, 2, 1, 100)
    for call in (lambda: norm_rope(host, ctx, 8), lambda: append(host, ctx, 2, b, 2, 4), lambda: attend(host, ctx, 2, 2, b, 2)):
        assert call() == NOLIB and b"did not load" in host.stub_error() and launches(host) == []
    host.stub_destroy(ctx)
