"""KV8AttentionKernel.workspaceBytes: which of the two queries a caller's number comes from.  No GPU:
queries that stand in for the library's, and the library's own up to the context that they lack."""
import ctypes as C
import types

import pytest

from edgerunner_amd import EdgeRunnerHIPError, KV8AttentionKernel, _ffi
from test_draft_abi import batch, cache

PLAIN, MASKED = "er_hip_kv8_attention_workspace", "er_hip_kv8_attention_masked_workspace"


class Lib:
    """Queries that give `needs`, or refuse, and remember that they were asked."""

    def __init__(self, needs):
        self.needs, self.asked = needs, []
        self.er_hip_kv8_attention = None
        self.er_hip_last_error = lambda: b"refused"

    def __getattr__(self, name):
        if name not in (PLAIN, MASKED):
            raise AttributeError(name)

        def query(ctx, c, b, heads, out):
            self.asked.append(name)
            out._obj.value = self.needs[name] or 0
            return 0 if self.needs[name] is not None else 5
        return query


def kernel(plain, masked):
    lib = Lib({PLAIN: plain, MASKED: masked})
    return lib, KV8AttentionKernel(types.SimpleNamespace(lib=lib, handle=None))


def described(x):
    return types.SimpleNamespace(ref=C.byref(x))


def test_plain_calls_pay_for_no_masks():
    c, b = described(cache()), described(batch())
    lib, k = kernel(100, 300)
    assert k.workspaceBytes(c, b, 4, masked=False) == 100 and lib.asked == [PLAIN]
    lib, k = kernel(100, 60)
    assert k.workspaceBytes(c, b, 4, masked=True) == 60 and lib.asked == [MASKED]
    for plain, masked in ((100, 300), (300, 100)):
        assert kernel(plain, masked)[1].workspaceBytes(c, b, 4) == 300


def test_batches_that_masked_calls_refuse():
    c, b = described(cache()), described(batch())
    assert kernel(100, None)[1].workspaceBytes(c, b, 4) == 100
    assert kernel(100, None)[1].workspaceBytes(c, b, 4, masked=False) == 100
    for plain, masked, which in ((100, None, True), (None, 100, None), (None, 100, False)):
        with pytest.raises(EdgeRunnerHIPError):
            kernel(plain, masked)[1].workspaceBytes(c, b, 4, masked=which)


def test_there_are_such_batches():
    """Sequences of 513 tokens and 256 rows of a head of width 256: the plain call counts fewer steps."""
    n, query = ((1 << 32) - 1) // (25 * 2 * 16) + 1, C.c_uint64()
    c, b = cache(100, 2, 64, 256), batch(n, n, 1, 513, 64)
    status = [getattr(_ffi.load(), f)(None, C.byref(c), C.byref(b), 512, C.byref(query)) for f in (PLAIN, MASKED)]
    assert status == [8, 5]  # the plain query gets as far as the missing context
