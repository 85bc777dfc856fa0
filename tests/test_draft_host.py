"""What the host of the operators on drafts and logits launches and refuses
beyond test_draft_abi.py, whose calls and recorded runtime it shares: no GPU."""
import ctypes as C

import pytest

from edgerunner_amd import _ffi
from test_draft_abi import BF16, ENC, F32, NULL, accept, attend, batch, buf, cache, launches, ref, rows
from test_draft_abi import ctx, host  # noqa: F401  (fixtures)


def test_acceptance_of_idle_sequences(host, ctx):  # noqa: F811
    """Sequences without rows have counts, tokens and lengths too: written where none has any, and checked as others'."""
    idle = _ffi.er_kv8_batch(NULL, buf(8, 2 << 40), buf(12, 3 << 40), 2, 7, 0, 0, 100)
    none = _ffi.er_drafts(NULL, NULL, NULL, NULL, 0)
    on = {"lib": host, "ctx": ctx, "d": none, "chosen": NULL, "path": NULL}
    assert accept(b=idle, **on) == 0, host.stub_error()
    assert [g for g, _ in launches(host)] == [2 * 2 * 2]
    for part, n in (("kv_len", 7), ("row_start", 11)):
        b = _ffi.er_kv8_batch(NULL, buf(8, 2 << 40), buf(12, 3 << 40), 2, 7, 0, 0, 100)
        getattr(b, part).length = n
        assert accept(b=b, **on) == ENC, part
    for part in ("count", "next", "kv_len"):
        assert accept(b=idle, **on, **{part: buf(7, 50 << 40)}) == ENC, part
        assert accept(b=idle, **on, **{part: buf(8, 2 << 40)}) != 0, part  # the batch's lengths
    assert accept(b=batch(0, 0, 0), **on) == 0
    assert launches(host) == []


@pytest.mark.parametrize("d,P,out,grid", [(256, 16, F32, 256), (256, 16, BF16, 512), (256, 32, F32, 512), (128, 16, F32, 512)])
def test_shares_are_as_many_as_the_chip_holds(host, ctx, d, P, out, grid):  # noqa: F811
    """One workgroup a CU of the kernel that leaves room for one, two of the others, in the workspace of either type."""
    c, b, n = cache(4000, 2, P, d), batch(2, 6, 4, 4000, P), C.c_uint64()
    assert host.er_hip_kv8_attention_masked_workspace(ctx, ref(c), ref(b), 4, C.byref(n)) == 0
    assert n.value == 2 * 512 * 16 * (d + 2) * 4
    q, o = rows(4, 6, 5 << 50, d), rows(4, 6, 6 << 50, d, 2 if out == BF16 else 4)
    assert attend(c, b, q, o, ot=out, ws=buf(n.value, 7 << 50), lib=host, ctx=ctx) == 0, host.stub_error()
    assert launches(host)[0][0] == grid
