"""What the host of the operators on drafts and logits launches and refuses
beyond test_draft_abi.py, whose calls and recorded runtime it shares: no GPU."""
import pytest

from edgerunner_amd import _ffi
from test_draft_abi import ENC, NULL, accept, batch, buf, drafts, launches
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
