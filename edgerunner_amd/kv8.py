"""Between the projections: head norms with the position rotation, the 8-bit
paged key/value cache, and attention over it (the er_hip_qk_norm_rope and
er_hip_kv8_* entry points of include/er_hip.h, which states their rules).

encode appends to a stream and never allocates, as the other kernels' does;
the descriptors (HeadRows, Rope, KV8Cache, KV8Batch) wrap buffers that the
caller keeps, and are meant to be made once and passed to every call.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

from . import _ffi
from .runtime import Buffer, Context, Stream, check, default_context

TYPE_F32 = 0
TYPE_F16 = 1
TYPE_BF16 = 30

_NULL = _ffi.er_buffer(None, 0)


def _sh(stream: Optional[Stream]):
    return stream.handle if stream is not None else None


def _raw(buffer: Optional[Buffer]) -> _ffi.er_buffer:
    return buffer.raw if buffer is not None else _NULL


class _Descriptor:
    """A C struct over buffers; holds the buffers while it lives."""

    def __init__(self, raw, *buffers):
        self.raw = raw
        self.ref = C.byref(raw)
        self.buffers = buffers


def _ref(d: Optional[_Descriptor]):
    return d.ref if d is not None else None


class HeadRows(_Descriptor):
    """Rows of heads: head h of row r begins at element r * rowStride + h * headDim."""

    def __init__(self, buffer: Buffer, heads: int, rowStride: int):
        super().__init__(_ffi.er_head_rows(buffer.raw, heads, rowStride), buffer)


class Rope(_Descriptor):
    """Rotation of the first rotaryDim elements of a head: fp32 frequencies
    [rotaryDim / 2], pairs (i, i + rotaryDim / 2) or, interleaved, (2i, 2i + 1)."""

    def __init__(self, invFreq: Optional[Buffer], rotaryDim: int, interleaved: bool = False):
        super().__init__(_ffi.er_rope(_raw(invFreq), rotaryDim, 1 if interleaved else 0), invFreq)


class KV8Cache(_Descriptor):
    """Paged cache of one layer: e4m3 codes [pages][kvHeads][pageTokens][headDim]
    and power-of-two scales [pages][kvHeads], of keys and of values."""

    def __init__(self, k: Buffer, v: Buffer, kScale: Buffer, vScale: Buffer, pages: int, kvHeads: int,
                 pageTokens: int, headDim: int):
        super().__init__(_ffi.er_kv8_cache(k.raw, v.raw, kScale.raw, vScale.raw, pages, kvHeads, pageTokens, headDim),
                         k, v, kScale, vScale)

    @classmethod
    def alloc(cls, ctx: Context, pages: int, kvHeads: int, pageTokens: int, headDim: int) -> "KV8Cache":
        codes, scales = pages * kvHeads * pageTokens * headDim, 4 * pages * kvHeads
        return cls(ctx.alloc(codes), ctx.alloc(codes), ctx.alloc(scales), ctx.alloc(scales), pages, kvHeads,
                   pageTokens, headDim)


class KV8Batch(_Descriptor):
    """The sequences of a call: int32 page table [sequences][tableStride], cached
    lengths [sequences] (the call's rows included) and row starts [sequences + 1]."""

    def __init__(self, pageTable: Buffer, kvLen: Buffer, rowStart: Buffer, sequences: int, tableStride: int, rows: int,
                 maxRows: int, maxKvLen: int):
        super().__init__(_ffi.er_kv8_batch(pageTable.raw, kvLen.raw, rowStart.raw, sequences, tableStride, rows,
                                           maxRows, maxKvLen), pageTable, kvLen, rowStart)


class Drafts(_Descriptor):
    """The rows of a call as a tree of drafted tokens, at most 1024 of a sequence: uint32 masks [rows][seenWords] of the rows
    of its sequence that each sees (its ancestors and itself), and int32 positions, parents (index in the sequence, -1:
    none) and tokens [rows], each where an operator reads it."""

    def __init__(self, seen: Optional[Buffer], seenWords: int, position: Optional[Buffer] = None,
                 parent: Optional[Buffer] = None, token: Optional[Buffer] = None):
        super().__init__(_ffi.er_drafts(_raw(seen), _raw(position), _raw(parent), _raw(token), seenWords), seen, position,
                         parent, token)


class _Kernel:
    entry = ""

    def __init__(self, ctx: Optional[Context] = None):
        self.ctx = ctx or default_context()
        self.lib = self.ctx.lib
        self._call = getattr(self.lib, self.entry)  # a decode step's calls are bound by the host: looked up once


class QKNormRopeKernel(_Kernel):
    """RMS norm of each query and key head and the position rotation in one pass."""

    entry = "er_hip_qk_norm_rope"

    def encode(self, stream: Optional[Stream], q: HeadRows, k: Optional[HeadRows], qOut: HeadRows,
               kOut: Optional[HeadRows], positions: Optional[Buffer], rows: int, headDim: int, rope: Rope,
               qNorm: Optional[Buffer] = None, kNorm: Optional[Buffer] = None, eps: float = 1e-6) -> None:
        """q, k fp32 rows; a norm weight of None leaves that norm out; outputs may be their own inputs."""
        status = self._call(self.ctx.handle, _sh(stream), q.ref, _ref(k), qOut.ref, _ref(kOut), _raw(positions),
                            _raw(qNorm), _raw(kNorm), rope.ref, rows, headDim, eps)
        if status:
            check(status, self.lib)


class KV8AppendKernel(_Kernel):
    """Appends keys (normed and rotated on the way) and values to the cache; queries may ride along."""

    entry = "er_hip_kv8_append"

    def encode(self, stream: Optional[Stream], cache: KV8Cache, batch: KV8Batch, k: HeadRows, v: HeadRows, rope: Rope,
               kNorm: Optional[Buffer] = None, q: Optional[HeadRows] = None, qOut: Optional[HeadRows] = None,
               qNorm: Optional[Buffer] = None, eps: float = 1e-6, vHalf: bool = False) -> None:
        """k fp32, v fp32 or (vHalf) fp16, with the cache's heads."""
        status = self._call(self.ctx.handle, _sh(stream), cache.ref, batch.ref, k.ref, v.ref,
                            TYPE_F16 if vHalf else TYPE_F32, _ref(q), _ref(qOut), _raw(kNorm), _raw(qNorm), rope.ref, eps)
        if status:
            check(status, self.lib)


class KV8AttentionKernel(_Kernel):
    """Causal attention of the batch's rows over the cache."""

    entry = "er_hip_kv8_attention"

    def workspaceBytes(self, cache: KV8Cache, batch: KV8Batch, qHeads: int, masked: Optional[bool] = None) -> int:
        """Bytes of scratch that encode needs for such a batch, whatever its window and output type: with masks (sinks or
        drafts), without (False: often fewer), or for either (None; a batch that masked calls refuse, as it has
        too many steps to count, has the other's)."""
        n, m = C.c_uint64(), C.c_uint64()
        if not masked:
            check(self.lib.er_hip_kv8_attention_workspace(self.ctx.handle, cache.ref, batch.ref, qHeads, C.byref(n)),
                  self.lib)
        if masked is not False:
            status = self.lib.er_hip_kv8_attention_masked_workspace(self.ctx.handle, cache.ref, batch.ref, qHeads, C.byref(m))
            if masked:
                check(status, self.lib)
        return max(int(n.value), int(m.value))

    def encode(self, stream: Optional[Stream], cache: KV8Cache, batch: KV8Batch, q: HeadRows, out: HeadRows,
               scale: float, window: int = 0, workspace: Optional[Buffer] = None, outBF16: bool = False, sinks: int = 0,
               drafts: Optional["Drafts"] = None) -> None:
        """q fp32; out fp32 or bf16; window: the latest tokens that a row sees (0: all); sinks: the first tokens, which
        stay visible; drafts: the rows are a tree of drafted tokens (Drafts: seen, and position under a window)."""
        if sinks or drafts is not None:
            status = self.lib.er_hip_kv8_attention_masked(
                self.ctx.handle, _sh(stream), cache.ref, batch.ref, q.ref, out.ref, TYPE_BF16 if outBF16 else TYPE_F32, scale,
                window, sinks, _ref(drafts), _raw(workspace))
            if status:
                check(status, self.lib)
            return
        status = self._call(self.ctx.handle, _sh(stream), cache.ref, batch.ref, q.ref, out.ref,
                            TYPE_BF16 if outBF16 else TYPE_F32, scale, window, _raw(workspace))
        if status:
            check(status, self.lib)


class KV8AcceptKernel(_Kernel):
    """Keeps the chosen drafts: their keys and values move behind the sequence's earlier tokens."""

    entry = "er_hip_kv8_accept"

    def encode(self, stream: Optional[Stream], cache: KV8Cache, batch: KV8Batch, drafts: Drafts, chosen: Buffer, path: Buffer,
               count: Buffer, next: Buffer, kvLen: Buffer) -> None:
        """drafts: parent and token; chosen int32 [rows].  Writes path int32 [rows] and count, next, kvLen int32 [sequences]."""
        status = self._call(self.ctx.handle, _sh(stream), cache.ref, batch.ref, drafts.ref, chosen.raw, path.raw, count.raw,
                            next.raw, kvLen.raw)
        if status:
            check(status, self.lib)
