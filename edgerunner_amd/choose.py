"""Rules on logits and the choice of a token (er_hip_choose_logits of
include/er_hip.h, which states the rules): penalties for tokens of the context,
biases, masks of allowed tokens.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

from . import _ffi
from .kv8 import Drafts, _Descriptor, _Kernel, _raw, _ref, _sh
from .runtime import Buffer, Stream, check


class LogitRules(_Descriptor):
    """Rules of a call's sequences; one that is None is left out.  penalty fp32 [sequences][3]: repetition, presence,
    frequency; history int32 [sequences][historyStride] and historyLen; biasToken int32 and bias fp32
    [sequences][biasStride] and biasLen; allowed uint32 [rows][allowedStride].  rowStart None: row r is sequence r."""

    def __init__(self, rowStart: Optional[Buffer] = None, sequences: int = 0, maxRows: int = 0, *,
                 penalty: Optional[Buffer] = None, history: Optional[Buffer] = None, historyLen: Optional[Buffer] = None,
                 historyStride: int = 0, biasToken: Optional[Buffer] = None, bias: Optional[Buffer] = None,
                 biasLen: Optional[Buffer] = None, biasStride: int = 0, allowed: Optional[Buffer] = None,
                 allowedStride: int = 0):
        buffers = (rowStart, penalty, history, historyLen, biasToken, bias, biasLen, allowed)
        super().__init__(_ffi.er_logit_rules(*(_raw(b) for b in buffers), sequences, maxRows, historyStride, biasStride,
                                             allowedStride), *buffers)


class LogitChoiceKernel(_Kernel):
    """Applies rules to logits and chooses the largest that is left."""

    entry = "er_hip_choose_logits"

    def workspaceBytes(self, rows: int, vocab: int) -> int:
        """Bytes of scratch that encode needs to choose."""
        n = C.c_uint64()
        check(self.lib.er_hip_choose_logits_workspace(self.ctx.handle, rows, vocab, C.byref(n)), self.lib)
        return int(n.value)

    def encode(self, stream: Optional[Stream], logits: Buffer, rows: int, vocab: int, rules: Optional[LogitRules] = None,
               drafts: Optional[Drafts] = None, out: Optional[Buffer] = None, chosen: Optional[Buffer] = None,
               workspace: Optional[Buffer] = None, rowStride: Optional[int] = None) -> None:
        """logits and out fp32 [rows][rowStride] (vocab, if not given); out may be logits; chosen int32 [rows], -1 where no
        token is left; drafts (seen, token): the rows' own tokens and their ancestors' count as context."""
        status = self._call(self.ctx.handle, _sh(stream), logits.raw, rows, vocab, vocab if rowStride is None else rowStride,
                            _ref(rules), _ref(drafts), _raw(out), _raw(chosen), _raw(workspace))
        if status:
            check(status, self.lib)
