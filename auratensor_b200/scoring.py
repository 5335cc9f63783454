"""Log probabilities of given tokens, with entropy and top alternatives
(at_logprobs of the C ABI). The reference's server returns sampled ids only
(server/InferenceServer.java:111-134)."""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from ._lib import IllegalArgumentException, lib
from .core import context
from .kvblock import _code

TOP_MAX = 32


@dataclass
class LogProbs:
    """Per row of logits: logSumExp and entropy (nats), logProb of the given
    token (None without tokens), topIds and topLogProbs [rows][top] in
    descending order, equal logits by the lower id (None for top 0)."""
    logProb: torch.Tensor | None
    logSumExp: torch.Tensor
    entropy: torch.Tensor
    topIds: torch.Tensor | None
    topLogProbs: torch.Tensor | None

    @staticmethod
    def of(logits: torch.Tensor, tokenIds: torch.Tensor | None = None, top: int = 0) -> "LogProbs":
        """logits: [rows][vocab] CUDA tensor, float32, float16 or bfloat16 (rows
        may be strided; not changed); tokenIds: int32 [rows], an id outside
        [0, vocab) gives NaN; top: 0 to 32 alternatives."""
        if logits.dim() != 2 or not logits.is_cuda:
            raise IllegalArgumentException(_lib.AT_ERR_INVALID_ARG, "logits must be a [rows][vocab] CUDA tensor")
        rows, vocab = logits.shape
        code = _code(logits.dtype, "logits")
        if vocab == 0 or (vocab > 1 and logits.stride(1) != 1):
            raise IllegalArgumentException(_lib.AT_ERR_INVALID_ARG, "logits need a vocabulary, contiguous in memory")
        dev = logits.device
        if tokenIds is not None and (tokenIds.dtype != torch.int32 or tokenIds.shape != (rows,) or tokenIds.device != dev
                                     or not tokenIds.is_contiguous()):
            raise IllegalArgumentException(_lib.AT_ERR_INVALID_ARG, f"tokenIds must be int32 [{rows}] on the logits' device")
        top = int(top)
        if not 0 <= top <= vocab:
            raise IllegalArgumentException(_lib.AT_ERR_INVALID_ARG, f"top must be in [0, {vocab}], got {top}")
        # one allocation: logsumexp, entropy, log probability per row, then the alternatives' ids and log probabilities
        buf = torch.empty(rows * (3 + 2 * top), dtype=torch.float32, device=dev)
        lse, ent = buf[:rows], buf[rows:2 * rows]
        lp = None if tokenIds is None else buf[2 * rows:3 * rows]
        ids = alt = None
        at = buf.data_ptr()
        if top:
            ids = buf.view(torch.int32).as_strided((rows, top), (top, 1), 3 * rows)
            alt = buf.as_strided((rows, top), (top, 1), (3 + top) * rows)
        rc = lib().at_logprobs(
            context(dev.index), logits.data_ptr(), code, rows, vocab, logits.stride(0) if rows > 1 else vocab,
            None if tokenIds is None else tokenIds.data_ptr(), top, None if tokenIds is None else at + 8 * rows, at, at + 4 * rows,
            at + 12 * rows if top else None, at + 4 * (3 + top) * rows if top else None)
        if rc:
            _lib.check(rc)
        return LogProbs(lp, lse, ent, ids, alt)
