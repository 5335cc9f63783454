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
        dev, f32 = logits.device, torch.float32
        if tokenIds is not None and (tokenIds.dtype != torch.int32 or tokenIds.shape != (rows,) or tokenIds.device != dev
                                     or not tokenIds.is_contiguous()):
            raise IllegalArgumentException(_lib.AT_ERR_INVALID_ARG, f"tokenIds must be int32 [{rows}] on the logits' device")
        top = int(top)
        if not 0 <= top <= vocab:
            raise IllegalArgumentException(_lib.AT_ERR_INVALID_ARG, f"top must be in [0, {vocab}], got {top}")
        per_row = torch.empty((3, rows), dtype=f32, device=dev)
        lse, ent, lp = per_row.unbind(0)
        ids = torch.empty((rows, top), dtype=torch.int32, device=dev) if top else None
        alt = torch.empty((rows, top), dtype=f32, device=dev) if top else None
        _lib.check(lib().at_logprobs(
            context(dev.index), logits.data_ptr(), code, rows, vocab, logits.stride(0) if rows > 1 else vocab,
            None if tokenIds is None else tokenIds.data_ptr(), top, None if tokenIds is None else lp.data_ptr(), lse.data_ptr(),
            ent.data_ptr(), ids.data_ptr() if top else None, alt.data_ptr() if top else None))
        return LogProbs(None if tokenIds is None else lp, lse, ent, ids, alt)
