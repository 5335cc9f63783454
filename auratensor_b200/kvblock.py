"""Block-quantized KV cache: K and V in 8 bits with one scale for each block of
tokens and KV head, in pages that a per-sequence table names, and the causal
attention over it (at_kvb_* of the C ABI).

A ``BlockKvCache`` holds every layer of a model; a ``TokenBatch`` names runs of
tokens, one per sequence, and serves ``append``, ``attention`` and ``read`` of
all layers of a step. Decode steps (one token per sequence), prompts, and
mixtures of both are the same calls:

    cache = BlockKvCache.allocate(layers, 1024, 8, 128, maxSeqs=64, maxBlocks=128)
    cache.reserve(slot, len(prompt) + maxNew)
    batch = TokenBatch.of([slot], [0], [len(prompt)])
    for layer in range(layers):
        cache.append(layer, batch, k, v)
        y = cache.attention(layer, batch, q)

Every launch goes to torch's current stream. The reference keeps K and V in
FP32 (inference/KVCache.java:56-61).
"""
from __future__ import annotations

import ctypes as C
import math
import threading

import torch

from . import _lib
from ._lib import GGML_BF16, GGML_F16, GGML_F32, IllegalArgumentException, IllegalStateException, KvBlocksC, TokenBatchC, lib
from .core import _current_stream, context

INT32_MAX, INT64_MAX = (1 << 31) - 1, (1 << 63) - 1
NO_PAGE = -1  # table entry of a position that was not reserved: outside the pool, so that the kernels report it
DTYPE_CODES = {torch.float32: GGML_F32, torch.float16: GGML_F16, torch.bfloat16: GGML_BF16}


def _bad(msg: str):
    raise IllegalArgumentException(_lib.AT_ERR_INVALID_ARG, msg)


def _code(dtype: torch.dtype, what: str) -> int:
    code = DTYPE_CODES.get(dtype)
    if code is None:
        raise _lib.UnsupportedOperationException(_lib.AT_ERR_UNSUPPORTED, f"{what} must be float32, float16 or bfloat16, got {dtype}")
    return code


class TokenBatch:
    """Runs of consecutive tokens, one per sequence: sequence s has the packed
    tokens offsets[s] .. offsets[s + 1], at positions starts[s] and on, of slot
    slots[s]. slots and offsets are int32, starts int64 CUDA tensors; nTokens,
    maxTokens (longest run) and maxEnd (highest position + 1) are the host's
    upper bounds of them, which size the launches."""

    def __init__(self, slots: torch.Tensor, starts: torch.Tensor, offsets: torch.Tensor, nTokens: int, maxTokens: int, maxEnd: int):
        n = slots.numel()
        if slots.dtype != torch.int32 or offsets.dtype != torch.int32 or starts.dtype != torch.int64:
            _bad("slots and offsets must be int32, starts int64")
        if starts.numel() != n or offsets.numel() != n + 1:
            _bad(f"{n} slots need {n} starts and {n + 1} offsets, got {starts.numel()} and {offsets.numel()}")
        device = slots.get_device()  # -1: the host
        if device < 0 or starts.get_device() != device or offsets.get_device() != device:
            _bad("batch tensors must be on one device, a CUDA device")
        if not (slots.is_contiguous() and starts.is_contiguous() and offsets.is_contiguous()):
            _bad("batch tensors must be contiguous")
        if not (0 <= nTokens <= INT32_MAX and 0 <= maxTokens <= INT32_MAX and 0 <= maxEnd <= INT64_MAX):
            _bad(f"nTokens and maxTokens must be in [0, {INT32_MAX}], maxEnd in [0, {INT64_MAX}], got {nTokens}, {maxTokens}, {maxEnd}")
        self.slots, self.starts, self.offsets = slots, starts, offsets
        self.nSeqs, self.nTokens, self.maxTokens, self.maxEnd = n, int(nTokens), int(maxTokens), int(maxEnd)
        self._c = TokenBatchC(n, self.nTokens, self.maxTokens, 0, self.maxEnd, slots.data_ptr(), starts.data_ptr(), offsets.data_ptr())
        self._ref = C.addressof(self._c)

    @classmethod
    def of(cls, slots, starts, counts, device=None) -> "TokenBatch":
        """A batch from host lists (one copy to the device)."""
        slots, starts, counts = [int(x) for x in slots], [int(x) for x in starts], [int(x) for x in counts]
        n = len(slots)
        if len(starts) != n or len(counts) != n:
            _bad("slots, starts and counts must have the same length")
        if len(set(slots)) != n:
            _bad("a slot may appear once in a batch")
        if any(x < 0 for x in slots + starts + counts):
            _bad("slots, starts and counts must not be negative")
        offsets = [0]
        for c in counts:
            offsets.append(offsets[-1] + c)
        if max(slots, default=0) > INT32_MAX or offsets[-1] > INT32_MAX or any(s + c > INT64_MAX for s, c in zip(starts, counts)):
            _bad("slots and the number of tokens must fit 32 bits, positions 64")
        dev = torch.device("cuda") if device is None else device
        flat = torch.tensor(starts + slots + offsets, dtype=torch.int64).to(dev)
        i32 = flat[n:].to(torch.int32)
        return cls(i32[:n], flat[:n], i32[n:], offsets[-1], max(counts, default=0),
                   max((s + c for s, c in zip(starts, counts)), default=0))


class BlockKvCache:
    """The cache of every layer: int8 blocks, scales, tails, the page table and
    a free list of pages (host)."""

    def __init__(self, kBlocks, vBlocks, kScales, vScales, table, kTail, vTail, kTailMax, vTailMax, dtype, status=None):
        if kBlocks.dim() != 5 or kBlocks.dtype != torch.int8:
            _bad("kBlocks must be int8 [layers][blocks][kv heads][block tokens][head dim]")
        self.layers, self.nBlocks, self.headCountKv, self.blockTokens, self.headDim = kBlocks.shape
        if table.dim() != 2 or table.dtype != torch.int32:
            _bad("table must be int32 [sequences][blocks per sequence]")
        self.maxSeqs, self.maxBlocks = table.shape
        self.dtype = dtype
        code = _code(dtype, "the cache's type")
        f32 = torch.float32
        blocks, scales = kBlocks.shape, (self.layers, self.nBlocks, self.headCountKv)
        ring = (self.layers, self.maxSeqs, self.headCountKv, 2 * self.blockTokens)
        rows = ring + (self.headDim,)
        tails = (kTail, vTail, kTailMax, vTailMax)
        absent = sum(t is None for t in tails)
        if 0 < absent < 4:
            _bad("kTail, vTail, kTailMax and vTailMax go together")
        self.device = kBlocks.device
        index = self.device.index
        if not kBlocks.is_cuda or table.get_device() != index or not table.is_contiguous():
            _bad("the cache must be on one CUDA device, its table contiguous")
        for t, name, dt, shape in ((kBlocks, "kBlocks", torch.int8, blocks), (vBlocks, "vBlocks", torch.int8, blocks),
                                   (kScales, "kScales", f32, scales), (vScales, "vScales", f32, scales), (kTail, "kTail", dtype, rows),
                                   (vTail, "vTail", dtype, rows), (kTailMax, "kTailMax", f32, ring), (vTailMax, "vTailMax", f32, ring)):
            if t is None and absent == 4:
                continue
            if t.dtype != dt or t.shape != shape:
                _bad(f"{name} must be {dt} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")
            if t.get_device() != index or not t.is_contiguous():
                _bad(f"{name} must be contiguous and on the device of kBlocks")
        if status is not None and (status.dtype != torch.int32 or status.numel() != 1 or status.get_device() != index):
            _bad("status must be one int32 on the device of kBlocks")
        self.kBlocks, self.vBlocks, self.kScales, self.vScales, self.table = kBlocks, vBlocks, kScales, vScales, table
        self.kTail, self.vTail, self.kTailMax, self.vTailMax, self.status = kTail, vTail, kTailMax, vTailMax, status
        # layer l's buffers start l slices into each tensor
        buffers = (kBlocks, vBlocks, kScales, vScales) + (tails if absent == 0 else ())
        at = [t.data_ptr() for t in buffers]
        step = [t.stride(0) * t.element_size() for t in buffers] if self.layers > 1 else None
        none = (None,) * (8 - len(at))
        shared = (table.data_ptr(), None if status is None else status.data_ptr())
        self._c = [KvBlocksC(code, self.headCountKv, self.headDim, self.blockTokens, self.nBlocks, self.maxSeqs, self.maxBlocks, 0,
                             *(at if l == 0 else [p + l * s for p, s in zip(at, step)]), *none, *shared) for l in range(self.layers)]
        self._refs = [C.addressof(c) for c in self._c]
        self._ws = threading.local()  # attention workspaces by thread and stream
        self._scale = 1.0 / math.sqrt(self.headDim)
        self._free = None
        self._pages = None

    @classmethod
    def allocate(cls, layers: int, nBlocks: int, headCountKv: int, headDim: int, maxSeqs: int, maxBlocks: int,
                 blockTokens: int = 64, dtype: torch.dtype = torch.float32, device=None) -> "BlockKvCache":
        """An empty cache of nBlocks pages of blockTokens positions (16, 32, 64
        or 128) per layer; dtype is the type of appended K and V."""
        for name, x in (("layers", layers), ("nBlocks", nBlocks), ("headCountKv", headCountKv), ("maxSeqs", maxSeqs), ("maxBlocks", maxBlocks)):
            if x <= 0:
                _bad(f"{name} must be positive, got {x}")
        if headDim not in (64, 128):
            raise _lib.UnsupportedOperationException(_lib.AT_ERR_UNSUPPORTED, f"head_dim must be 64 or 128, got {headDim}")
        if blockTokens not in (16, 32, 64, 128):
            _bad(f"block_tokens must be 16, 32, 64 or 128, got {blockTokens}")
        _code(dtype, "the cache's type")
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)

        def zeros(*shape, dt=torch.float32):
            return torch.zeros(shape, dtype=dt, device=dev)

        blocks, scales = (layers, nBlocks, headCountKv, blockTokens, headDim), (layers, nBlocks, headCountKv)
        ring = (layers, maxSeqs, headCountKv, 2 * blockTokens)
        self = cls(zeros(*blocks, dt=torch.int8), zeros(*blocks, dt=torch.int8), zeros(*scales), zeros(*scales),
                   torch.full((maxSeqs, maxBlocks), NO_PAGE, dtype=torch.int32, device=dev), zeros(*ring, headDim, dt=dtype), zeros(*ring, headDim, dt=dtype),
                   zeros(*ring), zeros(*ring), dtype, zeros(1, dt=torch.int32))
        self._free = list(range(nBlocks - 1, -1, -1))
        self._pages = [[] for _ in range(maxSeqs)]
        return self

    @classmethod
    def wrap(cls, kBlocks, vBlocks, kScales, vScales, table, kTail=None, vTail=None, kTailMax=None, vTailMax=None,
             dtype: torch.dtype = torch.float32, status=None) -> "BlockKvCache":
        """A cache over existing tensors, whose page table the caller fills
        (every entry a reserved position needs, before its first use). Without
        the tails it can be read but not appended to. status: an int32 CUDA
        tensor of one zero for ``check``."""
        return cls(kBlocks, vBlocks, kScales, vScales, table, kTail, vTail, kTailMax, vTailMax, dtype, status)

    # ---- pages (host) ----
    def _own_pages(self):
        if self._free is None:
            raise IllegalStateException(_lib.AT_ERR_STATE, "the page table of a wrapped cache is the caller's")

    def reserve(self, slot: int, length: int) -> None:
        """Gives slot the pages of its first `length` positions. Calls on
        positions without a page write nothing, read NaN, and make ``check``
        raise."""
        self._own_pages()
        if not 0 <= slot < self.maxSeqs:
            _bad(f"slot {slot} out of range [0, {self.maxSeqs})")
        need = -(-length // self.blockTokens)
        if need > self.maxBlocks:
            raise IllegalStateException(_lib.AT_ERR_STATE, f"{length} positions need {need} blocks, a sequence has {self.maxBlocks} at most")
        have = self._pages[slot]
        more = need - len(have)
        if more <= 0:
            return
        if more > len(self._free):
            raise IllegalStateException(_lib.AT_ERR_STATE, f"the pool has {len(self._free)} free blocks, {more} are needed")
        new = [self._free.pop() for _ in range(more)]
        self.table[slot, len(have):need] = torch.tensor(new, dtype=torch.int32).to(self.device)
        have.extend(new)

    def release(self, slot: int) -> None:
        """Returns the slot's pages to the pool (the sequence is over)."""
        self._own_pages()
        if not 0 <= slot < self.maxSeqs:
            _bad(f"slot {slot} out of range [0, {self.maxSeqs})")
        pages = self._pages[slot]
        if pages:
            self.table[slot, :len(pages)] = NO_PAGE
            self._free.extend(reversed(pages))
            self._pages[slot] = []

    def freeBlocks(self) -> int:
        self._own_pages()
        return len(self._free)

    # ---- operators ----
    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.layers:
            _bad(f"layer {layer} out of range [0, {self.layers})")
        return self._refs[layer]

    def _on_device(self, *tensors):
        for t in tensors:
            if t.get_device() != self.device.index:
                _bad(f"expected a tensor on {self.device}, got {t.device}")

    def _workspace(self, stream: int, need: int) -> torch.Tensor:
        """At least `need` bytes that this thread's calls on this stream share
        (they run one after the other; another thread's launches may come
        between a call's two kernels). A captured graph gets memory of its own."""
        if torch.cuda.is_current_stream_capturing():
            return torch.empty(need, dtype=torch.uint8, device=self.device)
        mine = self._ws.__dict__
        ws = mine.get(stream)
        if ws is None or ws.numel() < need:
            ws = mine[stream] = torch.empty(need, dtype=torch.uint8, device=self.device)
        return ws

    def append(self, layer: int, batch: TokenBatch, k: torch.Tensor, v: torch.Tensor) -> None:
        """Quantizes the batch's K and V ([tokens][kv heads][head dim], the
        cache's dtype; token and head strides are free) into the cache. A run
        starts at its slot's next position or goes back: to the first row of
        any block, or inside the last block written or the one before it, but
        not further for having gone back before (``check`` reports it)."""
        ref = self._layer(layer)
        shape, ks, vs = (batch.nTokens, self.headCountKv, self.headDim), k.stride(), v.stride()
        for t, s, name in ((k, ks, "k"), (v, vs, "v")):
            if t.dtype != self.dtype or t.shape != shape:
                _bad(f"{name} must be {self.dtype} {shape}, got {t.dtype} {tuple(t.shape)}")
            if s[2] != 1:
                _bad(f"{name}'s last dimension must be contiguous")
        self._on_device(k, v, batch.slots)
        rc = lib().at_kvb_append(context(self.device.index), ref, batch._ref, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1])
        if rc:
            _lib.check(rc)

    def read(self, layer: int, batch: TokenBatch, dtype: torch.dtype | None = None):
        """K and V of the batch's positions as values, [tokens][kv heads][head dim] each."""
        ref = self._layer(layer)
        dtype = self.dtype if dtype is None else dtype
        code = _code(dtype, "the output")
        self._on_device(batch.slots)
        k = torch.empty((batch.nTokens, self.headCountKv, self.headDim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        rc = lib().at_kvb_read(context(self.device.index), ref, batch._ref, code, k.data_ptr(), v.data_ptr())
        if rc:
            _lib.check(rc)
        return k, v

    def attention(self, layer: int, batch: TokenBatch, q: torch.Tensor, scale: float | None = None, window: int = 0,
                  out: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of q ([tokens][heads][head dim], float32, float16 or
        bfloat16) over the cached keys of each token's sequence, its own
        included (append first). window > 0: the last `window` keys only.
        scale defaults to 1 / sqrt(head dim)."""
        ref = self._layer(layer)
        if q.dim() != 3 or q.shape[0] != batch.nTokens or q.shape[2] != self.headDim:
            _bad(f"q must be [{batch.nTokens}][heads][{self.headDim}], got {tuple(q.shape)}")
        code = _code(q.dtype, "q")
        s = q.stride()
        if s[2] != 1:
            _bad("q's last dimension must be contiguous")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.dtype != q.dtype or out.shape != q.shape or not out.is_contiguous():
            _bad("out must be contiguous and of q's type and shape")
        self._on_device(q, out, batch.slots)
        window = int(window)
        if window < 0:
            _bad("window must not be negative")
        heads, window = q.shape[1], min(window, INT32_MAX)  # positions fit 31 bits: a longer window hides nothing either
        index, L = self.device.index, lib()
        ctx, need = context(index), C.c_size_t()
        rc = L.at_kvb_attention_workspace(ctx, ref, batch._ref, heads, window, C.byref(need))
        if rc:
            _lib.check(rc)
        n = need.value
        ws = self._workspace(_current_stream(index), n).data_ptr() if n else None
        rc = L.at_kvb_attention(ctx, ref, batch._ref, code, heads, q.data_ptr(), s[0], s[1], out.data_ptr(),
                                self._scale if scale is None else float(scale), window, ws, n)
        if rc:
            _lib.check(rc)
        return out

    def check(self) -> None:
        """Raises when a kernel met a slot, position or page outside its range,
        or an append that it could not make, since the last check (waits for
        the device). A cache wrapped without a status tensor cannot tell."""
        if self.status is None:
            return
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise IllegalStateException(_lib.AT_ERR_STATE, "block KV cache: " + " and ".join(
                m for b, m in ((_lib.KVB_BAD_SEQ, "a slot, start or offset out of range (its sequence was skipped)"),
                               (_lib.KVB_STALLED, "a wait inside a kernel that ran out (its output is not valid)"),
                               (_lib.KVB_BAD_BLOCK, "a page outside the pool (writes dropped, reads NaN)"),
                               (_lib.KVB_STALE_TAIL, "an append inside a block whose older rows the tail no longer has (not written there)"))
                if bits & b))
