"""Scores token sequences with a block-quantized KV cache: the log probability
of every token given those before it, through the paged int8 cache, the
attention over it and the log-probability operator, next to the same scores
through ``LlamaModel`` with its FP32 cache.

    python -m auratensor_b200.score                                   # small synthetic model, 4 texts
    python -m auratensor_b200.score --model llama-3.2-1b --tokens 500 --block 32
    python -m auratensor_b200.score --gguf model.gguf --ids 1,15043,29892
    python -m auratensor_b200.score --projections bf16                # prompts on the tensor cores

``BlockLlama`` is the model's forward pass (inference/LlamaModel.java:141-308)
put together from the library's operators, for any number of sequences at once:
prompts of different lengths and decode steps are the same call. Output: one
JSON line.
"""
from __future__ import annotations

import argparse
import json

import numpy as np
import torch

from . import synth
from ._lib import AT_ERR_INVALID_ARG, AT_ERR_STATE, IllegalArgumentException, IllegalStateException
from .core import DType, Kernels, Tensor
from .gguf import GgufFile
from .inference import LlamaConfig, LlamaModel
from .kvblock import BlockKvCache, TokenBatch
from .quant import ORIENT_N, ORIENT_T, Q4_0, Q8_0, QMatrix
from .scoring import LogProbs

_CODECS = {Q4_0.TYPE: Q4_0, Q8_0.TYPE: Q8_0}
GEMV_ROWS = 8  # tokens that one FP32 projection (GEMV) takes at a time


def _f32(t: dict, device) -> torch.Tensor:
    data = torch.as_tensor(np.ascontiguousarray(t["data"]) if not isinstance(t["data"], torch.Tensor) else t["data"]).to(device)
    return data.view(torch.uint8).reshape(-1).view(torch.float32).contiguous()


class BlockLlama:
    """A Llama-family model over a BlockKvCache. tensors: {name: {"type", "data"}}
    in the reference's layout (Q4_0 or Q8_0 matrices, F32 norms). projections:
    "auto" multiplies in FP32 while a call has at most 8 tokens and on the
    tensor cores (bf16 operands) above, so a token's logits move in the third
    digit with how many others share the call; "f32" always multiplies in FP32,
    8 tokens at a time, as LlamaModel's steps do."""

    def __init__(self, config: LlamaConfig, tensors: dict, nBlocks: int, maxSeqs: int, blockTokens: int = 64, device=None,
                 projections: str = "auto"):
        if projections not in ("auto", "f32"):
            raise IllegalArgumentException(AT_ERR_INVALID_ARG, f"projections must be auto or f32, got {projections}")
        self.projections = projections
        self.config = c = config
        self.device = dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        hd, d = c.headDim(), c.embeddingLength
        q, kv = c.headCount * hd, c.headCountKv * hd

        def matrix(name, orient, rows, cols):
            return QMatrix(tensors[name]["type"], orient, rows, cols, tensors[name]["data"])

        self.layers = []
        for i in range(c.blockCount):
            p = f"blk.{i}."
            self.layers.append({
                "q": matrix(p + "attn_q.weight", ORIENT_T, d, q), "k": matrix(p + "attn_k.weight", ORIENT_T, d, kv),
                "v": matrix(p + "attn_v.weight", ORIENT_T, d, kv), "o": matrix(p + "attn_output.weight", ORIENT_T, q, d),
                "gate": matrix(p + "ffn_gate.weight", ORIENT_N, c.feedForwardLength, d),
                "up": matrix(p + "ffn_up.weight", ORIENT_N, c.feedForwardLength, d),
                "down": matrix(p + "ffn_down.weight", ORIENT_N, d, c.feedForwardLength),
                "attn_norm": _f32(tensors[p + "attn_norm.weight"], dev), "ffn_norm": _f32(tensors[p + "ffn_norm.weight"], dev)})
        self.out_norm = _f32(tensors["output_norm.weight"], dev)
        self.head = matrix("output.weight", ORIENT_N, c.vocabSize, d)
        emb = tensors["token_embd.weight"]
        self._codec = _CODECS[emb["type"]]
        raw = emb["data"] if isinstance(emb["data"], torch.Tensor) else torch.from_numpy(np.ascontiguousarray(emb["data"]))
        self._embd = raw.to(dev).reshape(c.vocabSize, -1)  # the rows' raw blocks
        # RopeCache (inference/RopeCache.java:154-177): angles from double powers, cos and sin per pair
        freq = (float(np.float32(c.ropeFrequencyBase)) ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)).float()
        angle = (torch.arange(c.contextLength, dtype=torch.float32)[:, None] * freq[None]).double()
        self._cos, self._sin = angle.cos().float().to(dev), angle.sin().float().to(dev)
        per_seq = -(-c.contextLength // blockTokens)
        self.cache = BlockKvCache.allocate(c.blockCount, nBlocks, c.headCountKv, hd, maxSeqs, per_seq, blockTokens, torch.float32, dev)

    def _project(self, m: QMatrix, x: torch.Tensor, tokens: int | None = None) -> torch.Tensor:
        """x: all of a call's tokens, or some of `tokens`."""
        n = x.shape[0]
        if self.projections == "auto" and (tokens or n) > GEMV_ROWS:
            return m.gemm(x)
        if n <= GEMV_ROWS:
            return m.gemv(x)
        y = torch.empty((n, m.out_features), dtype=torch.float32, device=x.device)
        for i in range(0, n, GEMV_ROWS):
            m.gemv(x[i:i + GEMV_ROWS], y[i:i + GEMV_ROWS])
        return y

    def _norm(self, x: torch.Tensor, w: torch.Tensor) -> None:
        Kernels.rmsNormInPlace(Tensor.wrap(x, DType.FP32, x.shape), Tensor.wrap(w, DType.FP32, w.shape), self.config.rmsNormEpsilon)

    def _rope(self, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
        """Pairs (2 i, 2 i + 1) of every head turned by their position's angle."""
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)

    def _check(self, sequences) -> None:
        """What LlamaModel refuses: ids and positions index tables on the device."""
        for _, start, toks in sequences:
            bad = next((t for t in toks if not 0 <= int(t) < self.config.vocabSize), None)
            if bad is not None:
                raise IllegalArgumentException(AT_ERR_INVALID_ARG, f"token id {bad} out of range")
            if start < 0:
                raise IllegalArgumentException(AT_ERR_INVALID_ARG, "negative position")
            if start + len(toks) > self.config.contextLength:
                raise IllegalStateException(AT_ERR_STATE, f"position {start + len(toks) - 1} exceeds maxContext {self.config.contextLength}")

    def forward(self, sequences) -> torch.Tensor:
        """sequences: [(slot, start, token ids)], one run of consecutive tokens
        each; reserves their pages, appends them and returns the logits of every
        token, [tokens][vocab] on the device."""
        x = self._hidden(sequences)
        return self._project(self.head, x)

    def _hidden(self, sequences) -> torch.Tensor:
        """forward up to the output matrix."""
        self._check(sequences)
        c, hd = self.config, self.config.headDim()
        slots, starts = [s for s, _, _ in sequences], [p for _, p, _ in sequences]
        counts = [len(t) for _, _, t in sequences]
        for slot, start, toks in sequences:
            self.cache.reserve(slot, start + len(toks))
        batch = TokenBatch.of(slots, starts, counts, self.device)
        ids = torch.tensor([int(t) for _, _, toks in sequences for t in toks], dtype=torch.int64).to(self.device)
        pos = torch.tensor([p + i for p, n in zip(starts, counts) for i in range(n)], dtype=torch.int64).to(self.device)
        n = ids.numel()
        x = self._codec.dequantToFloat(self._embd[ids].reshape(-1), None, n * c.embeddingLength).view(n, c.embeddingLength)
        cos, sin = self._cos[pos][:, None], self._sin[pos][:, None]
        for i, w in enumerate(self.layers):
            self._norm(x, w["attn_norm"])  # in place: the residual stream is the normed one, as the reference's
            q = self._rope(self._project(w["q"], x).view(n, c.headCount, hd), cos, sin)
            k = self._rope(self._project(w["k"], x).view(n, c.headCountKv, hd), cos, sin)
            v = self._project(w["v"], x).view(n, c.headCountKv, hd)
            self.cache.append(i, batch, k, v)
            y = self.cache.attention(i, batch, q)
            x = x + self._project(w["o"], y.reshape(n, -1))
            self._norm(x, w["ffn_norm"])
            g = self._project(w["gate"], x)
            Kernels.siluInPlaceSegment(g, g.numel())
            x = x + self._project(w["down"], g * self._project(w["up"], x))
        self._norm(x, self.out_norm)
        return x

    def score(self, texts, top: int = 0, chunk: int = 512):
        """Log probabilities of each text's tokens 1.. given those before them
        (LogProbs per text, None for a text of less than two), in slots 0..,
        `chunk` tokens of each per call. The logits of one text's chunk are held
        at a time."""
        for slot in range(len(texts)):
            self.cache.release(slot)
        parts = [[] for _ in texts]
        longest = max((len(t) for t in texts), default=0)
        for at in range(0, longest, chunk):
            runs = [(s, at, t[at:at + chunk]) for s, t in enumerate(texts) if len(t) > at]
            x, row = self._hidden(runs), 0
            for slot, start, toks in runs:
                follow = torch.tensor([int(t) for t in texts[slot][start + 1:start + len(toks) + 1]], dtype=torch.int32).to(self.device)
                if follow.numel():
                    parts[slot].append(LogProbs.of(self._project(self.head, x[row:row + follow.numel()], x.shape[0]), follow, top))
                row += len(toks)

        def cat(xs):
            return None if xs[0] is None else torch.cat(xs)

        fields = ("logProb", "logSumExp", "entropy", "topIds", "topLogProbs")
        return [LogProbs(*(cat([getattr(r, f) for r in p]) for f in fields)) if p else None for p in parts]


def main(argv=None) -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--model", default="tiny", choices=["tiny", "tiny-q8", "llama-3.2-1b"], help="synthetic model (random weights)")
    ap.add_argument("--gguf", help="a GGUF file in the reference's layout instead")
    ap.add_argument("--ids", help="token ids to score, comma-separated (default: random texts)")
    ap.add_argument("--tokens", type=int, default=60, help="length of the longest random text")
    ap.add_argument("--texts", type=int, default=4)
    ap.add_argument("--block", type=int, default=64, help="tokens per cache block: 16, 32, 64 or 128")
    ap.add_argument("--projections", default="f32", choices=["f32", "bf16"],
                    help="f32: as the FP32 cache's model, so that the difference is the cache's; bf16: prompts on the tensor cores")
    args = ap.parse_args(argv)
    if args.texts < 1:
        ap.error("--texts must be at least 1")
    if args.ids is not None and len(args.ids.split(",")) < 2:
        ap.error("--ids needs two ids at least: each but the first is scored")
    torch.cuda.set_device(0)
    if args.gguf:
        with GgufFile.open(args.gguf) as g:
            cfg = LlamaConfig.fromGguf(g.metadata)
            tensors = {t.name: {"type": t.type, "data": np.array(g.tensorData(t), dtype=np.uint8)} for t in g.tensor_infos}
        if "output.weight" not in tensors:
            tensors["output.weight"] = tensors["token_embd.weight"]
    else:
        shape = {"tiny": synth.TINY, "tiny-q8": synth.TINY_Q8, "llama-3.2-1b": synth.LLAMA32_1B}[args.model]
        if shape.ctx < args.tokens:
            import dataclasses
            shape = dataclasses.replace(shape, ctx=args.tokens)
        cfg = LlamaConfig.fromShape(shape)
        gen = torch.Generator(device="cuda").manual_seed(0)
        tensors = {n: {"type": t, "data": synth.generate_torch_tensor(dims, t, gen, "cuda")} for n, dims, t in shape.tensor_dims()}
    rng = np.random.default_rng(1)
    texts = ([[int(t) for t in args.ids.split(",")]] if args.ids is not None else
             [rng.integers(0, cfg.vocabSize, size=max(2, args.tokens - 7 * i)).tolist() for i in range(args.texts)])
    blocks = sum(-(-len(t) // args.block) for t in texts)
    model = BlockLlama(cfg, tensors, blocks, len(texts), args.block, projections="f32" if args.projections == "f32" else "auto")
    scores = model.score(texts)
    model.cache.check()
    # the same texts through the FP32 cache, token by token
    ref = LlamaModel(cfg, tensors)
    exact = []
    for t in texts:
        ref.kvCache().reset()
        exact.append([])
        for p, tok in enumerate(t[:-1]):
            ref.forwardStepDevice(tok, p)
            exact[-1].append(ref.logProbs([t[p + 1]]).logProb)
    exact = [torch.cat(e) for e in exact]
    got = torch.cat([s.logProb for s in scores])
    per_token = 2 * cfg.blockCount * cfg.headCountKv * (cfg.headDim() + 4 / args.block)
    print(json.dumps({
        "model": args.gguf or args.model, "texts": [len(t) for t in texts], "block_tokens": args.block, "projections": args.projections,
        "mean_log_prob": round(float(got.mean()), 6), "mean_log_prob_f32_cache": round(float(torch.cat(exact).mean()), 6),
        "max_difference": round(float((got - torch.cat(exact)).abs().max()), 6),
        "mean_entropy": round(float(torch.cat([s.entropy for s in scores]).mean()), 6),
        "kv_bytes_per_token": per_token, "kv_bytes_per_token_f32": 2 * cfg.blockCount * cfg.headCountKv * cfg.headDim() * 4}))


if __name__ == "__main__":
    main()
