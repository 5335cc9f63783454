"""The block cache, its attention and the log probabilities together, as a model's forward pass (auratensor_b200/score.py).

The oracle is the numpy restatement of the reference's model with its attention
reading K and V through the block quantizer's own restatement, so token by token
(FP32 projections) the FP32 rule of the other model tests holds: logits within
1e-3 of the oracle's logit range. Prompts run their projections on bf16 operands:
2e-2 of the range, the framework's prompt tolerance."""
import json
import subprocess
import sys

import numpy as np
import pytest
import torch

import kvblock_ref as kvb
from auratensor_b200 import _lib, synth
from auratensor_b200.inference import LlamaConfig, LlamaModel
from auratensor_b200.score import BlockLlama
from auratensor_b200.scoring import LogProbs
from oracle import ref

pytestmark = pytest.mark.gpu


class BlockRef(ref.LlamaModelRef):
    """The oracle with K and V as the block cache holds them."""
    block = 16

    def attention(self, L, pos, q):
        k, v = self.kv.k[L].copy(), self.kv.v[L].copy()
        for x in (self.kv.k[L], self.kv.v[L]):  # [kv head][position][dim]
            x[:, :pos + 1] = kvb.cache_values(np.ascontiguousarray(x[:, :pos + 1].transpose(1, 0, 2)), self.block).transpose(1, 0, 2)
        out = super().attention(L, pos, q)
        self.kv.k[L], self.kv.v[L] = k, v
        return out


def oracle(shape, t, block):
    cfg = ref.LlamaConfig(shape.ctx, shape.dim, shape.n_layers, shape.n_heads, shape.n_kv_heads, shape.ffn, shape.rope_theta, shape.eps, shape.vocab)
    m = BlockRef(cfg, t)
    m.block = block
    return m


def log_softmax(x):
    x = np.asarray(x, np.float64)
    return x - x.max(-1, keepdims=True) - np.log(np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True))


@pytest.mark.parametrize("shape", [synth.TINY, synth.TINY_Q8], ids=["q4_0", "q8_0"])
@pytest.mark.parametrize("block", [16, 64])
def test_teacher_forced_tokens(shape, block, cuda):
    t = synth.generate_numpy(shape, seed=5)
    gpu = BlockLlama(LlamaConfig.fromShape(shape), t, 16, 2, block)
    orc = oracle(shape, t, block)
    toks = synth.prompt_ids(shape, 5, 40).tolist()
    for p, tok in enumerate(toks):
        want = orc.forward_step(tok, p)
        got = gpu.forward([(1, p, [tok])])
        assert np.max(np.abs(got.cpu().numpy()[0] - want)) <= 1e-3 * (want.max() - want.min()), p
    gpu.cache.check()


def test_prompts_of_different_lengths_and_their_scores(cuda):
    shape, block = synth.TINY, 32
    t = synth.generate_numpy(shape, seed=6)
    gpu = BlockLlama(LlamaConfig.fromShape(shape), t, 16, 3, block)
    texts = [synth.prompt_ids(shape, 60 + i, n).tolist() for i, n in enumerate((50, 2, 33))]
    scores = gpu.score(texts, top=5, chunk=24)
    for text, s in zip(texts, scores):
        orc = oracle(shape, t, block)
        want = np.stack([orc.forward_step(tok, p) for p, tok in enumerate(text)])
        spread = want.max() - want.min()
        lp = log_softmax(want)
        follow = lp[np.arange(len(text) - 1), text[1:]]
        # two logits and the logsumexp each within 2e-2 of the range
        assert np.max(np.abs(s.logProb.cpu().numpy() - follow)) <= 4e-2 * spread
        assert s.topIds.shape == (len(text) - 1, 5) and torch.all(s.topLogProbs[:, :-1] >= s.topLogProbs[:, 1:])
    again = gpu.score(texts, top=5, chunk=24)  # the pages come back to the pool between texts
    for a, b in zip(scores, again):
        assert torch.equal(a.logProb, b.logProb) and torch.equal(a.topIds, b.topIds)


def test_log_probs_of_a_models_step(cuda):
    shape = synth.TINY
    model = LlamaModel(LlamaConfig.fromShape(shape), synth.generate_numpy(shape, seed=7), max_batch=3)
    logits = model.forwardBatch([3, 4, 5], [0, 0, 0])
    r = model.logProbs([9, 8, 7], top=4)
    want = log_softmax(logits)
    np.testing.assert_allclose(r.logProb.cpu().numpy(), want[[0, 1, 2], [9, 8, 7]], atol=1e-4)
    assert r.topIds.cpu().tolist() == [np.argsort(-row, kind="stable")[:4].tolist() for row in logits]
    assert np.array_equal(model.logitsDevice()[:3].cpu().numpy(), logits)
    assert isinstance(model.logProbs(), LogProbs) and model.logProbs().logProb is None
    with pytest.raises(_lib.IllegalArgumentException):
        model.logProbs([1, 2, 3, 4])


def test_command_line(cuda):
    out = subprocess.run([sys.executable, "-m", "auratensor_b200.score", "--texts", "2", "--tokens", "40", "--block", "16"],
                         capture_output=True, text=True, timeout=240)
    assert out.returncode == 0, out.stderr[-2000:]
    d = json.loads(out.stdout.strip().splitlines()[-1])
    # the two caches differ by the 8-bit rounding of K and V and the projections' bf16 operands
    assert d["texts"] == [40, 33] and abs(d["mean_log_prob"] - d["mean_log_prob_f32_cache"]) < 0.05
    assert d["kv_bytes_per_token"] < 0.26 * d["kv_bytes_per_token_f32"]
