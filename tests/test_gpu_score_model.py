"""What the scoring model and its command compare, and what they hold (auratensor_b200/score.py)."""
import dataclasses
import json
import subprocess
import sys

import numpy as np
import pytest
import torch

from auratensor_b200 import _lib, synth
from auratensor_b200.inference import LlamaConfig
from auratensor_b200.score import BlockLlama
from test_gpu_block_llama import oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [synth.TINY, synth.TINY_Q8], ids=["q4_0", "q8_0"])
def test_prompts_in_fp32_follow_the_oracle_as_steps_do(shape, cuda):
    """The rule of the token-by-token tests, 1e-3 of the logit range, for whole prompts that share a call."""
    block, texts = 32, [synth.prompt_ids(shape, 70 + i, n).tolist() for i, n in enumerate((50, 3, 33))]
    t = synth.generate_numpy(shape, seed=8)
    gpu = BlockLlama(LlamaConfig.fromShape(shape), t, 16, 3, block, projections="f32")
    got = gpu.forward([(s, 0, text) for s, text in enumerate(texts)]).cpu().numpy()
    gpu.cache.check()
    at = 0
    for text in texts:
        orc = oracle(shape, t, block)
        want = np.stack([orc.forward_step(tok, p) for p, tok in enumerate(text)])
        assert np.max(np.abs(got[at:at + len(text)] - want)) <= 1e-3 * (want.max() - want.min())
        at += len(text)


def test_fp32_logits_do_not_depend_on_what_shares_the_call(cuda):
    shape = synth.TINY
    texts = [synth.prompt_ids(shape, 80 + i, n).tolist() for i, n in enumerate((7, 50, 20))]
    gpu = BlockLlama(LlamaConfig.fromShape(shape), synth.generate_numpy(shape, seed=9), 16, 3, 16, projections="f32")
    together = gpu.forward([(s, 0, text) for s, text in enumerate(texts)])
    for s in range(3):
        gpu.cache.release(s)
    alone = torch.cat([gpu.forward([(s, 0, text)]) for s, text in enumerate(texts)])
    spread = float(alone.max() - alone.min())
    assert float((together - alone).abs().max()) <= 1e-4 * spread  # sums in another order


def test_scores_hold_the_logits_of_one_text_at_a_time(cuda):
    shape = dataclasses.replace(synth.TINY, vocab=32000)
    texts = [synth.prompt_ids(shape, 90 + i, 60).tolist() for i in range(16)]
    gpu = BlockLlama(LlamaConfig.fromShape(shape), synth.generate_numpy(shape, seed=10), 16, 16, 64)
    gpu.score(texts)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    gpu.score(texts)
    all_logits = 16 * 60 * 32000 * 4
    assert torch.cuda.max_memory_allocated() - base < all_logits / 4


def test_projections_are_checked(cuda):
    with pytest.raises(_lib.IllegalArgumentException, match="projections"):
        BlockLlama(LlamaConfig.fromShape(synth.TINY), {}, 1, 1, projections="f16")


def test_command_compares_the_caches_in_fp32(cuda):
    def run(*args):
        r = subprocess.run([sys.executable, "-m", "auratensor_b200.score", "--texts", "2", "--tokens", "60", "--block", "16", *args],
                           capture_output=True, text=True, timeout=240)
        assert r.returncode == 0, r.stderr[-2000:]
        return json.loads(r.stdout.strip().splitlines()[-1])

    d, b = run(), run("--projections", "bf16")
    assert d["projections"] == "f32" and b["projections"] == "bf16"
    assert d["mean_log_prob_f32_cache"] == b["mean_log_prob_f32_cache"] and 0 < d["max_difference"] < 0.05
