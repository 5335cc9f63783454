"""LlamaModel.logProbs: which logits it scores."""
import ctypes as C

import pytest
import torch

from auratensor_b200 import _lib, synth
from auratensor_b200.core import context
from auratensor_b200.inference import LlamaConfig, LlamaModel, SamplerConfig
from auratensor_b200.scheduler import BatchScheduler

pytestmark = pytest.mark.gpu


def model(batch=3):
    return LlamaModel(LlamaConfig.fromShape(synth.TINY), synth.generate_numpy(synth.TINY, seed=7), max_batch=batch)


def test_rows_that_the_last_step_did_not_compute_are_refused(cuda):
    m = model()
    with pytest.raises(_lib.IllegalStateException, match="computed 0 rows"):
        m.logProbs([1])
    m.forwardBatch([3, 4, 5], [0, 0, 0])
    assert m.logProbs([1, 2, 3]).logProb.shape == (3,)
    m.forwardBatch([6, 7], [1, 1])
    assert m.logProbs([1, 2]).logProb.shape == (2,)
    with pytest.raises(_lib.IllegalStateException, match="computed 2 rows"):
        m.logProbs([1, 2, 3])
    m.forwardStep(8, 2)
    with pytest.raises(_lib.IllegalStateException, match="computed 1 rows"):
        m.logProbs([1, 2])
    m.generateSampled([1, 2, 3], [3, 2, 1], 2, [SamplerConfig()] * 3)
    assert m.logProbs([1, 2, 3]).logProb.shape == (3,)
    m.generate(1, 5, 2)
    with pytest.raises(_lib.IllegalStateException, match="computed 1 rows"):
        m.logProbs([1, 2])
    s = BatchScheduler(m)
    for _ in range(2):
        s.submit([1, 2, 3], 4, SamplerConfig())
    s.step()
    assert m.logProbs([1, 2]).logProb.shape == (2,)


def test_penalised_logits_are_what_is_scored(cuda):
    """Sampling changes the logits in place, as the reference's Sampler: the scores are then of what it left."""
    import numpy as np
    m = model(1)
    m.forwardStep(3, 0)
    before = m.logitsDevice()[0].double()
    plain = m.logProbs([9]).logProb.item()
    m.sample([SamplerConfig(repetitionPenalty=2.0)], [np.array([9], dtype=np.int32)])
    after = before.clone()
    after[9] = after[9] / 2 if after[9] > 0 else after[9] * 2
    got = m.logProbs([9]).logProb.item()
    assert abs(got - after.log_softmax(0)[9].item()) < 1e-4 and abs(plain - before.log_softmax(0)[9].item()) < 1e-4 and got != plain


def test_scores_wait_for_steps_in_flight_on_another_stream(cuda):
    """generate(wait=False) returns before its steps have run."""
    m = model(1)
    m.generate(1, 0, 3)
    want = m.logProbs([5]).logProb.clone()
    m.generate(7, 3, 1)
    assert not torch.equal(m.logProbs([5]).logProb, want)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        context()
        torch.cuda._sleep(200_000_000)
        m.generate(1, 0, 3, wait=False)
    context()  # any operator in between
    got = m.logProbs([5]).logProb
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_scores_and_steps_of_a_model_with_a_context_of_its_own_are_in_order(cuda):
    """As under tensor parallelism: the model's stream is not the operators'."""
    own = C.c_void_p()
    _lib.call("at_ctx_create", 0, C.byref(own))
    m = LlamaModel(LlamaConfig.fromShape(synth.TINY), synth.generate_numpy(synth.TINY, seed=7), ctx=own.value)
    stream, side = C.c_void_p(), torch.cuda.Stream()
    _lib.call("at_ctx_stream", own, C.byref(stream))
    m.generate(7, 3, 1)
    other = m.logProbs([5]).logProb.clone()
    m.generate(1, 0, 3)
    want = m.logProbs([5]).logProb.clone()
    torch.cuda.synchronize()
    assert not torch.equal(want, other)
    # a step that is late: the scores wait for it
    m.generate(7, 3, 1)
    with torch.cuda.stream(torch.cuda.ExternalStream(stream.value)):
        torch.cuda._sleep(200_000_000)
    m.generate(1, 0, 3, wait=False)
    with torch.cuda.stream(side):
        got = m.logProbs([5]).logProb
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    # scores that are late: the next step waits for them
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        got = m.logProbs([5]).logProb
    m.generate(7, 3, 1)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    m.close()
    _lib.call("at_ctx_destroy", own)


def test_scores_can_be_captured(cuda):
    m = model(1)
    m.forwardStep(3, 0)
    want = m.logProbs([5], top=3)
    m.forwardStep(4, 0)
    tok = torch.tensor([5], dtype=torch.int32, device=cuda)
    m.logProbs(tok)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = m.logProbs(tok, top=3)
    m.forwardStep(3, 0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(r.logProb, want.logProb) and torch.equal(r.topIds, want.topIds)
