"""LlamaModel.logProbs: which logits it scores."""
import pytest

from auratensor_b200 import _lib, synth
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
