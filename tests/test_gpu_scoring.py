"""Log probabilities, entropy and top alternatives (at_logprobs) against 64 bits.

Tolerances: logsumexp and log probabilities are differences of FP32 numbers of
size at most |m| + log V, plus the log of a sum whose V terms are off by 2^-22
each and added in FP32 over at most a few thousand terms per thread:
4e-6 (1 + |m| + log V) in all; the entropy sums terms of size up to its own
value and one logarithm: 2e-5 (1 + H). Ids are exact.
"""
import math

import numpy as np
import pytest
import torch

from auratensor_b200 import _lib
from auratensor_b200.scoring import LogProbs

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def check(x, tokens, top):
    r = LogProbs.of(x, tokens, top)
    xd = x.double()
    logp = torch.log_softmax(xd, -1)
    p = logp.exp()
    m = xd.amax(-1).abs()
    tol = 4e-6 * (1 + m + math.log(x.shape[1]))
    lse = torch.logsumexp(xd, -1)
    assert torch.all((r.logSumExp - lse).abs() <= tol)
    h = -torch.special.xlogy(p, p).sum(-1)
    assert torch.all((r.entropy - h).abs() <= 2e-5 * (1 + h)), float(((r.entropy - h).abs() / (1 + h)).max())
    if tokens is not None:
        want = logp.gather(1, tokens.long()[:, None])[:, 0].float()  # -inf below FP32's range
        assert torch.all((want == r.logProb) | ((r.logProb - want).abs() <= 2 * tol + 2.0 ** -22 * want.abs()))
    if top:
        order = torch.sort(xd, dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(r.topIds.long(), order)
        want = logp.gather(1, order).float()
        assert torch.all((want == r.topLogProbs) | ((r.topLogProbs - want).abs() <= (2 * tol)[:, None] + 2.0 ** -22 * want.abs()))
    return r


def logits(rows, vocab, seed, cuda, dtype=F32, std=3.0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = (torch.randn((rows, vocab), generator=g, device=cuda) * std).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device=cuda, dtype=torch.int32)
    return x, t


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 31), (2, 33), (7, 257), (1, 4097), (3, 32000), (9, 32001), (1, 128256), (300, 1000), (2, 151937)])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_rows(rows, vocab, top, dtype, cuda):
    x, t = logits(rows, vocab, rows + vocab, cuda, dtype)
    check(x, t, min(top, vocab))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("pad", [1, 2, 3, 5, 8])
def test_strided_unaligned_rows(pad, dtype, cuda):
    x, t = logits(6, 5003 + 2 * pad, 70 + pad, cuda, dtype)
    view = x[:, pad:pad + 5003]
    t = t % 5003
    r = check(view, t, 7)
    again = LogProbs.of(view.contiguous(), t, 7)
    assert torch.equal(r.topIds, again.topIds)
    tol = dict(rtol=1e-5, atol=1e-5)  # the two add the same terms in different orders
    torch.testing.assert_close(r.logProb, again.logProb, **tol)
    torch.testing.assert_close(r.entropy, again.entropy, **tol)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ties_go_to_the_lower_id(dtype, cuda):
    vocab = 40007
    x = torch.zeros((6, vocab), device=cuda, dtype=dtype)
    x[1] = -2
    x[1, 39990:] = 1                                    # 17 equal maxima at the end
    x[2] = torch.arange(vocab, device=cuda).remainder(3).to(dtype)
    x[3, ::2] = -0.0                                    # equal to +0
    x[4, 20000:20010] = 5
    x[4, 19990] = 4
    x[5] = torch.arange(vocab, 0, -1, device=cuda).float().div(vocab).to(dtype)
    check(x, torch.arange(6, device=cuda, dtype=torch.int32), 32)


@pytest.mark.parametrize("step", [1, -1])
def test_sorted_rows(step, cuda):
    """Every large value in one place of the row."""
    x = (torch.arange(128256, device=cuda).float() * 1e-3 * step).repeat(2, 1).contiguous()
    check(x, torch.tensor([0, 128255], device=cuda, dtype=torch.int32), 32)


def test_masked_tokens_have_no_probability(cuda):
    x, t = logits(8, 32000, 5, cuda)
    x[:, 100:31000] = -math.inf
    x[1] = -math.inf
    x[1, 7] = 3.0                                       # one token allowed
    x[2, :] = -math.inf
    x[2, 31998:] = 1.0
    t[0] = 500
    r = check(x, t, 20)
    assert r.logProb[0] == -math.inf and abs(float(r.entropy[1])) < 1e-6 and r.topLogProbs[1, 0] == 0
    assert torch.equal(r.topIds[1, 1:4], torch.tensor([0, 1, 2], device=cuda, dtype=torch.int32))


def test_rows_without_a_distribution(cuda):
    x, t = logits(5, 3000, 6, cuda)
    x[0] = -math.inf
    x[1, 17] = math.nan
    x[2, 40] = math.inf
    x[3, 41] = math.nan
    x[3, 40] = math.inf
    t[4] = -1
    r = LogProbs.of(x, t, 3)
    assert r.logSumExp[0] == -math.inf and r.entropy[0] == 0 and r.logProb[0] == -math.inf and torch.all(r.topLogProbs[0] == -math.inf)
    assert r.topIds[0].tolist() == [0, 1, 2]
    for row in (1, 2, 3):
        assert torch.isnan(r.logSumExp[row]) and torch.isnan(r.entropy[row]) and torch.isnan(r.logProb[row]) and torch.isnan(r.topLogProbs[row]).all()
    assert r.topIds[1, 0] == 17 and r.topIds[2, 0] == 40 and r.topIds[3, :2].tolist() == [41, 40]
    assert torch.isnan(r.logProb[4]) and torch.isfinite(r.entropy[4])
    assert torch.isnan(LogProbs.of(x[4:], torch.tensor([3000], device=cuda, dtype=torch.int32)).logProb).all()


def test_large_and_small_logits(cuda):
    x, t = logits(4, 50000, 8, cuda)
    x[0] *= 1e4
    x[1] += 1e6
    x[2] *= 1e-6
    x[3] = -3e38
    x[3, 9] = 3e38
    check(x, t, 5)


def test_offsets_past_two_gigabytes(cuda):
    """A row that begins more than 2^32 bytes into the logits."""
    big = torch.empty((2, (1 << 31) + 64), dtype=BF16, device=cuda)
    x, t = logits(2, 2000, 9, cuda, BF16)
    view = big[:, :2000]
    view.copy_(x)
    check(view, t, 5)


def test_streams_and_inputs_unchanged(cuda):
    x, t = logits(64, 32000, 10, cuda)
    keep = x.clone()
    want = LogProbs.of(x, t, 5)
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got.append(LogProbs.of(x.clone(), t, 5))
    torch.cuda.synchronize()
    for g in got:
        for a, b in ((g.logProb, want.logProb), (g.entropy, want.entropy), (g.topIds, want.topIds), (g.topLogProbs, want.topLogProbs)):
            assert torch.equal(a, b)
    assert torch.equal(x, keep)


def test_no_tokens_and_no_rows(cuda):
    x, t = logits(3, 100, 11, cuda)
    r = LogProbs.of(x)
    assert r.logProb is None and r.topIds is None and r.topLogProbs is None
    assert torch.equal(r.entropy, LogProbs.of(x, t, 4).entropy)
    r = LogProbs.of(x[:0], t[:0], 4)
    assert r.logProb.shape == (0,) and r.topIds.shape == (0, 4)


def test_refusals(cuda):
    x, t = logits(3, 100, 12, cuda)
    for call in (lambda: LogProbs.of(x.cpu(), t), lambda: LogProbs.of(x[0], t), lambda: LogProbs.of(x, t.long()), lambda: LogProbs.of(x, t[:2]),
                 lambda: LogProbs.of(x.t().contiguous().t(), t), lambda: LogProbs.of(x, t, -1), lambda: LogProbs.of(x, t, 101),
                 lambda: LogProbs.of(x[:1].expand(3, 100), t)):
        with pytest.raises(_lib.IllegalArgumentException):
            call()
    for call in (lambda: LogProbs.of(x.double(), t), lambda: LogProbs.of(x, t, 33)):
        with pytest.raises(_lib.UnsupportedOperationException):
            call()
