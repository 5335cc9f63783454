"""The block-quantized KV cache (at_kvb_*): writing, reading back and attention, against a 64-bit restatement.

Tolerances, from the arithmetic:
  - what is written is exact: the quantizer is three FP32 operations (division,
    product, round-half-even), restated in numpy's FP32; read back in FP32 it is
    one exact product rounded once;
  - FP32 attention: a score is off by at most about 2^-20 sum|q k| (a two-part
    split of q, FP32 sums), which moves a weight by twice that relatively; for
    these inputs sum|q k| scale stays below 24, so an output is off by at most
    5e-5 sum_j w_j |v_j|, the splits and sums of the weights included;
  - F16/BF16 attention: the weights are rounded to 11 bits (2^-11 of the same
    sum) and the output once more to its type.
"""
import numpy as np
import pytest
import torch

import kvblock_ref as ref
from auratensor_b200 import _lib
from auratensor_b200.kvblock import BlockKvCache, TokenBatch

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ROUND = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def heads(shape, seed, dtype, cuda):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return torch.randn(shape, generator=g, device=cuda).to(dtype)


def new_cache(dtype=F32, seqs=4, heads_kv=2, hd=128, block=64, blocks=40, per_seq=12, layers=1):
    return BlockKvCache.allocate(layers, blocks, heads_kv, hd, seqs, per_seq, block, dtype)


def f64(t):
    return t.float().cpu().numpy().astype(np.float64)


def f32(t):
    return t.float().cpu().numpy()


def check_values(cache, layer, slot, k, v):
    """Positions 0..len(k)-1 of the slot hold exactly what the restatement holds."""
    gk, gv = cache.read(layer, TokenBatch.of([slot], [0], [len(k)]), F32)
    for got, x in ((gk, k), (gv, v)):
        want = ref.cache_values(f32(x), cache.blockTokens).astype(np.float32)
        np.testing.assert_array_equal(f32(got), want)


# ---------------------------------------------------------------- write and read
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hd,block", [(64, 16), (128, 16), (64, 32), (128, 64), (64, 128), (128, 128)])
@pytest.mark.parametrize("cuts", [[1], [129], [1, 1, 1, 5], [37, 300], [64, 64, 1], [5, 123, 130, 1, 61]])
def test_written_blocks_are_exact(hd, block, cuts, dtype, cuda):
    cache = new_cache(dtype, hd=hd, block=block, blocks=64, per_seq=24 * 2)
    n = sum(cuts)
    k, v = heads((n, 2, hd), 1, dtype, cuda), heads((n, 2, hd), 2, dtype, cuda) * 3
    k *= torch.linspace(0.2, 2, n, device=cuda)[:, None, None].to(dtype)  # later tokens raise the maxima
    cache.reserve(2, n)
    at = 0
    for c in cuts:
        cache.append(0, TokenBatch.of([2], [at], [c]), k[at:at + c], v[at:at + c])
        at += c
        check_values(cache, 0, 2, k[:at], v[:at])
    cache.check()


def test_contents_do_not_depend_on_how_appends_cut_them(cuda):
    n = 333
    k, v = heads((n, 2, 128), 3, BF16, cuda), heads((n, 2, 128), 4, BF16, cuda)
    rng = np.random.default_rng(5)
    got = []
    for trial in range(4):
        cache = new_cache(BF16, block=32, per_seq=12)
        cache.reserve(1, n)
        at = 0
        while at < n:
            c = n if trial == 0 else int(min(n - at, rng.integers(1, [2, 40, 150][trial - 1])))
            cache.append(0, TokenBatch.of([1], [at], [c]), k[at:at + c], v[at:at + c])
            at += c
        pages = cache.table[1, :-(-n // 32)].long()
        got.append((cache.kBlocks[0, pages].reshape(-1, 2, 32, 128)[:10], cache.kScales[0, pages], cache.vScales[0, pages]))
    for g in got[1:]:
        for a, b in zip(got[0], g):
            assert torch.equal(a, b)


@pytest.mark.parametrize("back", [1, 7, 36, 60])
def test_rewinding_overwrites_what_follows(back, cuda):
    """A later append may start in the last block written or the one before it."""
    block, n = 32, 100
    cache = new_cache(F32, hd=64, block=block)
    k, v = heads((n, 2, 64), 6, F32, cuda) * 4, heads((n, 2, 64), 7, F32, cuda)
    cache.reserve(0, 200)
    for at, c in ((0, 70), (70, 30)):
        cache.append(0, TokenBatch.of([0], [at], [c]), k[at:at + c], v[at:at + c])
    at = n - back if (n - back) // block >= (n - 1) // block - 1 else block * ((n - 1) // block - 1)
    k2, v2 = heads((9, 2, 64), 8, F32, cuda), heads((9, 2, 64), 9, F32, cuda)  # smaller: the old maxima must not stay
    cache.append(0, TokenBatch.of([0], [at], [9]), k2, v2)
    check_values(cache, 0, 0, torch.cat([k[:at], k2]), torch.cat([v[:at], v2]))


def test_batches_of_ragged_runs_layers_and_empty_sequences(cuda):
    cache = new_cache(F16, seqs=6, hd=64, block=16, blocks=80, per_seq=20, layers=2)
    runs = {3: (0, 50), 0: (0, 1), 5: (0, 0), 1: (0, 17), 4: (0, 16)}
    data = {}
    for slot, (_, n) in runs.items():
        cache.reserve(slot, n + 40)
        data[slot] = [heads((n + 40, 2, 64), 10 * slot + i, F16, cuda) for i in range(4)]
    for step in range(2):
        slots, starts, counts = list(runs), [runs[s][0] for s in runs], [runs[s][1] for s in runs]
        batch = TokenBatch.of(slots, starts, counts)
        for layer in range(2):
            k = torch.cat([data[s][2 * layer][a:a + n] for s, a, n in zip(slots, starts, counts)])
            v = torch.cat([data[s][2 * layer + 1][a:a + n] for s, a, n in zip(slots, starts, counts)])
            cache.append(layer, batch, k, v)
        for layer in range(2):
            for s in slots:
                n = runs[s][0] + runs[s][1]
                check_values(cache, layer, s, data[s][2 * layer][:n], data[s][2 * layer + 1][:n])
        runs = {s: (a + n, (7 * s + 3) % 20) for s, (a, n) in runs.items()}
    cache.append(0, TokenBatch.of([], [], []), torch.empty((0, 2, 64), dtype=F16, device=cuda), torch.empty((0, 2, 64), dtype=F16, device=cuda))
    cache.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided_and_unaligned_sources(dtype, cuda):
    cache = new_cache(dtype, heads_kv=3, hd=64, block=32)
    n = 45
    qkv = heads((n, 11, 64), 11, dtype, cuda)                      # fused projection rows
    odd = heads((3, n, 67), 12, dtype, cuda)[:, :, 2:66].transpose(0, 1)  # head-major, odd strides, unaligned start
    cache.reserve(0, n)
    cache.append(0, TokenBatch.of([0], [0], [n]), qkv[:, 5:8], odd)
    check_values(cache, 0, 0, qkv[:, 5:8], odd)


@pytest.mark.parametrize("case", ["zeros", "subnormal", "smallest", "largest", "negative zero"])
def test_extreme_blocks(case, cuda):
    x = {"zeros": torch.zeros(40, 2, 64), "subnormal": torch.full((40, 2, 64), 1e-41), "smallest": torch.full((40, 2, 64), 1.6e-36),
         "largest": torch.linspace(-3.4e38, 3.4e38, 40 * 128).reshape(40, 2, 64), "negative zero": -torch.zeros(40, 2, 64)}[case].to(cuda)
    cache = new_cache(F32, hd=64, block=32)
    cache.reserve(0, 40)
    cache.append(0, TokenBatch.of([0], [0], [40]), x, x)
    check_values(cache, 0, 0, x, x)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_non_finite_value_poisons_its_block_only(bad, cuda):
    cache = new_cache(F32, hd=64, block=32)
    k, v = heads((100, 2, 64), 13, F32, cuda), heads((100, 2, 64), 14, F32, cuda)
    k[40, 1, 3] = bad
    cache.reserve(0, 100)
    for at in range(0, 100, 20):  # later rows of the poisoned block arrive after it
        cache.append(0, TokenBatch.of([0], [at], [20]), k[at:at + 20], v[at:at + 20])
    gk, gv = cache.read(0, TokenBatch.of([0], [0], [100]))
    nan = torch.isnan(gk)
    assert nan[32:64, 1].all() and nan.sum() == 32 * 64 and not torch.isnan(gv).any()
    # attention: the rows that see the block are NaN (of the heads that read KV head 1), the others are not
    q = heads((100, 4, 64), 15, F32, cuda)
    y = torch.isnan(cache.attention(0, TokenBatch.of([0], [0], [100]), q))
    assert y[32:, 2:].all() and not y[:32].any() and not y[:, :2].any()
    y = torch.isnan(cache.attention(0, TokenBatch.of([0], [0], [100]), q, window=10))
    assert y[32:73, 2:].all() and not y[:32].any() and not y[73:].any() and not y[:, :2].any()
    for p in (31, 32, 99):  # single tokens
        y = torch.isnan(cache.attention(0, TokenBatch.of([0], [p], [1]), q[p:p + 1]))
        assert y[:, 2:].all() == (p >= 32) and not y[:, :2].any()


# ---------------------------------------------------------------- attention
def run_attention(cuda, dtype, hd, block, kvh, group, runs, window=0, seed=0, scale=None, q_scale=1.0, kv_scale=1.0):
    """runs: [(start, count)] per sequence; compares the call with the restatement over what the cache holds."""
    seqs = len(runs)
    per_seq = max(1, max(-(-(s + n) // block) for s, n in runs))
    cache = BlockKvCache.allocate(1, sum(-(-(s + n) // block) for s, n in runs) + 3, kvh, hd, seqs + 1, per_seq, block, dtype)
    slots = [(i + 1) % (seqs + 1) for i in range(seqs)][::-1]
    keys = []
    for i, (s, n) in enumerate(runs):
        cache.reserve(slots[i], s + n)
        k = heads((s + n, kvh, hd), seed + 100 + i, dtype, cuda) * kv_scale
        v = heads((s + n, kvh, hd), seed + 200 + i, dtype, cuda) * kv_scale
        v *= torch.logspace(-2, 1, kvh * hd, device=cuda).reshape(kvh, hd).to(dtype)
        cache.append(0, TokenBatch.of([slots[i]], [0], [s + n]), k, v)
        keys.append((ref.cache_values(f32(k), block), ref.cache_values(f32(v), block)))
    total = sum(n for _, n in runs)
    q = heads((total, kvh * group, hd), seed + 1, dtype, cuda) * q_scale
    batch = TokenBatch.of(slots, [s for s, _ in runs], [n for _, n in runs])
    y = f64(cache.attention(0, batch, q, scale=scale, window=window))
    cache.check()
    qd, at = f64(q), 0
    sc = hd ** -0.5 if scale is None else scale
    for i, (s, n) in enumerate(runs):
        want, mag = ref.attention(qd[at:at + n], *keys[i], s, sc, window)
        tol = 5e-5 * mag + ROUND[dtype] * np.abs(want) + (0 if dtype == F32 else 2.0 ** -11 * mag)
        err = np.abs(y[at:at + n] - want)
        assert np.all(err <= tol + 1e-30), (i, float(np.max(err / (tol + 1e-30))))
        at += n
    return y


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_single_tokens(hd, block, dtype, cuda):
    run_attention(cuda, dtype, hd, block, 2, 4, [(0, 1), (1, 1), (15, 1), (63, 1), (64, 1), (200, 1), (517, 1), (1030, 1)])


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 16, 20])
def test_head_groups(group, cuda):
    run_attention(cuda, F32, 64, 32, 2, group, [(130, 1), (7, 1)])
    run_attention(cuda, BF16, 128, 64, 1, group, [(70, 3), (0, 2), (300, 1)])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hd,block,group", [(128, 64, 4), (64, 16, 8), (128, 128, 3), (64, 32, 1)])
def test_prompts(hd, block, group, dtype, cuda):
    run_attention(cuda, dtype, hd, block, 2, group, [(0, 150), (0, 1), (33, 97), (5, 0), (260, 129), (200, 2)])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [1, 2, 17, 64, 100, 4096])
def test_windows(window, dtype, cuda):
    run_attention(cuda, dtype, 64, 32, 2, 4, [(300, 1), (0, 1), (64, 1), (129, 1)], window=window)
    run_attention(cuda, dtype, 128, 64, 1, 2, [(0, 200), (170, 67)], window=window)


def test_long_single_token_is_split(cuda):
    run_attention(cuda, F32, 64, 64, 1, 4, [(9000, 1)])
    run_attention(cuda, BF16, 128, 128, 1, 8, [(5001, 1), (12000, 1), (0, 1)])


@pytest.mark.parametrize("q_scale,kv_scale,scale", [(1e-3, 1.0, None), (30.0, 0.01, None), (1e4, 1e-5, 1.0), (1.0, 1e4, 1e-5), (1e-6, 1e-6, None)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ranges(q_scale, kv_scale, scale, dtype, cuda):
    """Values far from 1 in either operand: what is held in fewer bits on the way must not leave its range."""
    run_attention(cuda, dtype, 64, 32, 1, 4, [(100, 1), (333, 1)], scale=scale, q_scale=q_scale, kv_scale=kv_scale)
    run_attention(cuda, dtype, 64, 32, 1, 4, [(40, 130)], scale=scale, q_scale=q_scale, kv_scale=kv_scale)


@pytest.mark.parametrize("n", [1, 40])
def test_blocks_of_very_different_scales(n, cuda):
    """The values' scale changes from block to block by factors of 1e4, keys stay alike."""
    cache = new_cache(F32, seqs=1, heads_kv=1, hd=64, block=16, blocks=20, per_seq=20)
    k, v = heads((200, 1, 64), 31, F32, cuda), heads((200, 1, 64), 32, F32, cuda)
    v *= (10.0 ** torch.tensor([(-4, 4, 0, -8, 2)[p // 16 % 5] for p in range(200)], device=cuda))[:, None, None]
    cache.reserve(0, 200)
    cache.append(0, TokenBatch.of([0], [0], [200]), k, v)
    q = heads((n, 4, 64), 33, F32, cuda)
    y = f64(cache.attention(0, TokenBatch.of([0], [200 - n], [n]), q))
    want, mag = ref.attention(f64(q), ref.cache_values(f32(k), 16), ref.cache_values(f32(v), 16), 200 - n, 0.125)
    assert np.all(np.abs(y - want) <= 5e-5 * mag + 2.0 ** -24 * np.abs(want))


def test_hidden_keys_do_not_matter(cuda):
    """Everything a query does not see may hold anything: later blocks with NaN scales, the rest of the open block, other pages."""
    for n in (1, 40):
        cache = new_cache(F32, seqs=2, hd=64, block=32, blocks=30, per_seq=10)
        k, v = heads((300, 2, 64), 21, F32, cuda), heads((300, 2, 64), 22, F32, cuda)
        q = heads((n, 4, 64), 23, F32, cuda)
        cache.reserve(0, 300)
        cache.append(0, TokenBatch.of([0], [0], [300]), k, v)
        batch = TokenBatch.of([0], [151 - n], [n])
        want = cache.attention(0, batch, q)
        keep = cache.table[0, :5].long()  # positions 0..159; 151.. are hidden
        other = torch.ones(cache.nBlocks, dtype=torch.bool, device=cuda)
        other[keep] = False
        cache.kScales[0, other] = float("nan")
        cache.vScales[0, other] = float("inf")
        cache.kBlocks[0, keep[4], :, 23:] = 127
        cache.vBlocks[0, keep[4], :, 23:] = -128
        assert torch.equal(cache.attention(0, batch, q), want)


def test_pages_past_two_gigabytes(cuda):
    """Page addresses beyond 32 bits: 70000 pages of 64 KB."""
    cache = BlockKvCache.allocate(1, 70000, 8, 128, 2, 8, 64, BF16)
    pages = torch.tensor([69999, 3, 40000, 65535, 65536], dtype=torch.int32, device=cuda)
    cache.table[1, :5] = pages
    k, v = heads((290, 8, 128), 41, BF16, cuda), heads((290, 8, 128), 42, BF16, cuda)
    cache.append(0, TokenBatch.of([1], [0], [290]), k, v)
    check_values(cache, 0, 1, k, v)
    kd, vd = ref.cache_values(f32(k), 64), ref.cache_values(f32(v), 64)
    for n in (1, 30):
        q = heads((n, 8, 128), 43, BF16, cuda)
        y = f64(cache.attention(0, TokenBatch.of([1], [290 - n], [n]), q))
        want, mag = ref.attention(f64(q), kd, vd, 290 - n, 128 ** -0.5)
        assert np.all(np.abs(y - want) <= (5e-5 + 2.0 ** -11) * mag + 2.0 ** -8 * np.abs(want))


def test_strided_queries_and_given_output(cuda):
    for n in (1, 50):
        cache = new_cache(F32, hd=64, block=32)
        k, v = heads((120, 2, 64), 51, F32, cuda), heads((120, 2, 64), 52, F32, cuda)
        cache.reserve(0, 120)
        cache.append(0, TokenBatch.of([0], [0], [120]), k, v)
        wide = heads((n, 13, 67), 53, F32, cuda)
        q = wide[:, 2:8, 1:65]
        batch = TokenBatch.of([0], [120 - n], [n])
        out = torch.empty((n, 6, 64), device=cuda)
        assert cache.attention(0, batch, q, out=out) is out
        assert torch.equal(out, cache.attention(0, batch, q.contiguous()))


def test_other_streams_and_repeatability(cuda):
    cache = new_cache(BF16, seqs=8, hd=128, block=64, blocks=100, per_seq=12)
    k, v = heads((8 * 700, 2, 128), 61, BF16, cuda), heads((8 * 700, 2, 128), 62, BF16, cuda)
    for s in range(8):
        cache.reserve(s, 701)
    cache.append(0, TokenBatch.of(range(8), [0] * 8, [700] * 8), k, v)
    q = heads((8, 8, 128), 63, BF16, cuda)
    batch = TokenBatch.of(range(8), [699] * 8, [1] * 8)
    want = cache.attention(0, batch, q)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for rep in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                q2 = q.clone().mul_(1.0)  # made on this stream
                got.append(cache.attention(0, batch, q2))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_captured_steps_advance_on_the_device(cuda):
    """A graph of append + attention whose positions advance on the device gives the eager results."""
    n0, steps = 60, 10
    k, v = heads((n0 + steps, 2, 64), 71, F32, cuda), heads((n0 + steps, 2, 64), 72, F32, cuda)
    qs = heads((steps, 4, 64), 73, F32, cuda)

    def filled():
        cache = new_cache(F32, seqs=1, hd=64, block=32)
        cache.reserve(0, n0 + steps)
        cache.append(0, TokenBatch.of([0], [0], [n0]), k[:n0], v[:n0])
        return cache

    eager = filled()
    want = []
    for i in range(steps):
        batch = TokenBatch.of([0], [n0 + i], [1])
        eager.append(0, batch, k[n0 + i:n0 + i + 1], v[n0 + i:n0 + i + 1])
        want.append(eager.attention(0, batch, qs[i:i + 1]))
    cache = filled()
    one = TokenBatch.of([0], [n0], [1])
    batch = TokenBatch(one.slots, one.starts.clone(), one.offsets, 1, 1, n0 + steps)
    kk, vv, qq = k[:1].clone(), v[:1].clone(), qs[:1].clone()
    cache.attention(0, batch, qq)  # warm-up before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(0, batch, kk, vv)
        y = cache.attention(0, batch, qq)
        batch.starts.add_(1)
    batch.starts.fill_(n0)
    for i in range(steps):
        kk.copy_(k[n0 + i:n0 + i + 1]); vv.copy_(v[n0 + i:n0 + i + 1]); qq.copy_(qs[i:i + 1])
        graph.replay()
        torch.testing.assert_close(y, want[i], rtol=1e-5, atol=1e-6)
    assert torch.equal(cache.kBlocks, eager.kBlocks) and torch.equal(cache.vScales, eager.vScales)


# ---------------------------------------------------------------- refusals
def test_bad_device_descriptors_are_reported_not_followed(cuda):
    cache = new_cache(F32, hd=64, block=32)
    k = heads((3, 2, 64), 81, F32, cuda)
    q = heads((3, 4, 64), 82, F32, cuda)
    cache.reserve(0, 100)
    cache.append(0, TokenBatch.of([0], [0], [3]), k, k)
    cache.check()
    before = cache.kBlocks.clone()
    dev = dict(dtype=torch.int32, device=cuda)
    good = TokenBatch.of([0], [0], [3])
    for slots, starts, offsets in (([4], [0], [0, 3]), ([-1], [0], [0, 3]), ([0], [-1], [0, 3]), ([0], [12 * 32 - 2], [0, 3]),
                                   ([0], [1 << 40], [0, 3]), ([0], [0], [1, 4]), ([0], [0], [3, 0]), ([0], [0], [-1, 2])):
        batch = TokenBatch(torch.tensor(slots, **dev), torch.tensor(starts, dtype=torch.int64, device=cuda), torch.tensor(offsets, **dev), 3, 3, 100)
        for call in (lambda: cache.append(0, batch, k, k), lambda: cache.read(0, batch), lambda: cache.attention(0, batch, q)):
            call()
            with pytest.raises(_lib.IllegalStateException, match="out of range"):
                cache.check()
    assert torch.equal(before, cache.kBlocks)
    cache.table[0, 0] = cache.nBlocks
    for call in (lambda: cache.append(0, good, k, k), lambda: cache.read(0, good), lambda: cache.attention(0, good, q),
                 lambda: cache.attention(0, TokenBatch.of([0], [0], [1]), q[:1])):
        r = call()
        assert r is None or torch.isnan(r if torch.is_tensor(r) else r[0]).all()
        with pytest.raises(_lib.IllegalStateException, match="outside the pool"):
            cache.check()
    assert torch.equal(before, cache.kBlocks)


def test_refusals(cuda):
    cache = new_cache(F32, hd=64, block=32)
    k, q = heads((2, 2, 64), 1, F32, cuda), heads((2, 4, 64), 2, F32, cuda)
    batch = TokenBatch.of([0], [0], [2])
    cache.reserve(0, 2)
    bad = _lib.IllegalArgumentException
    for call in (lambda: cache.append(1, batch, k, k), lambda: cache.append(0, batch, k.half(), k), lambda: cache.append(0, batch, k[:1], k),
                 lambda: cache.append(0, batch, k, k.transpose(1, 2).contiguous().transpose(1, 2)), lambda: cache.append(0, batch, k.cpu(), k),
                 lambda: cache.attention(-1, batch, q), lambda: cache.attention(0, batch, q[:, :3]), lambda: cache.attention(0, batch, q[:1]),
                 lambda: cache.attention(0, batch, q[:, :, :32]), lambda: cache.attention(0, batch, q, window=-1),
                 lambda: cache.attention(0, batch, q, scale=0.0), lambda: cache.attention(0, batch, q, scale=float("nan")),
                 lambda: cache.attention(0, batch, q, out=torch.empty_like(q, dtype=F16)), lambda: cache.reserve(9, 1),
                 lambda: TokenBatch(batch.slots.long(), batch.starts, batch.offsets, 2, 2, 2),
                 lambda: TokenBatch(batch.slots, batch.starts, batch.offsets[:1], 2, 2, 2)):
        with pytest.raises(bad):
            call()
    with pytest.raises(_lib.UnsupportedOperationException):
        cache.attention(0, batch, q.double())
    with pytest.raises(_lib.UnsupportedOperationException):
        BlockKvCache.allocate(1, 4, 2, 96, 1, 4)
    for call in (lambda: cache.append(0, TokenBatch.of([0], [383], [2]), k, k), lambda: cache.reserve(0, 12 * 32 + 1),
                 lambda: [cache.reserve(s, 12 * 32) for s in range(4)]):
        with pytest.raises(_lib.IllegalStateException):
            call()
    reader = BlockKvCache.wrap(cache.kBlocks, cache.vBlocks, cache.kScales, cache.vScales, cache.table)
    reader.read(0, batch)
    with pytest.raises(_lib.IllegalStateException):
        reader.append(0, batch, k, k)
    with pytest.raises(_lib.IllegalStateException):
        reader.reserve(0, 1)
    with pytest.raises(bad):
        BlockKvCache.wrap(cache.kBlocks, cache.vBlocks, cache.kScales[:, :1], cache.vScales, cache.table)
    free = cache.freeBlocks()
    cache.release(0)
    assert cache.freeBlocks() > free


def test_reserve_and_release_give_distinct_pages(cuda):
    cache = new_cache(F32, seqs=3, hd=64, block=16, blocks=9, per_seq=6)
    cache.reserve(0, 40)
    cache.reserve(1, 33)
    cache.reserve(0, 41)
    assert cache.freeBlocks() == 3
    used = cache.table[0, :3].tolist() + cache.table[1, :3].tolist()
    assert len(set(used)) == 6
    cache.release(0)
    cache.reserve(2, 96)
    assert cache.freeBlocks() == 0 and not set(cache.table[2].tolist()) & set(cache.table[1, :3].tolist())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,step", [(1, 40), (150, 1), (150, 32), (150, 128), (260, 17)])
def test_scores_that_grow_along_the_keys(n, step, dtype, cuda):
    """Each `step` keys the scores rise by 12 (in powers of e): the running reference has to follow, inside tiles and
    across them, and what came before fades without upsetting the sums; in the second half they fall again."""
    total = 300
    cache = new_cache(dtype, seqs=1, heads_kv=1, hd=64, block=16, blocks=20, per_seq=20)
    level = torch.arange(total, device=cuda) // step
    level = torch.minimum(level, level.max() - level).float() * 12
    k = heads((total, 1, 64), 91, F32, cuda) * 0.1
    k[:, 0, 0] = level  # the first dimension alone carries the level
    k, v = k.to(dtype), heads((total, 1, 64), 92, dtype, cuda)
    q = heads((n, 4, 64), 93, F32, cuda) * 0.1
    q[:, :, 0] = 8.0
    q = q.to(dtype)
    cache.reserve(0, total)
    cache.append(0, TokenBatch.of([0], [0], [total]), k, v)
    y = f64(cache.attention(0, TokenBatch.of([0], [total - n], [n]), q))
    kd, vd = ref.cache_values(f32(k), 16), ref.cache_values(f32(v), 16)
    want, mag = ref.attention(f64(q), kd, vd, total - n, 0.125)
    # a score of size |s| is rounded to FP32 a few times: 2^-22 |s| more on its weight
    smax = float(np.abs(f64(q)[..., 0]).max() * np.abs(kd[:, 0, 0]).max() * 0.125)
    tol = (5e-5 + 2.0 ** -21 * smax + (0 if dtype == F32 else 2.0 ** -11)) * mag + ROUND[dtype] * np.abs(want)
    assert np.all(np.abs(y - want) <= tol), float((np.abs(y - want) / tol).max())
    cache.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,hd", [(1, 128), (3, 64), (150, 128), (70, 64)])
def test_queries_with_one_large_component(n, hd, dtype, cuda):
    """A component of 4096 that meets zero keys adds nothing, and what stands beside it (0.25 and more of 1) keeps its
    digits: the row is scaled as a whole, and its other components still lie 2^13 above where f16 ends."""
    total = 200
    cache = new_cache(dtype, seqs=1, heads_kv=2, hd=hd, block=32, blocks=8, per_seq=8)
    k, v = heads((total, 2, hd), 95, dtype, cuda), heads((total, 2, hd), 96, dtype, cuda)
    k[:, :, 5] = 0
    q = heads((n, 8, hd), 97, F32, cuda)
    q = torch.where(q >= 0, q + 0.25, q - 0.25)
    q[:, :, 5] = torch.where(q[:, :, 5] > 0, 4096.0, -4096.0)
    q = q.to(dtype)
    cache.reserve(0, total)
    cache.append(0, TokenBatch.of([0], [0], [total]), k, v)
    y = f64(cache.attention(0, TokenBatch.of([0], [total - n], [n]), q))
    want, mag = ref.attention(f64(q), ref.cache_values(f32(k), 32), ref.cache_values(f32(v), 32), total - n, hd ** -0.5)
    tol = (5e-5 + (0 if dtype == F32 else 2.0 ** -11)) * mag + ROUND[dtype] * np.abs(want)
    assert np.all(np.abs(y - want) <= tol), float((np.abs(y - want) / tol).max())
    cache.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [0, 33])
@pytest.mark.parametrize("group,n", [(3, 100), (48, 5), (100, 2), (128, 3)])
def test_query_tiles_with_padding_rows(group, n, window, dtype, cuda):
    """Groups that leave rows of a tile without a token, and last tiles that are not full."""
    run_attention(cuda, dtype, 64, 32, 1, group, [(130, n), (0, n + 1)], window=window, seed=group)


def test_more_query_heads_than_a_tile_has_rows_are_refused(cuda):
    cache = new_cache(F16, seqs=1, heads_kv=1, hd=64, block=16, blocks=4, per_seq=4)
    cache.reserve(0, 1)
    with pytest.raises(_lib.UnsupportedOperationException, match="128 query heads"):
        cache.attention(0, TokenBatch.of([0], [0], [1]), heads((1, 129, 64), 1, F16, cuda))


@pytest.mark.parametrize("seqs,n", [(1, 130), (150, 1)])
@pytest.mark.parametrize("hd", [64, 128])
def test_float32_sums_stay_exact_over_long_caches(seqs, n, hd, cuda):
    """The tensor cores truncate what they accumulate, some 2^-24 of the sum with each product. Pieces of at most 16
    products added in FP32 are off by 16 2^-23 = 1.9e-6 at most, the scores (2^-20 each, independent) by less than 1e-6;
    one chain over 12000 keys by 1e-5 and more."""
    total = 12000
    cache = new_cache(F32, seqs=seqs, heads_kv=1, hd=hd, block=64, blocks=190, per_seq=190)
    k, v = heads((total, 1, hd), 98, F32, cuda), heads((total, 1, hd), 99, F32, cuda) + 0.5
    cache.reserve(0, total)
    cache.append(0, TokenBatch.of([0], [0], [total]), k, v)
    cache.table[:] = cache.table[0].clone()  # every sequence reads the same pages
    q = heads((n, 4, hd), 100, F32, cuda)
    batch = TokenBatch.of(range(seqs), [total - n] * seqs, [n] * seqs)
    y = f64(cache.attention(0, batch, q.repeat(seqs, 1, 1)))
    want, _ = ref.attention(f64(q), ref.cache_values(f32(k), 64), ref.cache_values(f32(v), 64), total - n, hd ** -0.5)
    for got in y.reshape(seqs, n, 4, hd):
        assert np.linalg.norm(got - want) <= 3e-6 * np.linalg.norm(want), np.linalg.norm(got - want) / np.linalg.norm(want)
    cache.check()
