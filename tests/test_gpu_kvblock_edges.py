"""The block cache where a call is at, or past, the edge of what it may ask for: sizes that are only upper bounds,
positions without pages, rewinds, values of extreme scales. Tolerances are those of test_gpu_kvblock.py."""
import numpy as np
import pytest
import torch

import kvblock_ref as ref
from auratensor_b200 import _lib
from auratensor_b200.kvblock import BlockKvCache, TokenBatch
from test_gpu_kvblock import BF16, F16, F32, ROUND, check_values, f32, f64, heads, new_cache

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- the host's sizes as upper bounds
def loose(batch, nTokens, maxTokens, maxEnd):
    return TokenBatch(batch.slots, batch.starts, batch.offsets, nTokens, maxTokens, maxEnd)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("counts,n_tokens,max_tokens", [((3,), 64, 64), ((10,), 512, 512), ((16,), 17, 17), ((1, 40, 16, 0), 160, 40),
                                                        ((1, 2), 400, 200), ((5, 130), 260, 130), ((1, 1), 9, 3)])
def test_sizes_may_be_upper_bounds(counts, n_tokens, max_tokens, dtype, cuda):
    """What a captured graph has: the sizes of the launch are the largest, the runs on the device are shorter."""
    seqs, group, prefix, total = len(counts), 4, 50, sum(counts)
    cache = new_cache(dtype, seqs=seqs, hd=64, block=32, blocks=60, per_seq=12)
    k, v = heads((seqs, 400, 2, 64), 101, dtype, cuda), heads((seqs, 400, 2, 64), 102, dtype, cuda)
    for s in range(seqs):
        cache.reserve(s, prefix + counts[s])
        cache.append(0, TokenBatch.of([s], [0], [prefix]), k[s, :prefix], v[s, :prefix])
    batch = loose(TokenBatch.of(range(seqs), [prefix] * seqs, counts), n_tokens, max_tokens, 12 * 32)
    pad = torch.zeros((n_tokens - total, 2, 64), dtype=dtype, device=cuda)
    new = [torch.cat([x[s, prefix:prefix + n] for s, n in enumerate(counts)] + [pad]) for x in (k, v)]
    cache.append(0, batch, *new)
    q = heads((n_tokens, 2 * group, 64), 103, dtype, cuda)
    y = cache.attention(0, batch, q, out=torch.full_like(q, float("nan")))
    gk, gv = cache.read(0, batch, F32)
    cache.check()
    y, qd, at = f64(y), f64(q), 0
    for s, n in enumerate(counts):
        check_values(cache, 0, s, k[s, :prefix + n], v[s, :prefix + n])
        kd, vd = (ref.cache_values(f32(x[s, :prefix + n]), 32) for x in (k, v))
        assert np.array_equal(f32(gk)[at:at + n], kd[prefix:].astype(np.float32)) and np.array_equal(f32(gv)[at:at + n], vd[prefix:].astype(np.float32))
        want, mag = ref.attention(qd[at:at + n], kd, vd, prefix, 0.125)
        tol = 5e-5 * mag + ROUND[dtype] * np.abs(want) + (0 if dtype == F32 else 2.0 ** -11 * mag)
        assert np.all(np.abs(y[at:at + n] - want) <= tol), s
        at += n


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_many_keys_without_values(dtype, cuda):
    """38000 keys whose values are all zero, then 1000 that have some: the zeros' weights count in full."""
    total, empty, n = 39000, 38000, 130
    cache = new_cache(dtype, seqs=1, heads_kv=1, hd=64, block=128, blocks=310, per_seq=310)
    k, v = heads((total, 1, 64), 121, F32, cuda) * 0.1, heads((total, 1, 64), 122, F32, cuda) + 1
    v[:empty] = 0
    k[:, 0, 0] = 1
    k[128:, 0, 0] = 1 + 4.1  # after the first tile the scores are 4.1 higher (in powers of e), 5.9 in powers of 2
    k, v = k.to(dtype), v.to(dtype)
    q = heads((n, 2, 64), 123, F32, cuda) * 0.01
    q[:, :, 0] = 8.0
    q = q.to(dtype)
    cache.reserve(0, total)
    cache.append(0, TokenBatch.of([0], [0], [total]), k, v)
    y = f64(cache.attention(0, TokenBatch.of([0], [total - n], [n]), q))
    want, mag = ref.attention(f64(q), ref.cache_values(f32(k), 128), ref.cache_values(f32(v), 128), total - n, 0.125)
    # a chain of 39000 keys in 16 bits: 128-key pieces, each off by 2^-23 of the sum
    tol = (5e-5 + (0 if dtype == F32 else 2.0 ** -11 + 39000 / 16 * 2.0 ** -23)) * mag + ROUND[dtype] * np.abs(want)
    assert np.all(np.abs(y - want) <= tol), float((np.abs(y - want) / tol).max())
    cache.check()


def test_a_bound_of_many_tokens_is_not_cut_to_32_bits(cuda):
    """2^27 tokens of 16 chunks each are 2^31 chunks."""
    bound, n = 1 << 27, 100
    cache = new_cache(F16, seqs=1, hd=128, block=128, blocks=4, per_seq=4)
    cache.reserve(0, n)
    row = heads((1, 2, 128), 111, F16, cuda)
    batch = loose(TokenBatch.of([0], [0], [n]), bound, bound, 512)
    cache.append(0, batch, row.expand(bound, 2, 128), row.expand(bound, 2, 128))
    cache.check()
    check_values(cache, 0, 0, row.expand(n, 2, 128), row.expand(n, 2, 128))


# ---------------------------------------------------------------- positions without a page
def test_positions_that_were_not_reserved_have_no_page(cuda):
    cache = new_cache(F32, seqs=3, hd=64, block=32)
    k, v = heads((40, 2, 64), 151, F32, cuda), heads((40, 2, 64), 152, F32, cuda)
    other, q = heads((40, 2, 64), 153, F32, cuda), heads((1, 4, 64), 154, F32, cuda)
    cache.reserve(0, 40)
    cache.append(0, TokenBatch.of([0], [0], [40]), k, v)
    cache.check()

    def refused(call):
        r = call()
        with pytest.raises(_lib.IllegalStateException, match="outside the pool"):
            cache.check()
        check_values(cache, 0, 0, k, v)
        return r

    refused(lambda: cache.append(0, TokenBatch.of([1], [0], [40]), other, other))   # nothing reserved
    cache.reserve(1, 10)
    refused(lambda: cache.append(0, TokenBatch.of([1], [20], [40]), other, other))  # past what was
    assert torch.isnan(refused(lambda: cache.read(0, TokenBatch.of([2], [0], [5])))[0]).all()
    assert torch.isnan(refused(lambda: cache.attention(0, TokenBatch.of([2], [0], [1]), q))).all()
    # a released slot's pages may be another's by now
    cache.release(1)
    cache.reserve(2, 40)
    cache.append(0, TokenBatch.of([2], [0], [40]), other, other)
    cache.check()
    refused(lambda: cache.append(0, TokenBatch.of([1], [0], [10]), k[:10], k[:10]))
    check_values(cache, 0, 2, other, other)
    cache.reserve(1, 10)  # reserved anew it is usable
    cache.append(0, TokenBatch.of([1], [0], [10]), other[:10], k[:10])
    cache.check()
    check_values(cache, 0, 1, other[:10], k[:10])


# ---------------------------------------------------------------- rewinding
def test_a_second_rewind_behind_the_kept_rows_is_reported(cuda):
    """0..99 in blocks of 32 keeps the originals of blocks 2 and 3. After a rewind into block 2 those of block 1 are
    still gone: an append inside it cannot quantize its older rows again and must not take block 3's for them."""
    cache = new_cache(F32, hd=64, block=32)
    k, v = heads((100, 2, 64), 131, F32, cuda) * 4, heads((100, 2, 64), 132, F32, cuda)
    small = heads((9, 2, 64), 133, F32, cuda)
    cache.reserve(0, 200)
    cache.append(0, TokenBatch.of([0], [0], [100]), k, v)
    cache.append(0, TokenBatch.of([0], [70], [9]), small, small)
    cache.check()
    page = int(cache.table[0, 1])
    before = [x[0, page].clone() for x in (cache.kBlocks, cache.vBlocks, cache.kScales, cache.vScales)]
    cache.append(0, TokenBatch.of([0], [40], [5]), small[:5], small[:5])
    with pytest.raises(_lib.IllegalStateException, match="older rows"):
        cache.check()
    for a, x in zip(before, (cache.kBlocks, cache.vBlocks, cache.kScales, cache.vScales)):
        assert torch.equal(a, x[0, page])
    check_values(cache, 0, 0, torch.cat([k[:70], small]), torch.cat([v[:70], small]))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_repeated_rewinds_within_the_kept_rows(dtype, cuda):
    """Inside a block whose originals are still kept, and at the first row of any block, as often as one likes."""
    cache = new_cache(dtype, hd=64, block=32)
    held_k, held_v = [heads((0, 2, 64), 1, dtype, cuda) for _ in range(2)]
    cache.reserve(0, 200)
    for i, (at, c) in enumerate(((0, 100), (70, 9), (65, 3), (68, 40), (97, 2), (66, 1), (32, 50), (60, 4), (0, 33), (5, 1))):
        scale = 4.0 if i % 2 == 0 else 0.25
        k, v = heads((c, 2, 64), 140 + 2 * i, dtype, cuda) * scale, heads((c, 2, 64), 141 + 2 * i, dtype, cuda) * scale
        cache.append(0, TokenBatch.of([0], [at], [c]), k, v)
        cache.check()
        held_k, held_v = torch.cat([held_k[:at], k]), torch.cat([held_v[:at], v])
        check_values(cache, 0, 0, held_k, held_v)


def test_windows_of_more_than_31_bits(cuda):
    cache = new_cache(F32, hd=64, block=32)
    k, q = heads((50, 2, 64), 161, F32, cuda), heads((1, 4, 64), 162, F32, cuda)
    cache.reserve(0, 50)
    cache.append(0, TokenBatch.of([0], [0], [50]), k, k)
    batch = TokenBatch.of([0], [49], [1])
    want = cache.attention(0, batch, q)
    for window in ((1 << 32) + 5, 1 << 31, 1 << 40):
        assert torch.equal(cache.attention(0, batch, q, window=window), want)
    with pytest.raises(_lib.IllegalArgumentException):
        cache.attention(0, batch, q, window=5 - (1 << 32))


def test_sizes_that_do_not_fit_are_refused(cuda):
    b = TokenBatch.of([0], [0], [3])
    for sizes in (((1 << 32) + 3, 3, 3), (3, (1 << 32) + 3, 3), (-1, 3, 3), (3, -1, 3), (3, 3, 1 << 64), (3, 3, -1)):
        with pytest.raises(_lib.IllegalArgumentException, match="must be in"):
            loose(b, *sizes)


def test_a_status_word_that_the_kernels_cannot_write_is_refused(cuda):
    """No call is made with these: a kernel would write to a host address."""
    c = new_cache(F32, hd=64, block=32)
    for status in (torch.zeros(1, dtype=torch.int32), torch.zeros(1, device=cuda), torch.zeros(0, dtype=torch.int32, device=cuda),
                   torch.zeros(1, dtype=torch.int64, device=cuda)):
        with pytest.raises(_lib.IllegalArgumentException, match="status"):
            BlockKvCache.wrap(c.kBlocks, c.vBlocks, c.kScales, c.vScales, c.table, dtype=F32, status=status)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    w = BlockKvCache.wrap(c.kBlocks, c.vBlocks, c.kScales, c.vScales, c.table, dtype=F32, status=status)
    w.read(0, TokenBatch.of([0], [0], [3]))  # nothing is reserved
    with pytest.raises(_lib.IllegalStateException, match="outside the pool"):
        w.check()
