"""Host side of the block-quantized KV cache and of the log probabilities: refusals that need no GPU."""
import ctypes as C

import pytest

from auratensor_b200 import _lib
from auratensor_b200.kvblock import BlockKvCache, TokenBatch


def test_null_arguments_are_refused(built_lib):
    calls = {"at_kvb_append": (None, None, None, None, 0, 0, None, 0, 0), "at_kvb_read": (None, None, None, 0, None, None),
             "at_kvb_attention": (None, None, None, 0, 1, None, 0, 0, None, 1.0, 0, None, 0),
             "at_kvb_attention_workspace": (None, None, None, 1, 0, None),
             "at_logprobs": (None, None, 0, 1, 1, 1, None, 0, None, None, None, None, None)}
    for name, args in calls.items():
        assert getattr(built_lib, name)(*args) == _lib.AT_ERR_INVALID_ARG, name
        assert "null" in _lib.last_error()


def test_struct_layouts_match_the_header():
    # 8 ints then 10 pointers; 4 ints, one int64, 3 pointers
    assert C.sizeof(_lib.KvBlocksC) == 8 * 4 + 10 * 8 and _lib.KvBlocksC.k.offset == 32 and _lib.KvBlocksC.status.offset == 104
    assert C.sizeof(_lib.TokenBatchC) == 4 * 4 + 8 + 3 * 8 and _lib.TokenBatchC.max_end.offset == 16 and _lib.TokenBatchC.offsets.offset == 40


@pytest.mark.parametrize("args", [([0, 1], [0], [1, 1]), ([0, 0], [0, 0], [1, 1]), ([-1], [0], [1]), ([0], [-1], [1]), ([0], [0], [-1])])
def test_batches_from_lists_are_checked(args):
    with pytest.raises(_lib.IllegalArgumentException):
        TokenBatch.of(*args)


@pytest.mark.parametrize("change,exc", [({"layers": 0}, _lib.IllegalArgumentException), ({"nBlocks": 0}, _lib.IllegalArgumentException),
                                        ({"headDim": 80}, _lib.UnsupportedOperationException), ({"blockTokens": 48}, _lib.IllegalArgumentException)])
def test_allocations_are_checked(change, exc):
    with pytest.raises(exc):
        BlockKvCache.allocate(**{**dict(layers=1, nBlocks=4, headCountKv=2, headDim=64, maxSeqs=1, maxBlocks=4), **change})
