"""Host side of the block-quantized KV cache: numbers that its structures cannot hold (no GPU needed)."""
import pytest

from auratensor_b200 import _lib
from auratensor_b200.kvblock import TokenBatch


@pytest.mark.parametrize("args", [([1 << 32], [0], [1]), ([0], [1 << 63], [1]), ([0], [(1 << 63) - 1], [1]), ([0, 1], [0, 0], [1 << 31, 1]),
                                  ([0], [0], [1 << 31])])
def test_numbers_that_do_not_fit_are_refused(args):
    """Slot 2^32 must not become slot 0."""
    with pytest.raises(_lib.IllegalArgumentException, match="fit"):
        TokenBatch.of(*args)
