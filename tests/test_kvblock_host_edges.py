"""Host side of the block-quantized KV cache: numbers that its structures cannot hold (no GPU needed)."""
import pytest
import torch

from auratensor_b200 import _lib
from auratensor_b200.kvblock import TokenBatch


@pytest.mark.parametrize("args", [([1 << 32], [0], [1]), ([0], [1 << 63], [1]), ([0], [(1 << 63) - 1], [1]), ([0, 1], [0, 0], [1 << 31, 1]),
                                  ([0], [0], [1 << 31])])
def test_numbers_that_do_not_fit_are_refused(args):
    """Slot 2^32 must not become slot 0."""
    with pytest.raises(_lib.IllegalArgumentException, match="fit"):
        TokenBatch.of(*args)


class OnDevice:
    """What TokenBatch asks of a tensor, on a device of choice."""
    is_cuda = True

    def __init__(self, n, dtype, device):
        self.n, self.dtype, self.device = n, dtype, device

    def numel(self):
        return self.n

    def get_device(self):
        return self.device

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 0


@pytest.mark.parametrize("devices", [(0, 1, 0), (0, 0, 1), (1, 0, 0), (1, 2, 3)])
def test_descriptors_on_several_devices_are_refused(devices):
    """A kernel would read another GPU's memory."""
    def batch(a, b, c):
        return TokenBatch(OnDevice(1, torch.int32, a), OnDevice(1, torch.int64, b), OnDevice(2, torch.int32, c), 1, 1, 1)

    assert batch(1, 1, 1).nSeqs == 1
    with pytest.raises(_lib.IllegalArgumentException, match="one device"):
        batch(*devices)
