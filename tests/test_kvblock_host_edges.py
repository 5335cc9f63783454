"""Host side of the block-quantized KV cache: numbers that its structures cannot hold (no GPU needed)."""
import os
import subprocess
import sys

import pytest
import torch

from auratensor_b200 import _lib
from auratensor_b200.kvblock import TokenBatch

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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


@pytest.mark.parametrize("kv_heads", [0, -1])
def test_a_cache_without_heads_is_an_error_not_a_crash(kv_heads, built_lib):
    """In a process of its own: a division by zero would end it."""
    code = f"""
import ctypes as C
from auratensor_b200 import _lib
buf = C.create_string_buffer(4096)
ctx = C.addressof(buf)  # looked at only once the cache is found valid
at = ctx + 16 - ctx % 16
c = _lib.KvBlocksC(0, {kv_heads}, 64, 16, 4, 1, 4, 0, at, at, at, at, None, None, None, None, at, None)
b = _lib.TokenBatchC(1, 1, 1, 0, 1, at, at, at)
n = C.c_size_t(7)
calls = (("at_kvb_attention_workspace", (4, 0, C.byref(n))), ("at_kvb_attention", (0, 4, at, 256, 64, at, 1.0, 0, None, 0)),
         ("at_kvb_append", (at, 64, 64, at, 64, 64)), ("at_kvb_read", (0, at, at)))
for name, args in calls:
    rc = getattr(_lib.lib(), name)(ctx, C.addressof(c), C.addressof(b), *args)
    assert rc == _lib.AT_ERR_INVALID_ARG and "dimensions" in _lib.last_error(), (name, rc, _lib.last_error())
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=_ROOT)
    assert r.returncode == 0, (r.returncode, r.stderr[-800:])
