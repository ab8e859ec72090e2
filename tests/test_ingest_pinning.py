"""What a registration of store memory that fails is taken for (no GPU needed: without one every registration fails)."""
import ctypes
import mmap

import pytest
import torch


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="registration does not fail for want of a GPU here")
def test_a_failed_registration_is_not_taken_for_a_system_that_refuses_all():
    from raydp_amd.ops import _hip
    lib, u64 = _hip.lib(), ctypes.c_uint64
    mem = mmap.mmap(-1, 8 << 20)
    base = ctypes.addressof(ctypes.c_char.from_buffer(mem))
    for _ in range(2):                        # (remembered, the second would be 0)
        rc = lib.rx_pin_range(u64(base), u64(8 << 20), u64(base), u64(4096), u64(2 << 20))
        assert rc > 1, rc                     # the HIP error: no device
    assert lib.rx_pin_range(u64(base), u64(8 << 20), u64(base - 4096), u64(4096), u64(2 << 20)) == -1
    lib.rx_unpin_arena(u64(base))
