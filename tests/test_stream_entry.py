"""rt_hip_create_on_stream without a device: refusals are statuses, not crashes (what it does on a device: tests/test_gpu_streams.py)."""
import ctypes as C

import pytest


def test_refusals_without_a_device(lib):
    from rustorch_amd import DeviceNotAvailable
    from rustorch_amd.executor import HipKernelExecutor
    assert lib.rt_hip_create_on_stream(0, None, None) == 1
    assert b"rt_hip_create_on_stream" in lib.rt_hip_last_error(None)
    ctx = C.c_void_p()
    for device in (-1, 4096):
        assert lib.rt_hip_create_on_stream(device, None, C.byref(ctx)) == 3 and not ctx.value
        with pytest.raises(DeviceNotAvailable):
            HipKernelExecutor(device, stream=0)
