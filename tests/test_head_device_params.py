"""The optimiser's parameters in device memory: their address is checked before a launch
reads doubles from it. Runs without a GPU."""
import ctypes

import pytest

from gemmaedge_amd import head as H
from gemmaedge_amd import sampler as S


@pytest.mark.parametrize("offset", (1, 2, 4, 12))
def test_parameters_off_their_alignment_are_refused(offset):
    L = H._library()
    t = H.AdamwTensor()
    t.param = t.grad = t.m = t.v = 4096
    t.n, t.param_dtype, t.grad_dtype = 5000, S.GE_DTYPE_F32, S.GE_DTYPE_F32
    size = ctypes.c_int64()
    assert L.ge_adamw_table_bytes(ctypes.byref(t), 1, 32, ctypes.byref(size)) == S.GE_OK
    a = H.AdamwArgs(4096, size.value, 1, 32)
    a.device_params = 4096 + offset
    assert L.ge_adamw_step(None, ctypes.byref(a)) == S.GE_ERR_INVALID_ARG
    assert "device_params" in S.last_error()
