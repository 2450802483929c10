"""What layer norm's backward pass refuses beside test_linear8_cpu.py, before anything is launched."""
import ctypes as C

import pytest

from speedplusbaseline_amd import _args8 as A8, _lib as L


@pytest.mark.parametrize("lib", [L.lib, L.lib_f16], ids=["bf16", "f16"])
@pytest.mark.parametrize("dtype", [0, 1])
def test_one_buffer_for_both_parameter_gradients(lib, dtype):
    """two sums into one buffer have no order"""
    p = 1 << 20                 # an aligned address that is never read
    a = A8.LayerNormArgs(p, p, None, None, p, p, p, p, p, p, 1 << 20, 4, 32, 32, 32, 32, 1e-5, 1)
    a.dgamma = a.dbeta = p
    assert lib().spb_layernorm_bwd(dtype, C.byref(a), None) == -1
