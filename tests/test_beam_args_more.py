"""CPU tests: calls of the beam-search operators that are refused before they touch a device."""
import ctypes

import synapse_b200 as sb

L = sb.lib
ONE = ctypes.c_void_p(8)


def test_get_error_needs_its_pointers():
    v = ctypes.c_int32()
    assert L.syn_cuda_decode_plan_get_error(None, ctypes.byref(v)) == 1
    assert L.syn_cuda_decode_plan_get_error(ONE, None) == 1
