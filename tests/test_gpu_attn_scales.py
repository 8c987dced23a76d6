"""Scales and caps whose ratio no fp32 number holds are refused (no GPU): every capped score would come out as 0."""
import ctypes as C

import pytest

from rocwmma_b200 import _lib
from test_gpu_attn import args
from test_gpu_attn_tree import call, targs


@pytest.mark.parametrize("how", [dict(scale=1e-10, cap=1e30), dict(scale=-1e-20, cap=1e20), dict(scale=1e-38, cap=1.0)])
def test_refused(how):
    L, a = _lib.lib(), args(**how)
    assert L.b200wmma_attn_fwd(C.byref(a), 16, 16, 16, 16, 16, 16, 1 << 30, None) == 2
    assert L.b200wmma_attn_bwd(C.byref(a), *[16] * 9, 16, 1 << 30, None) == 2
    assert call(targs(**how)) == 2
    assert b"attn_tree" in L.b200wmma_last_error_string()
