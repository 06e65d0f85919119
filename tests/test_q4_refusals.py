"""What the 4-bit cache refuses without a device: the checks run before anything else."""
import ctypes as C

import pytest

import spissa_amd as sa
from spissa_amd import _ffi


@pytest.mark.parametrize("shape", [(0, 64, 8), (2, 0, 8), (2, 64, 0), (2, 32, 8), (2, 96, 8), (2, 80, 8), (2, 512, 8),
                                   (2, 64, (1 << 24) + 1), (65536, 64, 8), (1 << 40, 64, 1 << 20)])
def test_cache_shapes(shape):
    with pytest.raises(sa.ShapeError):
        sa.Q4KvCache(*shape)


def test_null_handles():
    lib = _ffi.load()
    assert lib.spissa_kv_cache_q4_new(2, 64, 8, None) == _ffi.ERR_ARGUMENT
    assert lib.spissa_kv_cache_q4_new_in(None, 2, 64, 8, C.byref(C.c_void_p())) == _ffi.ERR_ARGUMENT
    assert lib.spissa_kv_cache_is_q4(None) == 0
    assert lib.spissa_kv_cache_rows_device(None, 0, 0, None, None) == _ffi.ERR_ARGUMENT
    cfg = _ffi.AttnConfigC(1, 2, 2, 64, 1, 0)
    assert lib.spissa_attention_cached_batch_device(None, None, None, 0, C.byref(cfg), None) == _ffi.ERR_ARGUMENT
