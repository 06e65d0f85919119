"""What sampling and the calls for drafted tokens refuse without a device: those checks run before anything else."""
import ctypes as C

import pytest

from spissa_amd import _ffi

INF, NAN = float("inf"), float("nan")


def sampling(**kw):
    c = _ffi.SamplingConfigC(2, 100, 1.0, 0, 1.0, 0.0, None, None, None, None)
    for name, value in kw.items():
        setattr(c, name, value)
    return _ffi.load().spissa_sample_device(None, None, None, C.byref(c), None, None)


@pytest.mark.parametrize("kw", [{"temperature": -1.0}, {"temperature": INF}, {"temperature": NAN}, {"top_p": -0.1}, {"top_p": 1.5},
                                {"top_p": NAN}, {"min_p": -0.1}, {"min_p": 1.01}, {"min_p": NAN}, {"vocab": 0}])
def test_sampling_settings(kw):
    assert sampling(**kw) == _ffi.ERR_INVALID_TENSOR_DATA


@pytest.mark.parametrize("kw", [{"vocab": (1 << 22) + 1}, {"rows": 1 << 31}])
def test_sampling_sizes(kw):
    assert sampling(**kw) == _ffi.ERR_SHAPE


def test_sampling_null_handles():
    assert sampling() == _ffi.ERR_ARGUMENT
    assert _ffi.load().spissa_sample_device(None, None, None, None, None, None) == _ffi.ERR_ARGUMENT


def tree(nodes, gemma=False, **kw):
    lib = _ffi.load()
    cfg = _ffi.AttnConfigC(sum(nodes), 4, 2, 64, 1, 0)
    for name, value in kw.items():
        setattr(cfg, name, value)
    counts = (_ffi.c_size * max(1, len(nodes)))(*nodes)
    args = (None, None, None, None, None, None, counts, len(nodes), None, C.byref(cfg))
    return lib.spissa_gemma_tree_step_device(*args, None, None, 1e-6, 1.0, None) if gemma else lib.spissa_tree_step_device(*args, None)


@pytest.mark.parametrize("gemma", [False, True])
@pytest.mark.parametrize("nodes,kw", [([257], {}), ([3, 4], {"query_len": 6}), ([3], {"query_len": 0}), ([2], {"causal": 0}),
                                      ([2], {"head_dim": 96}), ([2], {"head_dim": 0}), ([2], {"head_dim": 1 << 40})])
def test_tree_shapes(nodes, kw, gemma):
    assert tree(nodes, gemma, **kw) == _ffi.ERR_SHAPE


def test_null_handles():
    lib = _ffi.load()
    counts = (_ffi.c_size * 1)(3)
    assert tree([3]) == tree([3], True) == _ffi.ERR_ARGUMENT
    assert lib.spissa_tree_step_device(None, None, None, None, None, None, None, 0, None, None, None) == _ffi.ERR_ARGUMENT
    assert lib.spissa_tree_accept_device(None, None, None, None, counts, 1, None, None, None) == _ffi.ERR_ARGUMENT
    assert lib.spissa_tree_accept_device(None, None, None, None, None, 1, None, None, None) == _ffi.ERR_ARGUMENT
    assert lib.spissa_kv_cache_keep_device(None, None, 1, counts, 1, None, None) == _ffi.ERR_ARGUMENT
    assert lib.spissa_kv_cache_keep_device(None, None, 1, None, 1, None, None) == _ffi.ERR_ARGUMENT
    counts[0] = 257
    assert lib.spissa_tree_accept_device(None, None, None, None, counts, 1, None, None, None) == _ffi.ERR_SHAPE
    assert lib.spissa_kv_cache_keep_device(None, None, 1, counts, 1, None, None) == _ffi.ERR_SHAPE
    counts[0] = 3
    assert lib.spissa_kv_cache_keep_device(None, None, 1 << 63, (_ffi.c_size * 2)(3, 3), 2, None, None) == _ffi.ERR_SHAPE


def test_the_rust_settings_follow_the_header():
    from tests.test_integration_recipe import LIB_RS, c_struct_fields, rust_struct_fields

    assert rust_struct_fields("spissa_sampling_config") == c_struct_fields("spissa_sampling_config")
    assert "#[repr(C)]" in LIB_RS.split("pub struct spissa_sampling_config")[0][-80:]


@pytest.mark.parametrize("shape,rows", [((4, 8), 2), ((4, 8), 8), ((2, 2, 8), 2), ((4, 8), 0), ((1, 8), 2), ((3, 0), 1), ((9,), 2)])
def test_sampling_takes_one_number_a_row(shape, rows):
    """Rows of logits are not joined or parted, also where their number divides."""
    import torch

    from spissa_amd.device import SamplingConfig, Session

    with pytest.raises(TypeError, match="rows"):
        Session.sample(None, torch.zeros(shape), torch.zeros(rows), SamplingConfig(), torch.zeros(rows, dtype=torch.int32))


@pytest.mark.parametrize("top_k,kept", [(-3, 0), (0, 0), (7, 7), (100, 100), (1 << 40, 100), ((1 << 64) + 5, 100)])
def test_a_top_k_of_any_size(top_k, kept):
    from spissa_amd.device import SamplingConfig

    assert SamplingConfig(top_k=top_k)._c(2, 100).top_k == kept
