"""Block caches, accumulated weights and eviction: what is refused before any device work."""

import ctypes

import pytest
import torch

import gguf_train_amd as g
from gguf_train_amd import _C, _bridge

I8, E4M3 = _C.GT_I8, _C.GT_F8E4M3


@pytest.mark.parametrize("args,why", [
    ((0, 1, 8, 64, I8, 32, 0), "must be positive"), ((1, 0, 8, 64, I8, 32, 0), "must be positive"),
    ((1, 1, 0, 64, I8, 32, 0), "must be positive"), ((1, 1, 8, 0, I8, 32, 0), "must be positive"),
    ((-1, 1, 8, 64, I8, 32, 0), "must be positive"),
    ((1, 1, 8, 64, _C.GT_F16, 32, 0), "dtype must be int8 or float8_e4m3, got float16"),
    ((1, 1, 8, 64, _C.GT_Q8_0, 32, 0), "dtype must be int8 or float8_e4m3, got q8_0"),
    ((1, 1, 8, 64, I8, 16, 0), "block_tokens must be 32, 64 or 128, got 16"),
    ((1, 1, 8, 64, E4M3, 0, 0), "block_tokens must be"), ((1, 1, 8, 64, E4M3, 256, 0), "block_tokens must be"),
    ((1, 1, 8, 257, I8, 32, 0), "head_dim must be at most 256"),
    ((1, 1, 1 << 30, 64, I8, 32, 0), "capacity must be below"),
    ((256, 256, 8, 64, I8, 32, 0), "batch \\* n_head_kv at most 65535"),
    ((1 << 40, 1 << 40, 8, 64, I8, 32, 0), "batch \\* n_head_kv at most 65535"),
])
def test_create(args, why):
    assert not _C.lib.gt_kv_cache_create_blocks(*args)
    with pytest.raises(RuntimeError, match=why):
        _C.check_ptr(None, "kv_cache")


def test_null_caches():
    q = _bridge.borrow(torch.ones(1, 1, 1, 64))
    out = ctypes.c_void_p(), ctypes.c_void_p()
    sec = (ctypes.c_int * 1)(32)
    lib = _C.lib
    assert not lib.gt_kv_cache_attention_accumulate(None, q.ptr, 0.0, 1, 1.0) and "NULL cache" in _C.last_error()
    assert not lib.gt_kv_cache_weights(None) and "NULL cache" in _C.last_error()
    assert lib.gt_kv_cache_evict(None, 1, 0, None, None) != 0 and "NULL cache" in _C.last_error()
    assert lib.gt_kv_cache_read(None, _C.GT_F32, ctypes.byref(out[0]), ctypes.byref(out[1])) != 0
    assert lib.gt_kv_cache_position(None, 0) == -1
    assert lib.gt_kv_cache_append_rope_axes(None, q.ptr, q.ptr, -1, q.ptr, 1, sec, 0, 64, 2, 10000.0, 1.0) != 0
    lib.gt_kv_cache_free(None)


@pytest.mark.parametrize("keep", [-0.5, 1.5, float("nan"), float("inf")])
def test_accumulation_factor(keep):
    q = _bridge.borrow(torch.ones(1, 1, 1, 64))
    assert not _C.lib.gt_kv_cache_attention_accumulate(None, q.ptr, 0.0, 1, keep)
    assert "must be in [0, 1]" in _C.last_error()


def test_python_arguments():
    with pytest.raises(ValueError, match="unsupported cache dtype"):
        g.KVCache(1, 1, 8, 64, torch.int16)
    with pytest.raises(ValueError, match="block_tokens is for int8"):
        g.KVCache(1, 1, 8, 64, torch.float16, block_tokens=32)
    with pytest.raises(ValueError, match="cuda device"):
        g.KVCache(1, 1, 8, 64, torch.int8, "cpu")
