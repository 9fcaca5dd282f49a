"""A key/value cache for decoding, on the device.

The reference decodes through llama.cpp's context (LlamaContext.forward_logits / clear_kv,
gguf_train/llama/__init__.py:174-190, csrc/llama_bridge.cpp:245-296): tokens are fed at
positions that continue what the context holds, the context has a fixed size (n_ctx) and
clear_kv() empties it.  KVCache keeps that behaviour for attention: `batch` sequences of
n_head_kv heads, room for `capacity` tokens each, stored in HBM as float16 / bfloat16 /
float32 or GGUF Q8_0 (each appended row quantized exactly as `quantize` does).  Attention
over the cache runs the library's kernels with each sequence's own length:
split-K decode for one query row (straight from the Q8_0 blocks for a Q8_0 cache), the MFMA
prefill kernel for several.

Beyond that, for long contexts: a cache of 8-bit codes (dtype torch.int8 or torch.float8_e4m3fn) with one
power-of-two scale for each block of `block_tokens` tokens and kv head, whose last, unfinished block stays
float32 and whose attention reads the codes; keys rotated by positions on several axes on the way in
(`append(rope={"positions": ...})`); the attention weight that each token receives, counted along with the
attention (`attention(accumulate=...)`, `weights()`); and eviction of the tokens of the smallest weights
(`evict`), after which positions run ahead of the lengths.
"""

from __future__ import annotations

import ctypes

import torch

from . import _C
from ._bridge import adopt, adopt_quantized, bind_stream, borrow
from ._ops import section_list

_CACHE_DTYPES = {torch.float32: _C.GT_F32, torch.float16: _C.GT_F16, torch.bfloat16: _C.GT_BF16, "q8_0": _C.GT_Q8_0}
_BLOCK_DTYPES = {torch.int8: _C.GT_I8, torch.float8_e4m3fn: _C.GT_F8E4M3}
_READ_DTYPES = {torch.float32: _C.GT_F32, torch.float16: _C.GT_F16, torch.bfloat16: _C.GT_BF16}


class KVCache:
    def __init__(self, batch: int, n_head_kv: int, capacity: int, head_dim: int, dtype=torch.float16,
                 device: str | torch.device = "cuda", block_tokens: int | None = None) -> None:
        """block_tokens: tokens that share a scale in an int8 or float8_e4m3fn cache, 32 (the default), 64 or 128."""
        if dtype not in _CACHE_DTYPES and dtype not in _BLOCK_DTYPES:
            raise ValueError(f"unsupported cache dtype {dtype!r} (float32, float16, bfloat16, 'q8_0', int8 or float8_e4m3fn)")
        if block_tokens is not None and dtype not in _BLOCK_DTYPES:
            raise ValueError(f"block_tokens is for int8 and float8_e4m3fn caches, not {dtype!r}")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("the KV cache lives in device memory: pass a cuda device")
        self.dtype = dtype
        self.batch, self.n_head_kv, self.head_dim = int(batch), int(n_head_kv), int(head_dim)
        bind_stream(self.device)
        index = self.device.index if self.device.index is not None else torch.cuda.current_device()
        if dtype in _BLOCK_DTYPES:
            self.block_tokens = 32 if block_tokens is None else int(block_tokens)
            self._ptr = _C.check_ptr(_C.lib.gt_kv_cache_create_blocks(
                self.batch, self.n_head_kv, int(capacity), self.head_dim, _BLOCK_DTYPES[dtype], self.block_tokens, int(index)),
                "kv_cache")
            return
        self._ptr = _C.check_ptr(_C.lib.gt_kv_cache_create(self.batch, self.n_head_kv, int(capacity), self.head_dim,
                                                           _CACHE_DTYPES[dtype], int(index)), "kv_cache")

    def __del__(self, _free=_C.lib.gt_kv_cache_free):
        ptr = getattr(self, "_ptr", None)
        if ptr:
            _free(ptr)
            self._ptr = None

    @property
    def capacity(self) -> int:
        return int(_C.lib.gt_kv_cache_capacity(self._ptr))

    def n_ctx(self) -> int:
        """The number of tokens a sequence can hold (LlamaContext.n_ctx)."""
        return self.capacity

    def length(self, seq: int = 0) -> int:
        n = int(_C.lib.gt_kv_cache_length(self._ptr, int(seq)))
        if n < 0:
            raise IndexError(_C.last_error())
        return n

    @property
    def lengths(self) -> list[int]:
        return [self.length(b) for b in range(self.batch)]

    def position(self, seq: int = 0) -> int:
        """The position of a sequence's next token: the tokens appended to it, evicted ones included."""
        n = int(_C.lib.gt_kv_cache_position(self._ptr, int(seq)))
        if n < 0:
            raise IndexError(_C.last_error())
        return n

    def clear(self, seq: int | None = None) -> None:
        """Empties one sequence, or all of them (LlamaContext.clear_kv)."""
        bind_stream(self.device)
        _C.check_rc(_C.lib.gt_kv_cache_clear(self._ptr, -1 if seq is None else int(seq)), "kv_cache")

    clear_kv = clear

    def append(self, k: torch.Tensor, v: torch.Tensor, pos_offset: int | None = None, rope: dict | None = None) -> None:
        """Appends k, v (batch, n_head_kv, T, head_dim) to every sequence: float tensors, or Q8_0
        `QuantizedTensor`s (e.g. read from a GGUF file), whose blocks a Q8_0 cache stores as they
        are.  With pos_offset the positions must continue what each sequence holds, as
        forward_logits(pos_offset=...).  `rope` (keys n_dims, mode, freq_base, freq_scale, as
        nn.functional.rope) rotates each key row at its cache position on the way in; the cache
        then holds what rope() of the keys followed by append() would store.  With the keys
        `positions` (axes, T) or (axes, batch, T) and `sections` (and optionally interleaved) the
        rows are rotated as nn.functional.rope_axes does, by default in mode 2, at those positions."""
        bind_stream(self.device)
        hk, hv = borrow(k), borrow(v)
        off = -1 if pos_offset is None else int(pos_offset)
        if rope is None:
            rc = _C.lib.gt_kv_cache_append(self._ptr, hk.ptr, hv.ptr, off)
        elif "positions" in rope or "sections" in rope:
            rc = self._append_axes(hk, hv, off, **rope)
        else:
            r = dict(rope)
            unknown = set(r) - {"n_dims", "mode", "freq_base", "freq_scale"}
            if unknown:
                raise TypeError(f"unknown rope arguments {sorted(unknown)}")
            rc = _C.lib.gt_kv_cache_append_rope(self._ptr, hk.ptr, hv.ptr, off, int(r.get("n_dims", self.head_dim)),
                                                int(r.get("mode", 0)), ctypes.c_float(r.get("freq_base", 10000.0)),
                                                ctypes.c_float(r.get("freq_scale", 1.0)))
        _C.check_rc(rc, "kv_cache")

    def _append_axes(self, hk, hv, off, *, positions, sections, interleaved=False, n_dims=None, mode=2, freq_base=10000.0,
                     freq_scale=1.0) -> int:
        hp = borrow(positions)
        n, sec = section_list(sections)
        return _C.lib.gt_kv_cache_append_rope_axes(self._ptr, hk.ptr, hv.ptr, off, hp.ptr, n, sec, 1 if interleaved else 0,
                                                   self.head_dim if n_dims is None else int(n_dims), int(mode), float(freq_base),
                                                   float(freq_scale))

    def attention(self, q: torch.Tensor, scale: float | None = None, is_causal: bool = True,
                  accumulate: float | None = None) -> torch.Tensor:
        """Attention of q (batch, H, L, head_dim) whose rows are the last L tokens of each
        sequence, over what each sequence holds; causal: a token sees itself and earlier ones.
        accumulate (0 to 1): also counts the weight that each token receives: weights() becomes
        accumulate times itself plus the sum of this call's softmax weights over the rows and the
        query heads of a kv head (1.0 adds to the count, 0.0 starts it anew)."""
        bind_stream(self.device)
        hq = borrow(q)
        if accumulate is not None:
            ptr = _C.lib.gt_kv_cache_attention_accumulate(self._ptr, hq.ptr, ctypes.c_float(0.0 if scale is None else scale),
                                                          1 if is_causal else 0, ctypes.c_float(accumulate))
            return adopt(ptr, "kv_cache")
        ptr = _C.lib.gt_kv_cache_attention(self._ptr, hq.ptr, ctypes.c_float(0.0 if scale is None else scale),
                                           1 if is_causal else 0)
        return adopt(ptr, "kv_cache")

    def weights(self) -> torch.Tensor:
        """The accumulated attention weights (batch, n_head_kv, capacity) float32, shared, not copied;
        zeros past a sequence's length."""
        bind_stream(self.device)
        return adopt(_C.lib.gt_kv_cache_weights(self._ptr), "kv_cache")

    def evict(self, keep: int, recent: int = 0, weights: torch.Tensor | None = None) -> torch.Tensor:
        """Cuts each sequence that holds more than `keep` tokens to `keep`: per kv head, its `recent`
        last tokens and the others of the largest weights (the earliest of equal ones), in order.
        `weights` (batch, n_head_kv, tokens or more), by default the accumulated ones.  Returns the
        kept tokens' indices (batch, n_head_kv, keep) int64, -1 past a shorter sequence's length.
        Positions (append's pos_offset, its one-axis rope) go on counting evicted tokens."""
        bind_stream(self.device)
        hw = borrow(weights) if weights is not None else None
        out = ctypes.c_void_p()
        _C.check_rc(_C.lib.gt_kv_cache_evict(self._ptr, int(keep), int(recent), hw.ptr if hw else None, ctypes.byref(out)),
                    "kv_cache")
        return adopt(out.value, "kv_cache")

    def read(self, dtype: torch.dtype = torch.float32):
        """The keys and values that the cache stands for, (batch, n_head_kv, longest length, head_dim)
        each, copied as float32, float16 or bfloat16; zeros past a sequence's length."""
        if dtype not in _READ_DTYPES:
            raise ValueError(f"unsupported dtype {dtype!r} (float32, float16 or bfloat16)")
        bind_stream(self.device)
        k, v = ctypes.c_void_p(), ctypes.c_void_p()
        _C.check_rc(_C.lib.gt_kv_cache_read(self._ptr, _READ_DTYPES[dtype], ctypes.byref(k), ctypes.byref(v)), "kv_cache")
        return adopt(k.value, "kv_cache"), adopt(v.value, "kv_cache")

    def keys(self):
        """The key storage (batch, n_head_kv, capacity, head_dim), shared, not copied."""
        return self._storage(_C.lib.gt_kv_cache_keys)

    def values(self):
        return self._storage(_C.lib.gt_kv_cache_values)

    def _storage(self, fn):
        ptr = _C.check_ptr(fn(self._ptr), "kv_cache")
        if self.dtype == "q8_0":
            return adopt_quantized(ptr, (self.batch, self.n_head_kv, self.capacity, self.head_dim), "kv_cache")
        return adopt(ptr, "kv_cache")
