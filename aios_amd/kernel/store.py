"""Paged KV append entry point (HIP kernel (a) behind the C ABI).

Same signature, validation and error messages as the reference's Triton
``store_cache`` (python/aios/kernel/store.py:32-61): scatter a flat batch of
K/V rows into a ``(num_slots, num_heads, head_dim)`` cache view, with k and v
allowed independent token strides.
"""
from __future__ import annotations

import torch

from aios_amd import _lib


def store_cache(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    indices: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
) -> None:
    """Scatter ``k[t]``/``v[t]`` into cache row ``indices[t]``."""
    if k_cache.ndim != 3 or v_cache.ndim != 3:
        raise ValueError("KV cache must have shape (num_slots, num_heads, head_dim)")
    if k.shape[1:] != k_cache.shape[1:] or v.shape[1:] != v_cache.shape[1:]:
        raise ValueError("K/V input shape does not match the cache layout")
    if indices.numel() != k.shape[0] or k.shape != v.shape:
        raise ValueError("KV write indices and K/V tensors must have matching token counts")
    assert all(t.is_cuda for t in (k_cache, v_cache, indices, k, v))
    if k_cache.dtype != k.dtype or v_cache.dtype != v.dtype or k.dtype != v.dtype:
        raise ValueError("K/V dtype does not match the cache dtype")
    if k_cache.stride() != v_cache.stride():
        raise ValueError("K and V caches must share one layout")
    width = k_cache.shape[1] * k_cache.shape[2]
    # Rows must be contiguous inside a token; the token stride is free.
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache), ("k", k), ("v", v)):
        if t.stride(2) != 1 or t.stride(1) != t.shape[2]:
            raise ValueError(f"{name} must have contiguous (heads, head_dim) rows")
    if indices.dtype != torch.int32:
        indices = indices.to(torch.int32)
    indices = indices.contiguous()
    stream = _lib.raw_stream(k_cache)
    _lib.check(
        _lib.lib().aios_kv_append(
            k_cache.data_ptr(),
            v_cache.data_ptr(),
            k_cache.shape[0],
            k_cache.stride(0),
            indices.data_ptr(),
            k.data_ptr(),
            k.stride(0),
            v.data_ptr(),
            v.stride(0),
            k.shape[0],
            width,
            k.element_size(),
            stream,
        ),
        "aios_kv_append",
    )


def store_cache8(
    k8: torch.Tensor,
    v8: torch.Tensor,
    scales: torch.Tensor,
    indices: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
) -> None:
    """Quantise ``k[t]``/``v[t]`` (bfloat16) into page ``indices[t]`` of an
    8-bit cache: k8, v8 float8_e4m3fn (num_slots, num_heads, head_dim) codes
    and scales bfloat16 (num_heads, num_slots, 2), K's scale then V's, the
    power of two that brings the row's largest magnitude to at most 448.
    Indices outside the pool are not written; a page named twice holds some mix
    of its rows."""
    shape = k8.shape
    if len(shape) != 3 or v8.shape != shape:
        raise ValueError("KV cache must have shape (num_slots, num_heads, head_dim)")
    slots, heads, dim = shape
    new = k.shape
    if new[1:] != shape[1:]:
        raise ValueError("K/V input shape does not match the cache layout")
    tokens = new[0]
    if indices.numel() != tokens or v.shape != new:
        raise ValueError("KV write indices and K/V tensors must have matching token counts")
    if k8.dtype is not torch.float8_e4m3fn or v8.dtype is not torch.float8_e4m3fn:
        raise ValueError("the 8-bit KV cache holds float8_e4m3fn codes")
    bf16 = torch.bfloat16
    if k.dtype is not bf16 or v.dtype is not bf16:
        raise ValueError("the 8-bit KV cache takes bfloat16 K/V rows")
    if scales.dtype is not bf16 or scales.shape != (heads, slots, 2):
        raise ValueError("scales must be bfloat16 (num_heads, num_slots, 2)")
    if not (k8.is_contiguous() and v8.is_contiguous() and scales.is_contiguous()):
        raise ValueError("8-bit KV caches and their scales must be contiguous")
    k_stride, v_stride = k.stride(), v.stride()
    for name, stride in (("k", k_stride), ("v", v_stride)):
        if stride[2] != 1 or (stride[1] != dim and heads > 1):
            raise ValueError(f"{name} must have contiguous (heads, head_dim) rows")
    dev = k8.get_device()
    if not (dev == v8.get_device() == scales.get_device() == indices.get_device()
            == k.get_device() == v.get_device()):
        raise ValueError("the KV cache, its scales, the indices and K/V must be on one GPU")
    if indices.dtype != torch.int32:
        if indices.dtype.is_floating_point or indices.dtype == torch.bool:
            raise ValueError("KV write indices must be integers")
        indices = indices.clamp(-1, slots).to(torch.int32)  # (outside the pool stays outside)
    if not indices.is_contiguous():
        indices = indices.contiguous()
    _lib.check(
        _lib.lib().aios_kv8_append(
            k8.data_ptr(), v8.data_ptr(), scales.data_ptr(), slots, heads, dim,
            indices.data_ptr(), k.data_ptr(), k_stride[0], v.data_ptr(), v_stride[0], tokens,
            _lib.current_stream(k8)),
        "aios_kv8_append",
    )
