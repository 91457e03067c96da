"""Token-granular paged KV pool in 8 bits.

The layout of :class:`MHAKVCache` with float8_e4m3fn codes, ``[2, num_layers,
num_pages, page_size=1, num_kv_heads, head_dim]``, and one power-of-two scale
for each page's K row and V row of a kv-head: ``[num_layers, num_kv_heads,
num_pages, 2]`` bfloat16, K's first.  The value of the cache is code * scale,
exact in bfloat16.  Half the bytes of the bfloat16 pool plus 4 per (page,
kv-head): the long-context workload, 36 layers of 8 kv-heads x 128 over 65,536
pages, needs 4.6 GiB.

``store_kv`` quantises bfloat16 rows (aios_amd.kernel.store_cache8); the
attention backend reads the pool in both phases.
"""
from __future__ import annotations

import torch

from .base import BaseKVCache


class MHAKVCache8(BaseKVCache):
    def __init__(
        self,
        num_kv_heads: int,
        num_layers: int,
        head_dim: int,
        num_pages: int,
        page_size: int,
        dtype: torch.dtype,
        device: torch.device,
    ) -> None:
        device = torch.device(device)
        assert device.type == "cuda", "AIOS only supports GPU execution"
        assert page_size == 1, "the MI355X backend only supports page_size=1"
        if dtype != torch.float8_e4m3fn:
            raise ValueError("the 8-bit KV cache holds float8_e4m3fn codes")
        if head_dim not in (64, 96, 128):
            raise ValueError(f"head_dim {head_dim} is not supported by the 8-bit KV cache")
        self._kv_buffer = torch.empty(
            (2, num_layers, num_pages, page_size, num_kv_heads, head_dim),
            device=device,
            dtype=dtype,
        )
        self._scales = torch.empty((num_layers, num_kv_heads, num_pages, 2), device=device,
                                   dtype=torch.bfloat16)
        self._num_layers = num_layers
        self._k_buffer = self._kv_buffer[0]
        self._v_buffer = self._kv_buffer[1]
        self._device = device
        self._storage_shape = (num_pages * page_size, num_kv_heads, head_dim)

    def k_cache(self, index: int) -> torch.Tensor:
        return self._k_buffer[index]

    def v_cache(self, index: int) -> torch.Tensor:
        return self._v_buffer[index]

    def scales(self, index: int) -> torch.Tensor:
        """[num_kv_heads, num_pages, 2] of one layer."""
        return self._scales[index]

    def layer(self, index: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """(k8, v8 [num_pages, Hkv, D], scales) of one layer, as the functions of
        aios_amd.paged named ...8 and store_cache8 take them."""
        return (self._k_buffer[index].view(self._storage_shape),
                self._v_buffer[index].view(self._storage_shape), self._scales[index])

    def store_kv(
        self, k: torch.Tensor, v: torch.Tensor, out_loc: torch.Tensor, layer_id: int
    ) -> None:
        from aios_amd.kernel import store_cache8

        store_cache8(*self.layer(layer_id), out_loc, k, v)

    @property
    def row_shape(self) -> tuple[int, int]:
        """(num_kv_heads, head_dim) of a page's K or V row."""
        return self._storage_shape[1:]

    @property
    def device(self) -> torch.device:
        return self._device

    @property
    def dtype(self) -> torch.dtype:
        return self._kv_buffer.dtype

    @property
    def num_layers(self) -> int:
        return self._num_layers

    @property
    def num_pages(self) -> int:
        return self._storage_shape[0]
