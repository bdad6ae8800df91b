"""K and V pools of all layers in 4 bits: 3.76 times the tokens of ``MHAKVCache`` in the same memory.

A slot holds, for every kv head, the 4-bit floats of K and behind them V's (a line of 128 bytes at head_dim 128), and one byte to
each block of 32 dims for its power of two: 4.25 bits a value.  The writers are ``store_kv`` and
``qk_norm_rope_store_mxfp4``; attention reads the pool through ``paged_decode_attention_mxfp4`` and
``paged_prefill_attention_mxfp4``, which ``AttnBackend`` calls for a pool of this class.  Slots are handed out, shared by prefix caches and freed as
those of a 16-bit pool.  The reference's pool is 16 bits only (mini_sglang_mlx/kvcache/mha_pool.py:10-56).
"""
from __future__ import annotations

from typing import Tuple

import torch

from mini_sglang_amd_kernel import load_kv_cache_mxfp4, store_kv_cache_mxfp4

from .base import BaseKVCache

BLOCK = 32  # dims with a power of two in common


class MXFP4KVCache(BaseKVCache):
    """``dtype`` is the type of the rows that are stored and of the queries: bfloat16 or float16 (decode only)."""

    def __init__(self, num_kv_heads: int, num_layers: int, head_dim: int, num_pages: int,
                 dtype: torch.dtype, device="cuda"):
        if min(num_kv_heads, num_layers, head_dim, num_pages) <= 0:
            raise ValueError("MXFP4KVCache: every dimension must be positive")
        if head_dim not in (128, 256):
            raise ValueError("MXFP4KVCache: head_dim must be 128 or 256")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("MXFP4KVCache: dtype must be float16 or bfloat16")
        slab = (num_layers, num_pages, num_kv_heads, 2)
        self._codes = torch.zeros((*slab, head_dim // 2), dtype=torch.uint8, device=device)
        self._scales = torch.zeros((*slab, head_dim // BLOCK), dtype=torch.uint8, device=device)
        self._code_layers, self._scale_layers = self._codes.unbind(0), self._scales.unbind(0)
        self._dtype = dtype

    def codes(self, index: int) -> torch.Tensor:
        """A layer's ``(num_pages, num_kv_heads, 2, head_dim / 2)`` codes, K first."""
        return self._code_layers[index]

    def scales(self, index: int) -> torch.Tensor:
        """A layer's ``(num_pages, num_kv_heads, 2, head_dim / 32)`` block bytes."""
        return self._scale_layers[index]

    def require_rows(self, op: str, k: torch.Tensor, v: torch.Tensor) -> None:
        """Rows of another type may hold what this pool's queries cannot: bf16 reaches beyond half."""
        if k.dtype is not self._dtype or v.dtype is not self._dtype:
            raise ValueError(f"{op}: k is {k.dtype} and v {v.dtype}, the cache's dtype is {self._dtype}")

    # ---- the surface of a pool ---------------------------------------------------------------
    def k_cache(self, index: int) -> torch.Tensor:
        """K's codes; their block bytes are ``scales(index)[:, :, 0]``."""
        return self._code_layers[index][:, :, 0]

    def v_cache(self, index: int) -> torch.Tensor:
        return self._code_layers[index][:, :, 1]

    def store_kv(self, k: torch.Tensor, v: torch.Tensor, out_loc: torch.Tensor,
                 layer_id: int) -> None:
        """The rows of ``k`` and ``v`` as codes at slots ``out_loc``: one launch."""
        assert out_loc.dtype == torch.int32, "out_loc must be int32"
        rows = out_loc.shape[0]
        if k.shape[0] != rows or v.shape[0] != rows:
            raise ValueError(f"store_kv: {rows} slot ids for k of shape {tuple(k.shape)} and v of "
                             f"shape {tuple(v.shape)}")
        self.require_rows("store_kv", k, v)
        store_kv_cache_mxfp4(self._code_layers[layer_id], self._scale_layers[layer_id], out_loc, k, v)

    def load_kv(self, indices: torch.Tensor, layer_id: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """``(k, v)`` that slots ``indices`` hold, in this pool's dtype."""
        return load_kv_cache_mxfp4(self._code_layers[layer_id], self._scale_layers[layer_id], indices, dtype=self._dtype)

    @property
    def dtype(self) -> torch.dtype:
        return self._dtype

    @property
    def num_layers(self) -> int:
        return self._codes.shape[0]

    @property
    def pool_shape(self) -> Tuple[int, int, int]:
        """``(num_pages, num_kv_heads, head_dim)`` of one layer's pool."""
        pages, heads, _, half = self._codes.shape[1:]
        return pages, heads, 2 * half

    @property
    def nbytes(self) -> int:
        return self._codes.numel() + self._scales.numel()
