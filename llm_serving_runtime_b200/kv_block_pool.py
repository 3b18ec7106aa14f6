"""The KV-cache append of a block pool, on the sm_100a append kernel.

``write_tokens_batch_into(pool, layer_idx, block_tables, start_positions,
key_states, value_states)`` has the contract of the reference's
``GpuKVBlockPool.write_tokens_batch`` (runtime/phase2/paged_kv_kernel.py:176-227):
row b's token t lands in block ``block_tables[b, p // bs]`` at offset ``p % bs``,
with ``p = start_positions[b] + t``, in layer ``layer_idx`` of the pool.  One
``pa_kv_append`` launch moves every row instead of a Python loop of indexed
assignments per token.

The pool is any object with the reference pool's public surface: ``device``,
``block_size_tokens`` and the per-layer views ``k_layer_view(l)`` /
``v_layer_view(l)`` ([num_blocks, kv_heads, block_size, head_dim], strided
views of the pool are fine).  ``integration.install()`` binds this function as
the reference pool's ``write_tokens_batch``; a pool that records the blocks it
hands out and grows on first touch (the reference's ``_touch_blocks``,
paged_kv_kernel.py:117-122, :229-231) has that hook called before the views are
taken, so a grown pool is written in place.

``Fp8KVBlockPool`` is such a pool whose blocks are held in 8 bits (e4m3, one
scale for each block, layer and KV head), at half the bytes of a 16-bit pool.  The
reference has no counterpart.
"""

from __future__ import annotations

import torch

from .device_pages import copy_pages
from .paged_attention import CACHE_8BIT, kv_append

__all__ = ["write_tokens_batch_into", "Fp8KVBlockPool"]


def _capturing(device: torch.device) -> bool:
    return bool(device.type == "cuda" and torch.cuda.is_available() and torch.cuda.is_current_stream_capturing())


def write_tokens_batch_into(
    pool,
    layer_idx: int,
    block_tables: torch.Tensor,
    start_positions: torch.Tensor,
    key_states: torch.Tensor,
    value_states: torch.Tensor,
) -> None:
    """Batched KV write: states [B, kv_heads, kv_len, dim] at positions
    start_positions[b] + t through block_tables [B, max_blocks].

    Outside graph capture the reference's host checks stay (paged_kv_kernel.py:
    199-227): tables and positions move to the pool's device, a table too short
    for the positions raises IndexError, and the pool's block bookkeeping (when
    it has one) sees the touched blocks.  Under capture only the kernel runs,
    as in the reference's capture branch.
    """
    if key_states.shape != value_states.shape:
        raise ValueError("key_states and value_states must match shape")
    batch_size = int(key_states.shape[0])
    kv_len = int(key_states.shape[-2])
    if block_tables.shape[0] != batch_size or start_positions.shape[0] != batch_size:
        raise ValueError("batch dimension mismatch in write_tokens_batch")
    device = pool.device
    if device.type != "cuda":
        raise RuntimeError("the B200 paged KV append needs a CUDA pool (no CPU fallback)")
    if not _capturing(device):
        block_tables = block_tables.to(device=device, dtype=torch.int32)
        start_positions = start_positions.to(device=device, dtype=torch.int64)
        # the last position each row writes decides the underrun, as in the
        # reference's per-token check; one host synchronisation, as there
        if kv_len == 0:
            return
        bs = pool.block_size_tokens
        first = torch.div(start_positions, bs, rounding_mode="floor")
        logical_last = torch.div(start_positions + (kv_len - 1), bs, rounding_mode="floor")
        top, span = torch.stack([logical_last.max(), (logical_last - first).max()]).tolist()
        if top >= block_tables.shape[1]:
            raise IndexError("block table underrun during batched write")
        touch = getattr(pool, "_touch_blocks", None)
        if touch is not None:
            logical = (first[:, None] + torch.arange(span + 1, device=device)[None, :]).clamp_max(logical_last[:, None])
            touch(torch.gather(block_tables.to(torch.int64), 1, logical).reshape(-1))
    key_cache, scales = pool.k_layer_view(layer_idx), {}
    if key_cache.dtype == CACHE_8BIT:
        scales = {"key_scales": pool.k_layer_scales(layer_idx), "value_scales": pool.v_layer_scales(layer_idx)}
    kv_append(
        key_states,
        value_states,
        key_cache,
        pool.v_layer_view(layer_idx),
        None,
        block_tables=block_tables,
        positions=start_positions,
        **scales,
    )


class Fp8KVBlockPool:
    """A KV pool held in 8 bits: codes [num_blocks, layers, kv_heads, block_size, head_dim]
    and scales [num_blocks, layers, kv_heads].

        pool = Fp8KVBlockPool(num_blocks, layers, kv_heads, 16, 128, device)
        out = paged_attention_decode(q, pool.k_layer_view(l), pool.v_layer_view(l), tables, lens, scale,
                                     key=k, value=v, key_scales=pool.k_layer_scales(l),
                                     value_scales=pool.v_layer_scales(l))

    ``caches`` are the four tensors whose pages move together (``copy_pages``,
    ``DevicePages``); ``copy_blocks`` is the copy-on-write callback of
    ``BlockRefAllocator.make_writable``.
    """

    def __init__(self, num_blocks: int, num_layers: int, num_kv_heads: int, block_size: int, head_dim: int,
                 device: torch.device | str = "cuda") -> None:
        if min(num_blocks, num_layers, num_kv_heads) <= 0:
            raise ValueError("num_blocks, num_layers and num_kv_heads must be positive")
        if head_dim <= 0 or head_dim % 16 != 0:
            raise ValueError(f"an 8-bit cache needs a head_dim that is a multiple of 16, got {head_dim}")
        if block_size not in (8, 16, 32, 64, 128, 256):
            raise ValueError(f"an 8-bit cache needs a power-of-two block_size in [8, 256], got {block_size}")
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None and torch.cuda.is_available():
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.dtype = CACHE_8BIT
        self.block_size_tokens = block_size
        shape = (num_blocks, num_layers, num_kv_heads, block_size, head_dim)
        self.k = torch.zeros(shape, dtype=CACHE_8BIT, device=self.device)
        self.v = torch.zeros(shape, dtype=CACHE_8BIT, device=self.device)
        self.k_scales = torch.zeros(shape[:3], dtype=torch.float32, device=self.device)
        self.v_scales = torch.zeros(shape[:3], dtype=torch.float32, device=self.device)

    @property
    def caches(self) -> list[torch.Tensor]:
        return [self.k, self.v, self.k_scales, self.v_scales]

    def k_layer_view(self, layer: int) -> torch.Tensor:
        return self.k[:, layer]

    def v_layer_view(self, layer: int) -> torch.Tensor:
        return self.v[:, layer]

    def k_layer_scales(self, layer: int) -> torch.Tensor:
        return self.k_scales[:, layer]

    def v_layer_scales(self, layer: int) -> torch.Tensor:
        return self.v_scales[:, layer]

    def write_tokens_batch(self, layer_idx, block_tables, start_positions, key_states, value_states) -> None:
        write_tokens_batch_into(self, layer_idx, block_tables, start_positions, key_states, value_states)

    def copy_blocks(self, src_ids, dst_ids) -> None:
        """Whole blocks, every layer, codes and scales."""
        if len(src_ids) != len(dst_ids):
            raise ValueError("copy_blocks needs as many destinations as sources")
        if len(src_ids) == 0:
            return
        src, dst = (torch.as_tensor(list(x), dtype=torch.int32).to(self.device) for x in (src_ids, dst_ids))
        copy_pages(self.caches, src, dst)
