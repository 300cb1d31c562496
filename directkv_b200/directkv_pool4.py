"""Token-indexed KV cache held in 4 bits.

``DirectKV4BitTokenToKVPool`` is ``DirectKVTokenToKVPool`` (same constructor, slots and ``KVCache`` methods) with 72 instead of
256 bytes per row and head: a cache for 3.5 times the tokens in the same memory, and as many times fewer bytes over the host
link or out of HBM in every decode step.  The format stands in include/directkv_b200.h at ``dkv_kv4_pool``.  The arrays lie in
page-locked host memory (``location="host"``, the default) or in HBM (``"device"``).

``DirectKVBackend`` recognises the class: its token-pool path stores with ``set_kv_buffer``, attends short queries with
``kernel.decode_kv4`` and brings the rows of long prompts back to bf16 (``load_rows``) for the tensor-core extend kernel.
"""

from __future__ import annotations

import logging
from typing import List, Optional, Tuple

import torch

from . import kernel
from .directkv_pool import DirectKVTokenToKVPool

logger = logging.getLogger(__name__)

_IN_4_BITS = "the pool is held in 4 bits: read rows with load_rows, attend them with kernel.decode_kv4(..., pool.layer_pool(layer_id), ...)"


class DirectKV4BitTokenToKVPool(DirectKVTokenToKVPool):
    def __init__(self, size: int, page_size: int, dtype: torch.dtype, head_num: int, head_dim: int, layer_num: int, device: str = "cpu",
                 enable_memory_saver: bool = False, v_head_dim: Optional[int] = None, start_layer: Optional[int] = None,
                 end_layer: Optional[int] = None, location: str = "host", k_scale: float = 1.0, v_scale: float = 1.0):
        if dtype != torch.bfloat16:
            raise ValueError(f"DirectKV4BitTokenToKVPool stores bfloat16 rows in 4 bits, got {dtype}")
        if head_dim != kernel.HEAD_DIM or v_head_dim not in (None, kernel.HEAD_DIM):
            raise ValueError(f"DirectKV4BitTokenToKVPool requires head_dim={kernel.HEAD_DIM}")
        if location not in ("host", "device"):
            raise ValueError(f"location must be 'host' or 'device', got {location!r}")
        self.location = location
        self._k_scale, self._v_scale = float(k_scale), float(v_scale)
        self._storage_device = "cpu" if location == "host" else (device if torch.device(device).type == "cuda" else "cuda")
        super().__init__(size, page_size, dtype, head_num, head_dim, layer_num, device, enable_memory_saver, v_head_dim, start_layer, end_layer)

    # ---- storage ------------------------------------------------------------
    def _allocate(self) -> None:
        # Tokens are addressed by slot (page size 1), as in the bf16 pool.
        self._layers: List[kernel.KV4Pool] = [
            kernel.KV4Pool.empty(self.n_slots, self.head_num, 1, self._storage_device, self._k_scale, self._v_scale) for _ in range(self._n_layers)]
        k_bytes, v_bytes = self.get_kv_size_bytes()
        self.mem_usage = (k_bytes + v_bytes) / 2**30
        self.token_stride = self.head_num * self.head_dim
        logger.info("[DirectKV] %d layers x (%d slots, %d KV heads) in 4 bits, %s memory: %.2f GiB", self._n_layers, self.n_slots, self.head_num,
                    self.location, self.mem_usage)

    def get_kv_size_bytes(self) -> Tuple[int, int]:
        half = self._n_layers * self.n_slots * self.head_num * (kernel.HEAD_DIM // 2 + kernel.HEAD_DIM // kernel.KV4_BLOCK)
        return half, half

    def layer_pool(self, layer_id: int) -> kernel.KV4Pool:
        """The layer's arrays, as ``kernel.store_kv4`` / ``load_kv4`` / ``decode_kv4`` take them (page size 1)."""
        return self._layers[self._li(layer_id)]

    # ---- KVCache interface -------------------------------------------------------
    def get_key_buffer(self, layer_id: int) -> torch.Tensor:
        raise NotImplementedError(_IN_4_BITS)

    def get_value_buffer(self, layer_id: int) -> torch.Tensor:
        raise NotImplementedError(_IN_4_BITS)

    def set_kv_buffer(self, layer, loc: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, k_scale: Optional[float] = None,
                      v_scale: Optional[float] = None, layer_id_override: Optional[int] = None) -> None:
        """Quantises ``cache_k/v [n, H, D]`` (device tensors) into slots ``loc [n]`` on the current stream."""
        for given, own, name in ((k_scale, self._k_scale, "k_scale"), (v_scale, self._v_scale, "v_scale")):
            if given is not None and float(given) != own:
                raise ValueError(f"{name}={given}: the pool was made with {own}")
        if not cache_k.is_cuda:
            raise RuntimeError("DirectKV4BitTokenToKVPool stores device tensors; there is no CPU quantiser")
        pool = self.layer_pool(layer_id_override if layer_id_override is not None else layer.layer_id)
        if loc.dtype not in (torch.int32, torch.int64):
            loc = loc.long()
        loc = loc.to(cache_k.device).contiguous()
        k = cache_k.to(self.dtype).reshape(-1, self.head_num, self.head_dim)
        v = cache_v.to(self.dtype).reshape(-1, self.head_num, self.head_dim)
        self._compute_device = cache_k.device
        with torch.cuda.device(cache_k.device):
            kernel.store_kv4(pool, loc, k, v)
            for t in (k, v, loc):                     # they must outlive the kernel: tie them to the stream
                t.record_stream(torch.cuda.current_stream())

    def load_rows(self, layer_id: int, loc: torch.Tensor, k_out: Optional[torch.Tensor] = None, v_out: Optional[torch.Tensor] = None):
        """Rows of slots ``loc [n]`` (device) as bf16 ``(k, v)`` ``[n, H, D]`` on the current stream."""
        return kernel.load_kv4(self.layer_pool(layer_id), loc, k_out, v_out)

    # ---- block moves: bytes are copied, so nothing is rounded again ---------------------
    @staticmethod
    def _arrays(pool: kernel.KV4Pool):
        return pool.k_codes, pool.k_scales, pool.v_codes, pool.v_scales

    def _move(self, dst: kernel.KV4Pool, dst_idx: torch.Tensor, src: kernel.KV4Pool, src_idx: torch.Tensor) -> None:
        if (dst.k_scale, dst.v_scale) != (src.k_scale, src.v_scale):
            raise ValueError("the two 4-bit pools have different scales")
        for a, b in zip(self._arrays(dst), self._arrays(src)):
            a[dst_idx.to(a.device)] = b[src_idx.to(b.device)].to(a.device)

    def move_kv_cache(self, tgt_loc: torch.Tensor, src_loc: torch.Tensor):
        self.synchronize()
        tgt, src = self._as_index(tgt_loc), self._as_index(src_loc)
        for pool in self._layers:
            self._move(pool, tgt, pool, src)

    def load_from_host_per_layer(self, host_pool, host_indices, device_indices, layer_id, io_backend):
        self.synchronize()
        host_pool.synchronize()
        self._move(self.layer_pool(layer_id), self._as_index(device_indices), host_pool.layer_pool(layer_id), self._as_index(host_indices))

    def backup_to_host_all_layer(self, host_pool, host_indices, device_indices, io_backend):
        self.synchronize()
        host_pool.synchronize()
        h_idx, d_idx = self._as_index(host_indices), self._as_index(device_indices)
        for li in range(len(self._layers)):
            lid = self.start_layer + li
            self._move(host_pool.layer_pool(lid), h_idx, self.layer_pool(lid), d_idx)
