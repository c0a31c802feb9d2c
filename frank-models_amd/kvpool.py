"""The paged K/V pool in 8 bits, and the checks of pool arguments."""

from __future__ import annotations

from dataclasses import dataclass

import torch

from .api import _device


def here() -> int:
    """The current device's index."""
    if not torch.cuda.is_initialized():
        _device()  # NoDeviceError where there is none
    return torch.cuda.current_device()


@dataclass
class QuantizedKVPool:
    """A K or V pool in OCP fp8-e4m3: ``data [n_blocks, block_size, n_head_kv,
    head_dim]`` (torch.float8_e4m3fn or uint8 codes) and ``scales [n_blocks,
    n_head_kv]`` float32, both contiguous on the device.  A value is
    ``decode(data) * scales`` of its block and head."""

    data: torch.Tensor
    scales: torch.Tensor

    @classmethod
    def zeros(cls, n_blocks: int, block_size: int, n_head_kv: int, head_dim: int) -> "QuantizedKVPool":
        dev = _device()
        data = torch.zeros((n_blocks, block_size, n_head_kv, head_dim), dtype=torch.uint8, device=dev)
        return cls(data.view(torch.float8_e4m3fn), torch.zeros((n_blocks, n_head_kv), dtype=torch.float32, device=dev))

    @property
    def shape(self):
        return tuple(self.data.shape)

    def dequantize(self) -> torch.Tensor:
        """The values, float32."""
        return self.data.view(torch.float8_e4m3fn).float() * self.scales[:, None, :, None]


_CODES = (torch.float8_e4m3fn, torch.uint8)


def _check_pool(pool, name, dev):
    """-> (data, scales or None, shape) of a pool argument, checked."""
    quantized = isinstance(pool, QuantizedKVPool)
    data, scales = (pool.data, pool.scales) if quantized else (pool, None)
    if not isinstance(data, torch.Tensor) or data.get_device() != dev or not data.is_contiguous():
        raise TypeError(f"{name} must be a contiguous tensor on the current device, cuda:{dev}")
    shape = data.shape
    if len(shape) != 4:
        raise ValueError(f"{name} must be [n_blocks, block_size, n_head_kv, head_dim], got {tuple(shape)}")
    if quantized:
        if data.dtype not in _CODES:
            raise TypeError(f"{name}: codes must be float8_e4m3fn or uint8, got {data.dtype}")
        if (not isinstance(scales, torch.Tensor) or scales.dtype is not torch.float32 or scales.get_device() != dev
                or not scales.is_contiguous()):
            raise TypeError(f"{name}: scales must be a contiguous float32 tensor on the current device, cuda:{dev}")
        if scales.shape != (shape[0], shape[2]):
            raise ValueError(f"{name}: scales must be [n_blocks, n_head_kv] = [{shape[0]}, {shape[2]}]")
    return data, scales, shape


def check_pools(k_cache, v_cache, dev):
    k, ks, shape = _check_pool(k_cache, "k_cache", dev)
    v, vs, v_shape = _check_pool(v_cache, "v_cache", dev)
    if shape != v_shape or (ks is None) != (vs is None) or (ks is None and k.dtype is not v.dtype):
        raise ValueError(f"k_cache {tuple(shape)} and v_cache {tuple(v_shape)} must have one shape and type")
    if k.data_ptr() == v.data_ptr() and k.numel():
        raise ValueError("k_cache and v_cache must be two pools")
    return k, ks, v, vs, shape
