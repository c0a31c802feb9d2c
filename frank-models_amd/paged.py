"""A paged K/V cache in 8 bits: appending new tokens to it, and attention of
one or more new tokens of each sequence over it.

Extensions of the decode step's cache (components/kvcache/kvcache.mlir holds
fp32; its prefill attends the new tokens alone,
components/attention/attention_block_prefill.mlir).  ``kvcache_append`` also
writes pools of the activations' type, where it stands for the rotation and
``kvcache_scatter_prefill`` / ``kvcache_scatter_decode`` of both pools.

Device tensors stay on the device and the calls are asynchronous on torch's
current stream; NumPy ``q`` / ``k`` / ``v`` are copied there, and the result
comes back as NumPy.  Pools are device tensors, updated in place.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib as L
from .api import _TORCH_TO_DT, _device, _finish, _ptr, _stream, _to_device, _workspace
from .attention import _ints_to_device


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


def _check_pool(pool, name, dev):
    """-> (data, scales or None) of a pool argument, checked."""
    data, scales = (pool.data, pool.scales) if isinstance(pool, QuantizedKVPool) else (pool, None)
    if not isinstance(data, torch.Tensor) or data.device != dev or not data.is_contiguous():
        raise TypeError(f"{name} must be a contiguous tensor on {dev}")
    if data.dim() != 4:
        raise ValueError(f"{name} must be [n_blocks, block_size, n_head_kv, head_dim], got {tuple(data.shape)}")
    if isinstance(pool, QuantizedKVPool):
        if data.dtype not in (torch.float8_e4m3fn, torch.uint8):
            raise TypeError(f"{name}: codes must be float8_e4m3fn or uint8, got {data.dtype}")
        if (not isinstance(scales, torch.Tensor) or scales.dtype != torch.float32 or scales.device != dev
                or not scales.is_contiguous()):
            raise TypeError(f"{name}: scales must be a contiguous float32 tensor on {dev}")
        if scales.shape != (data.shape[0], data.shape[2]):
            raise ValueError(f"{name}: scales must be [n_blocks, n_head_kv] = [{data.shape[0]}, {data.shape[2]}]")
    return data, scales


def _check_pools(k_cache, v_cache, dev):
    k, ks = _check_pool(k_cache, "k_cache", dev)
    v, vs = _check_pool(v_cache, "v_cache", dev)
    if k.shape != v.shape or (ks is None) != (vs is None) or (ks is None and k.dtype != v.dtype):
        raise ValueError(f"k_cache {tuple(k.shape)} and v_cache {tuple(v.shape)} must have one shape and type")
    if k.data_ptr() == v.data_ptr():
        raise ValueError("k_cache and v_cache must be two pools")
    return k, ks, v, vs


def _tokens(x, name, heads, dim, dev):
    """A [batch, seq_len, heads, dim] operand -> (tensor, elements between
    tokens, came from NumPy).  Views whose tokens lie at one stride, as the
    parts of a fused projection row do, are read in place; others are copied."""
    x, from_np = (x, False) if isinstance(x, torch.Tensor) and x.dtype in _TORCH_TO_DT and x.is_cuda else _to_device(x, name)
    if x.device != dev:
        raise ValueError(f"{name} must be on the current device {dev}, got {x.device}")
    if x.dim() != 4 or x.shape[3] != dim or (heads is not None and x.shape[2] != heads):
        want = f"[batch, seq_len, {'n_head' if heads is None else heads}, {dim}]"
        raise ValueError(f"{name} must be {want}, got {tuple(x.shape)}")
    B, S, H, _ = x.shape
    sb, ss, sh, sd = x.stride()
    token = ss if S > 1 else sb if B > 1 else H * dim
    if not ((sd == 1) and (sh == dim or H == 1) and (S == 1 or B == 1 or sb == S * ss) and token >= H * dim
            and token * x.element_size() % 16 == 0 and x.data_ptr() % 16 == 0):
        x = torch.empty(x.shape, dtype=x.dtype, device=x.device).copy_(x)
        token = H * dim
    return x, token, from_np


def _check_tables(block_tables, batch):
    bt = _ints_to_device(block_tables, "block_tables")
    if bt.dim() != 3 or bt.shape[1] != batch:
        raise ValueError(f"block_tables must be [n_layers, {batch}, max_blocks], got {tuple(bt.shape)}")
    return bt


def _per_sequence(a, name, batch):
    if a is None:
        return None
    t = _ints_to_device(a, name)
    if t.shape != (batch,):
        raise ValueError(f"{name} must be [{batch}], got {tuple(t.shape)}")
    return t


def kvcache_append(k_cache, v_cache, layer: int, k, v, block_tables, start_positions, *, seq_lens=None, q=None,
                   q_out=None, rope: bool = True, rope_freq_base: float = 10000.0, rope_freq_scale: float = 1.0):
    """Writes new tokens' keys, rotated at their positions, and values into
    the pages of ``block_tables [n_layers, batch, max_blocks]``, and returns
    ``q`` rotated the same way (None without ``q``).

    ``k``, ``v`` ``[batch, seq_len, n_head_kv, head_dim]`` and ``q [batch,
    seq_len, n_head, head_dim]``, of one type (float32 or bfloat16); token s
    of sequence b is position ``start_positions[b] + s``.  Tokens at and past
    ``seq_lens[b]`` are padding: not cached.  The pools are
    ``QuantizedKVPool`` (a block that the append begins takes the scale of
    its new values, one that it continues keeps its scale or grows it, with
    its rows) or tensors of the activations' type.  ``rope=False`` appends
    keys that are rotated already.  ``q_out`` takes the rotated queries (it
    may be ``q``).

    An append ends its sequence: rows behind it in its last block stand for
    nothing.  Positions without a block in the pool are skipped; a block
    that the call's tables name several times is written by the last
    sequence and position alone."""
    dev = _device()
    kc, ks, vc, vs = _check_pools(k_cache, v_cache, dev)
    n_blocks, bs, hkv, d = kc.shape
    k, k_stride, _ = _tokens(k, "k", hkv, d, dev)
    v, v_stride, _ = _tokens(v, "v", hkv, d, dev)
    if k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError(f"k {tuple(k.shape)} {k.dtype} and v {tuple(v.shape)} {v.dtype} must agree")
    if ks is None and kc.dtype != k.dtype:
        raise TypeError(f"a {kc.dtype} pool takes {kc.dtype} keys and values, got {k.dtype}")
    batch, seq_len = k.shape[:2]
    bt = _check_tables(block_tables, batch)
    start = _per_sequence(start_positions, "start_positions", batch)
    if start is None:
        raise ValueError("start_positions must be [batch]")
    lens = _per_sequence(seq_lens, "seq_lens", batch)
    n_head, q_stride, out_stride, from_np, q_out_copy = 1, 0, 0, False, None
    if q is not None:
        q, q_stride, from_np = _tokens(q, "q", None, d, dev)
        if q.dtype != k.dtype or q.shape[:2] != k.shape[:2]:
            raise ValueError(f"q {tuple(q.shape)} {q.dtype} does not go with k {tuple(k.shape)} {k.dtype}")
        n_head = q.shape[2]
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        if not isinstance(q_out, torch.Tensor) or q_out.dtype != q.dtype or q_out.shape != q.shape \
                or q_out.device != dev:
            raise ValueError(f"q_out must be a {q.dtype} tensor {tuple(q.shape)} on {dev}")
        out, out_stride, _ = _tokens(q_out, "q_out", n_head, d, dev)
        if out is not q_out:
            q_out_copy, q_out = q_out, out
    elif q_out is not None:
        raise ValueError("q_out without q")
    L.call("fmoe_kvcache_append", _ptr(kc), _ptr(vc), _ptr(ks), _ptr(vs),
           _TORCH_TO_DT[kc.dtype] if ks is None else L.F8E4M3FN, n_blocks, bs, hkv, d, int(layer), _ptr(k), k_stride,
           _ptr(v), v_stride, _ptr(q), q_stride, _ptr(q_out), out_stride, n_head, _TORCH_TO_DT[k.dtype], batch,
           seq_len, _ptr(bt), bt.shape[0], bt.shape[2], _ptr(start), _ptr(lens), int(bool(rope)),
           float(rope_freq_base), float(rope_freq_scale), _stream())
    if q is None:
        return None
    if q_out_copy is not None:
        q_out = q_out_copy.copy_(q_out)
    return _finish(q_out, from_np)


def attention_paged(q, k_cache, v_cache, layer: int, block_tables, context_lens, max_context_len: int, *,
                    seq_lens=None, causal: bool = True, scale=None, out=None):
    """Attention of the last ``seq_lens[b]`` (default: ``seq_len``) tokens of
    each context over ``QuantizedKVPool`` pages -> ``[batch, seq_len, n_head,
    head_dim]`` in ``q``'s type.

    ``q [batch, seq_len, n_head, head_dim]`` (float32 or bfloat16, rotated);
    ``context_lens [n_layers, batch]`` counts the cached positions, the new
    tokens' own among them (``kvcache_append`` first), so token s is position
    ``context_lens[layer, b] - seq_lens[b] + s``.  It attends the positions
    below ``min(context_lens[layer, b], max_context_len)``, causal ones only
    up to its own; ``scale`` defaults to ``1 / sqrt(head_dim)``.  Tokens that
    attend nothing, and padding tokens, get zeros.  ``out`` must not overlap
    ``q``."""
    dev = _device()
    if not isinstance(k_cache, QuantizedKVPool) or not isinstance(v_cache, QuantizedKVPool):
        raise TypeError("attention_paged reads QuantizedKVPool caches")
    kc, ks, vc, vs = _check_pools(k_cache, v_cache, dev)
    n_blocks, bs, hkv, d = kc.shape
    q, q_stride, from_np = _tokens(q, "q", None, d, dev)
    batch, seq_len, n_head, _ = q.shape
    bt = _check_tables(block_tables, batch)
    cl = _ints_to_device(context_lens, "context_lens")
    if cl.shape != bt.shape[:2]:
        raise ValueError(f"context_lens must be {tuple(bt.shape[:2])}, got {tuple(cl.shape)}")
    lens = _per_sequence(seq_lens, "seq_lens", batch)
    if scale is not None and not float(scale) > 0.0:
        raise ValueError("scale must be positive")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    elif not isinstance(out, torch.Tensor) or out.dtype != q.dtype or out.shape != q.shape or out.device != dev \
            or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {q.dtype} tensor {tuple(q.shape)} on {dev}")
    dt, mc = _TORCH_TO_DT[q.dtype], int(max_context_len)
    nbytes = L.lib().fmoe_attention_paged_workspace_bytes(batch, seq_len, mc, n_head, hkv, d, dt)
    ws = _workspace(nbytes) if nbytes else None
    L.call("fmoe_attention_paged", _ptr(q), q_stride, _ptr(kc), _ptr(ks), _ptr(vc), _ptr(vs), n_blocks, bs,
           int(layer), _ptr(bt), _ptr(cl), _ptr(lens), bt.shape[0], batch, seq_len, bt.shape[2], mc, n_head, hkv, d,
           int(bool(causal)), 0.0 if scale is None else float(scale), dt, _ptr(out), _ptr(ws), nbytes, _stream())
    return _finish(out, from_np)
