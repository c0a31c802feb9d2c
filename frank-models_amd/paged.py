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

import functools

import torch

from . import _lib as L
from .api import _TORCH_TO_DT, _device, _finish, _to_device
from .attention import _ints_to_device
from .kvpool import QuantizedKVPool, check_pools, here

# A decode step makes a call of each per layer, whose kernels take a few
# microseconds: the checks ask tensors for plain numbers (device index, shape,
# strides) and leave what is in order as it is.


def _raw_stream(dev: int) -> int:
    return torch._C._cuda_getCurrentRawStream(dev)


def _tokens(x, name, heads, dim, dev):
    """A [batch, seq_len, heads, dim] operand -> (tensor, elements between
    tokens, shape, came from NumPy).  Views whose tokens lie at one stride, as
    the parts of a fused projection row do, are read in place; others are
    copied."""
    from_np = False
    if not (isinstance(x, torch.Tensor) and x.is_cuda and x.dtype in _TORCH_TO_DT):
        x, from_np = _to_device(x, name)
    if x.get_device() != dev:
        raise ValueError(f"{name} must be on the current device, cuda:{dev}, got {x.device}")
    shape = x.shape
    if len(shape) != 4 or shape[3] != dim or (heads is not None and shape[2] != heads):
        want = f"[batch, seq_len, {'n_head' if heads is None else heads}, {dim}]"
        raise ValueError(f"{name} must be {want}, got {tuple(shape)}")
    B, S, H, _ = shape
    sb, ss, sh, sd = x.stride()
    token = ss if S > 1 else sb if B > 1 else H * dim
    if not (sd == 1 and (sh == dim or H == 1) and (S == 1 or B == 1 or sb == S * ss) and token >= H * dim
            and token * x.element_size() % 16 == 0 and x.data_ptr() % 16 == 0):
        x = torch.empty(shape, dtype=x.dtype, device=x.device).copy_(x)
        token = H * dim
    return x, token, shape, from_np


def _ints(a, name):
    if type(a) is torch.Tensor and a.dtype is torch.int32 and a.is_cuda and a.is_contiguous():
        return a
    return _ints_to_device(a, name)


def _check_tables(block_tables, batch, dev):
    """-> (block_tables, n_layers, max_blocks)."""
    bt = _ints(block_tables, "block_tables")
    shape = bt.shape
    if len(shape) != 3 or shape[1] != batch:
        raise ValueError(f"block_tables must be [n_layers, {batch}, max_blocks], got {tuple(shape)}")
    if bt.get_device() != dev:
        raise ValueError(f"block_tables must be on the current device, cuda:{dev}")
    return bt, shape[0], shape[2]


def _per_sequence(a, name, batch, dev):
    t = _ints(a, name)
    if t.shape != (batch,):
        raise ValueError(f"{name} must be [{batch}], got {tuple(t.shape)}")
    if t.get_device() != dev:
        raise ValueError(f"{name} must be on the current device, cuda:{dev}")
    return t


@functools.lru_cache(maxsize=256)
def _workspace_bytes(batch, seq_len, max_context_len, n_head, n_head_kv, head_dim, dt):
    return L.lib().fmoe_attention_paged_workspace_bytes(batch, seq_len, max_context_len, n_head, n_head_kv, head_dim,
                                                        dt)


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
    dev = here()
    kc, ks, vc, vs, (n_blocks, bs, hkv, d) = check_pools(k_cache, v_cache, dev)
    k, k_stride, shape, _ = _tokens(k, "k", hkv, d, dev)
    v, v_stride, v_shape, _ = _tokens(v, "v", hkv, d, dev)
    dtype = k.dtype
    if shape != v_shape or dtype is not v.dtype:
        raise ValueError(f"k {tuple(shape)} {dtype} and v {tuple(v_shape)} {v.dtype} must agree")
    if ks is None and kc.dtype is not dtype:
        raise TypeError(f"a {kc.dtype} pool takes {kc.dtype} keys and values, got {dtype}")
    batch, seq_len = shape[0], shape[1]
    bt, n_layers, max_blocks = _check_tables(block_tables, batch, dev)
    start = _per_sequence(start_positions, "start_positions", batch, dev)
    lens = None if seq_lens is None else _per_sequence(seq_lens, "seq_lens", batch, dev)
    n_head, q_stride, out, out_stride, from_np = 1, 0, None, 0, False
    if q is not None:
        q, q_stride, q_shape, from_np = _tokens(q, "q", None, d, dev)
        if q.dtype is not dtype or q_shape[0] != batch or q_shape[1] != seq_len:
            raise ValueError(f"q {tuple(q_shape)} {q.dtype} does not go with k {tuple(shape)} {dtype}")
        n_head = q_shape[2]
        if q_out is None:
            q_out = out = q.new_empty(q_shape)
            out_stride = n_head * d
        elif (not isinstance(q_out, torch.Tensor) or q_out.dtype is not dtype or q_out.shape != q_shape
              or q_out.get_device() != dev):
            raise ValueError(f"q_out must be a {dtype} tensor {tuple(q_shape)} on cuda:{dev}")
        else:
            out, out_stride, _, _ = _tokens(q_out, "q_out", n_head, d, dev)
    elif q_out is not None:
        raise ValueError("q_out without q")
    L.call("fmoe_kvcache_append", kc.data_ptr(), vc.data_ptr(), None if ks is None else ks.data_ptr(),
           None if vs is None else vs.data_ptr(), _TORCH_TO_DT[dtype] if ks is None else L.F8E4M3FN, n_blocks, bs, hkv,
           d, int(layer), k.data_ptr(), k_stride, v.data_ptr(), v_stride, None if q is None else q.data_ptr(), q_stride,
           None if out is None else out.data_ptr(), out_stride, n_head, _TORCH_TO_DT[dtype], batch, seq_len,
           bt.data_ptr(), n_layers, max_blocks, start.data_ptr(), None if lens is None else lens.data_ptr(),
           int(bool(rope)), float(rope_freq_base), float(rope_freq_scale), _raw_stream(dev))
    if q is None:
        return None
    if out is not q_out:
        q_out.copy_(out)
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
    dev = here()
    if not isinstance(k_cache, QuantizedKVPool) or not isinstance(v_cache, QuantizedKVPool):
        raise TypeError("attention_paged reads QuantizedKVPool caches")
    kc, ks, vc, vs, (n_blocks, bs, hkv, d) = check_pools(k_cache, v_cache, dev)
    q, q_stride, shape, from_np = _tokens(q, "q", None, d, dev)
    batch, seq_len, n_head, _ = shape
    dtype = q.dtype
    bt, n_layers, max_blocks = _check_tables(block_tables, batch, dev)
    cl = _ints(context_lens, "context_lens")
    if cl.shape != (n_layers, batch):
        raise ValueError(f"context_lens must be [{n_layers}, {batch}], got {tuple(cl.shape)}")
    if cl.get_device() != dev:
        raise ValueError(f"context_lens must be on the current device, cuda:{dev}")
    lens = None if seq_lens is None else _per_sequence(seq_lens, "seq_lens", batch, dev)
    if scale is not None and not float(scale) > 0.0:
        raise ValueError("scale must be positive")
    if out is None:
        out = q.new_empty(shape)
    elif not isinstance(out, torch.Tensor) or out.dtype is not dtype or out.shape != shape or out.get_device() != dev \
            or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {dtype} tensor {tuple(shape)} on cuda:{dev}")
    dt, max_context_len = _TORCH_TO_DT[dtype], int(max_context_len)
    nbytes = _workspace_bytes(batch, seq_len, max_context_len, n_head, hkv, d, dt)
    # of this call alone: calls on other streams, and captured ones, share nothing
    ws = kc.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    L.call("fmoe_attention_paged", q.data_ptr(), q_stride, kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr(),
           n_blocks, bs, int(layer), bt.data_ptr(), cl.data_ptr(), None if lens is None else lens.data_ptr(), n_layers,
           batch, seq_len, max_blocks, max_context_len, n_head, hkv, d, int(bool(causal)),
           0.0 if scale is None else float(scale), dt, out.data_ptr(), None if ws is None else ws.data_ptr(), nbytes,
           _raw_stream(dev))
    return _finish(out, from_np)
