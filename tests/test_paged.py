"""The append to a paged cache and the attention over e4m3 pages without a
GPU: the oracle against plain loops and closed forms, and every refusal."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import numerics as nm
from oracle import paged as op

FAKE = 0x100000  # a non-null, aligned device address that nothing reads


def append_args(ll, **kw):
    a = dict(k_cache=FAKE, v_cache=FAKE, k_scales=FAKE, v_scales=FAKE, cache_dtype=ll.F8E4M3FN, n_blocks=8,
             block_size=4, n_head_kv=2, head_dim=16, layer=0, k=FAKE, k_stride=32, v=FAKE, v_stride=32, q=FAKE,
             q_stride=64, q_out=FAKE, q_out_stride=64, n_head=4, act_dtype=ll.BF16, batch=2, seq_len=3, tables=FAKE,
             n_layers=1, max_blocks=4, start=FAKE, seq_lens=None, rope=1, base=1e4, scale=1.0, stream=None)
    a.update(kw)
    return list(a.values())


def attn_args(ll, **kw):
    a = dict(q=FAKE, q_stride=64, k_cache=FAKE, k_scales=FAKE, v_cache=FAKE, v_scales=FAKE, n_blocks=8, block_size=4,
             layer=0, tables=FAKE, context=FAKE, seq_lens=None, n_layers=1, batch=2, seq_len=3, max_blocks=4,
             max_context=16, n_head=4, n_head_kv=2, head_dim=16, causal=1, scale=0.0, act=ll.BF16, out=FAKE,
             workspace=FAKE, nbytes=1 << 40, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(act_dtype=2), "ERR_DTYPE"), (dict(cache_dtype=0), "ERR_DTYPE"), (dict(cache_dtype=9), "ERR_DTYPE"),
    (dict(n_blocks=0), "ERR_SHAPE"), (dict(block_size=0), "ERR_SHAPE"),
    (dict(n_blocks=1 << 20, block_size=1 << 12), "ERR_SHAPE"),
    (dict(n_head_kv=0), "ERR_SHAPE"), (dict(head_dim=24), "ERR_SHAPE"), (dict(head_dim=256), "ERR_SHAPE"),
    (dict(head_dim=(1 << 32) + 16), "ERR_SHAPE"),
    (dict(layer=1), "ERR_SHAPE"), (dict(layer=-1), "ERR_SHAPE"), (dict(batch=-1), "ERR_SHAPE"),
    (dict(batch=65536), "ERR_SHAPE"), (dict(seq_len=-1), "ERR_SHAPE"), (dict(max_blocks=0), "ERR_SHAPE"),
    (dict(n_head=0), "ERR_SHAPE"), (dict(k_stride=31), "ERR_SHAPE"), (dict(q_out_stride=0), "ERR_SHAPE"),
    (dict(rope=2), "ERR_INVALID_ARGUMENT"), (dict(base=0.0), "ERR_INVALID_ARGUMENT"),
    (dict(base=float("nan")), "ERR_INVALID_ARGUMENT"), (dict(scale=float("inf")), "ERR_INVALID_ARGUMENT"),
    (dict(k_cache=None), "ERR_INVALID_ARGUMENT"), (dict(v_scales=None), "ERR_INVALID_ARGUMENT"),
    (dict(k=None), "ERR_INVALID_ARGUMENT"), (dict(tables=None), "ERR_INVALID_ARGUMENT"),
    (dict(start=None), "ERR_INVALID_ARGUMENT"), (dict(q_out=None), "ERR_INVALID_ARGUMENT"),
    (dict(k=FAKE + 8), "ERR_INVALID_ARGUMENT"), (dict(v_stride=36), "ERR_INVALID_ARGUMENT"),
    (dict(v_cache=FAKE + 8), "ERR_INVALID_ARGUMENT"),
])
def test_append_refuses(fm, kw, status):
    ll = fm.lowlevel
    assert ll.lib().fmoe_kvcache_append(*append_args(ll, **kw)) == getattr(ll, status), ll.last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(act=2), "ERR_DTYPE"), (dict(head_dim=48), "ERR_SHAPE"), (dict(n_head=3), "ERR_SHAPE"),
    (dict(n_head=1), "ERR_SHAPE"), (dict(layer=1), "ERR_SHAPE"), (dict(max_context=-1), "ERR_SHAPE"),
    (dict(max_context=1 << 31), "ERR_SHAPE"), (dict(batch=65536), "ERR_SHAPE"), (dict(q_stride=63), "ERR_SHAPE"),
    (dict(seq_len=1 << 30), "ERR_SHAPE"), (dict(block_size=1 << 30), "ERR_SHAPE"),
    (dict(causal=2), "ERR_INVALID_ARGUMENT"), (dict(scale=-1.0), "ERR_INVALID_ARGUMENT"),
    (dict(scale=float("nan")), "ERR_INVALID_ARGUMENT"), (dict(scale=float("inf")), "ERR_INVALID_ARGUMENT"),
    (dict(k_scales=None), "ERR_INVALID_ARGUMENT"), (dict(v_cache=None), "ERR_INVALID_ARGUMENT"),
    (dict(context=None), "ERR_INVALID_ARGUMENT"), (dict(out=None), "ERR_INVALID_ARGUMENT"),
    (dict(out=FAKE + 2), "ERR_INVALID_ARGUMENT"), (dict(q=FAKE + 2), "ERR_INVALID_ARGUMENT"),
    (dict(q=None), "ERR_INVALID_ARGUMENT"), (dict(k_cache=FAKE + 4), "ERR_INVALID_ARGUMENT"),
])
def test_attention_refuses(fm, kw, status):
    ll = fm.lowlevel
    assert ll.lib().fmoe_attention_paged(*attn_args(ll, **kw)) == getattr(ll, status), ll.last_error()


def step_args(ll, sublayer=False, **kw):
    a = dict(x=FAKE, norm=FAKE, eps=1e-5) if sublayer else dict(x=FAKE)
    a.update(positions=FAKE, k_cache=FAKE, v_cache=FAKE, k_scales=FAKE, v_scales=FAKE, n_blocks=8, block_size=4,
             layer=0, tables=FAKE, context=FAKE, n_layers=1, max_blocks=4, max_context=16, blocks=FAKE, rows=FAKE,
             wqkv=FAKE, wqkv_scales=None, wo=FAKE, wo_scales=None, w_dtype=ll.BF16, bq=None, bk=None, bv=None, bo=None,
             use_bias=0, batch=2, n_head=4, n_head_kv=2, n_embd=64, n_embd_kv=32, base=1e4, scale=1.0, act=ll.BF16,
             out=FAKE, k_new=FAKE, v_new=FAKE, workspace=FAKE, nbytes=1 << 40, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("sublayer", [False, True])
@pytest.mark.parametrize("kw,status", [
    (dict(act=2), "ERR_DTYPE"), (dict(n_head=3), "ERR_SHAPE"), (dict(layer=1), "ERR_SHAPE"),
    (dict(block_size=1 << 30), "ERR_SHAPE"), (dict(max_blocks=0), "ERR_SHAPE"),
    (dict(max_context=(1 << 31) - 4096), "ERR_SHAPE"), (dict(max_context=-1), "ERR_SHAPE"),
    (dict(k_scales=None), "ERR_INVALID_ARGUMENT"), (dict(v_scales=None), "ERR_INVALID_ARGUMENT"),
    (dict(v_cache=None), "ERR_INVALID_ARGUMENT"), (dict(blocks=None), "ERR_INVALID_ARGUMENT"),
    (dict(k_cache=FAKE + 8), "ERR_INVALID_ARGUMENT"), (dict(k_new=FAKE + 8), "ERR_INVALID_ARGUMENT"),
    (dict(workspace=None), "ERR_INVALID_ARGUMENT"), (dict(nbytes=64), "ERR_WORKSPACE"),
])
def test_decode_step_refuses(fm, sublayer, kw, status):
    ll = fm.lowlevel
    fn = f"fmoe_attention_{'sublayer_' if sublayer else ''}decode_paged_f8"
    assert getattr(ll.lib(), fn)(*step_args(ll, sublayer, **kw)) == getattr(ll, status), ll.last_error()
    assert getattr(ll.lib(), fn)(*step_args(ll, sublayer, batch=0)) == ll.OK or sublayer
    room = getattr(ll.lib(), fn + "_workspace_bytes")
    assert room(2, 16, 4, 2, 64, 32, ll.BF16) > 0
    for bad in ((-1, 16, 4, 2, 64, 32), (2, 1 << 31, 4, 2, 64, 32), (2, 16, 4, 3, 64, 32), (2, 16, 0, 2, 64, 32)):
        assert room(*bad, ll.BF16) == 0


def test_attention_workspace_is_checked(fm):
    """A decode step behind a long context is cut over blocks, whose partial results need room."""
    ll = fm.lowlevel
    shape = dict(batch=1, seq_len=1, max_context=1 << 16, n_blocks=1 << 13, block_size=16, n_head=32, n_head_kv=8,
                 head_dim=128, q_stride=4096)
    need = ll.lib().fmoe_attention_paged_workspace_bytes(1, 1, 1 << 16, 32, 8, 128, ll.BF16)
    for bad in (-1, 1 << 31):
        assert ll.lib().fmoe_attention_paged_workspace_bytes(1, bad, 64, 32, 8, 128, ll.BF16) == 0
    assert ll.lib().fmoe_attention_paged_workspace_bytes(1, 1, 64, 32, 5, 128, ll.BF16) == 0
    if need:
        assert ll.lib().fmoe_attention_paged(*attn_args(ll, **shape, nbytes=need - 1)) == ll.ERR_WORKSPACE
        assert ll.lib().fmoe_attention_paged(*attn_args(ll, **shape, workspace=None)) == ll.ERR_INVALID_ARGUMENT
        assert ll.lib().fmoe_attention_paged(*attn_args(ll, **shape, workspace=FAKE + 16)) == ll.ERR_INVALID_ARGUMENT


def test_empty_calls_are_no_ops(fm):
    ll = fm.lowlevel
    for kw in (dict(batch=0), dict(seq_len=0)):
        assert ll.lib().fmoe_kvcache_append(*append_args(ll, k=None, **kw)) == ll.OK
        assert ll.lib().fmoe_attention_paged(*attn_args(ll, q=None, **kw)) == ll.OK


@pytest.mark.skipif(torch.cuda.is_available(), reason="a GPU is visible")
def test_no_device_is_an_error(fm):
    ll = fm.lowlevel
    assert ll.lib().fmoe_kvcache_append(*append_args(ll)) == ll.ERR_NO_DEVICE
    assert ll.lib().fmoe_attention_paged(*attn_args(ll)) == ll.ERR_NO_DEVICE
    with pytest.raises(fm.NoDeviceError):
        fm.QuantizedKVPool.zeros(4, 4, 2, 16)
    with pytest.raises(fm.NoDeviceError):
        fm.kvcache_append(None, None, 0, None, None, None, None)
    with pytest.raises(fm.NoDeviceError):
        fm.attention_paged(None, None, None, 0, None, None, 4)


# ---------------------------------------------------------------- the oracle
def test_oracle_rope_is_a_rotation():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((5, 2, 16))
    y = op.rope(x, [0, 1, 7, 100000, -3])
    np.testing.assert_array_equal(y[0], x[0])
    np.testing.assert_allclose(np.linalg.norm(y, axis=-1), np.linalg.norm(x, axis=-1), rtol=1e-14)
    # the product of two rotated vectors depends on the distance alone
    a, b = op.rope(np.repeat(x[:1], 2, 0), [11, 40]), op.rope(np.repeat(x[1:2], 2, 0), [5, 34])
    np.testing.assert_allclose((a * b).sum(-1)[0], (a * b).sum(-1)[1], rtol=1e-12)
    z = (x[1, 0, 0] + 1j * x[1, 0, 1]) * np.exp(1j)  # pair 0 turns by the position
    np.testing.assert_allclose(y[1, 0, :2], [z.real, z.imag], rtol=1e-14)


@pytest.mark.parametrize("a", [0.0, 1e-40, 1.0, 448.0, np.nextafter(448.0, 500), 896.0, 3e30])
def test_oracle_scale(a):
    s = op.pow2_scale(a)
    assert a <= 448 * s and (s == 2.0 ** -126 or a > 224 * s)


def test_oracle_append_in_pieces_keeps_values():
    """Rows appended one by one stay within half a code step at the page's last
    scale of their values, at a grown scale a second half step of what falls
    below the codes' smallest normal value."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((1, 11, 2, 16)) * np.exp(rng.uniform(-3, 3, (1, 11, 1, 1)))
    codes, scales = np.zeros((3, 4, 2, 16), np.uint8), np.zeros((3, 2), np.float32)
    table = np.array([[2, 0, 1]])
    for s in range(11):
        op.append(codes, scales, x[:, s : s + 1], table, [s], [1])
    got = op.values(codes, scales)
    for s in range(11):
        page = table[0, s // 4]
        err = np.abs(got[page, s % 4] - x[0, s])
        assert np.all(err <= 2.0 ** -4 * np.abs(x[0, s]) + 2 * 2.0 ** -10 * scales[page][:, None])


def test_oracle_append_last_of_a_shared_page_wins():
    codes, scales = np.zeros((2, 2, 1, 16), np.uint8), np.zeros((2, 1), np.float32)
    x = np.stack([np.full((2, 1, 16), v) for v in (1.0, 2.0, 3.0)])
    done = op.append(codes, scales, x, np.array([[0], [0], [1]]), [0, 0, 0], [2, 1, 2])
    assert done == {(0, 0), (1, 0), (1, 1)}
    assert np.all(op.values(codes, scales)[0, 0] == 2.0) and np.all(codes[0, 1] == 0)


def test_oracle_attention_against_torch():
    rng = np.random.default_rng(2)
    k, v = rng.standard_normal((2, 4, 4, 2, 16))
    zero = np.zeros((1, 4, 2, 16))
    q = rng.standard_normal((1, 5, 4, 16))
    table = np.array([[3, 1, 0]])
    out, _ = op.attention(q, np.concatenate([k, zero]), np.concatenate([v, zero]), table, [10], 12, [5])
    flat = lambda p: torch.from_numpy(p[[3, 1, 0]].reshape(12, 2, 16)[:10]).transpose(0, 1).repeat_interleave(2, 0)  # noqa: E731
    mask = torch.ones(5, 10, dtype=torch.bool).tril(5)
    ref = torch.nn.functional.scaled_dot_product_attention(torch.from_numpy(q[0]).transpose(0, 1), flat(k), flat(v),
                                                           attn_mask=mask)
    np.testing.assert_allclose(out[0], ref.transpose(0, 1).numpy(), rtol=1e-12)


def test_oracle_attention_of_nothing_is_zero():
    k = np.concatenate([np.ones((1, 4, 1, 16)), np.zeros((1, 4, 1, 16))])
    out, _ = op.attention(np.ones((2, 3, 1, 16)), k, k, np.zeros((2, 1), int), [0, 2], 4, [3, 3])
    assert not out[0].any() and not out[1, 0].any() and np.all(out[1, 1:] == 1)  # one context shorter than its tokens
    # a page outside the pool: keys and values of zeros
    out, _ = op.attention(np.ones((1, 1, 1, 16)), k, k, np.array([[5]]), [3], 4, [1])
    assert not out.any()


def test_oracle_codes_of_what_is_not_finite():
    codes, scales = np.zeros((1, 2, 1, 16), np.uint8), np.zeros((1, 1), np.float32)
    x = np.ones((1, 2, 1, 16))
    x[0, 0, 0, :3] = np.nan, np.inf, -np.inf
    op.append(codes, scales, x, np.array([[0]]), [0], [2])
    got = nm.e4m3fn_decode(codes)[0, 0, 0] * scales[0]
    assert np.isnan(got[:3]).all() and np.all(got[3:] == 1)
