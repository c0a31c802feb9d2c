"""The append to a paged cache and the attention over e4m3 pages on the GPU,
against the 64-bit oracle, at the sizes, masks, strides and contents where
they can go wrong."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import assert_close_rms
from oracle import attention as oa
from oracle import numerics as nm
from oracle import paged as op

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}


def rounded(a, act):
    a = np.asarray(a, np.float32)
    return nm.bf16_round(a) if act == "bf16" else a


def dev(a, act=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t.to(DT[act]) if act else t


def random_pool(rng, n_blocks, bs, hkv, d):
    """Codes of normal values and a scale for each page and head, spread over a few binades and no powers of two."""
    x = rng.standard_normal((n_blocks, bs, hkv, d))
    scales = (np.exp2(rng.uniform(-9, -5, (n_blocks, hkv)))).astype(np.float32)
    return nm.e4m3fn_encode((x / (448 * scales[:, None, :, None]) * 448).clip(-448, 448)), scales


def gpu_pool(fm, codes, scales):
    return fm.QuantizedKVPool(dev(codes).view(torch.float8_e4m3fn), dev(scales))


def codes_of(pool):
    return pool.data.view(torch.uint8).cpu().numpy()


# ---------------------------------------------------------------- append
def check_append(fm, rng, act, pool, B, S, H, Hkv, D, bs, start, lens, table, n_blocks, fused=False, base=10000.0,
                 fscale=1.0, rope=True):
    x = rounded(rng.standard_normal((B, S, (H + 2 * Hkv) * D)) * np.exp(rng.uniform(-2, 2, (B, S, 1))), act)
    q, k, v = (p.reshape(B, S, -1, D) for p in np.split(x, [H * D, (H + Hkv) * D], axis=2))
    xd = dev(x, act)
    qd, kd, vd = (p.unflatten(2, (-1, D)) for p in xd.split([H * D, Hkv * D, Hkv * D], dim=2))
    if not fused:
        qd, kd, vd = (p.contiguous() for p in (qd, kd, vd))
    codes = pool == "e4m3"
    if codes:
        (kc, ks), (vc, vs) = (random_pool(rng, n_blocks, bs, Hkv, D) for _ in range(2))
        kp, vp = gpu_pool(fm, kc, ks), gpu_pool(fm, vc, vs)
    else:
        kc, vc = (rounded(rng.standard_normal((n_blocks, bs, Hkv, D)), act).astype(np.float64) for _ in range(2))
        ks = vs = None
        kp, vp = dev(kc.astype(np.float32), act), dev(vc.astype(np.float32), act)
    before = kc.copy(), vc.copy(), None if ks is None else (ks.copy(), vs.copy())
    tables = np.stack([np.full_like(table, -7), table])  # layer 1 is the call's
    n = np.full(B, S) if lens is None else np.asarray(lens)
    got_q = fm.kvcache_append(kp, vp, 1, kd, vd, dev(tables.astype(np.int32)), dev(np.asarray(start, np.int32)),
                              seq_lens=None if lens is None else dev(np.asarray(lens, np.int32)), q=qd, rope=rope,
                              rope_freq_base=base, rope_freq_scale=fscale)
    torch.cuda.synchronize()
    pos = np.asarray(start)[:, None] + np.arange(S)
    turn = (lambda a: np.stack([op.rope(a[b], pos[b], base, fscale) for b in range(B)])) if rope else np.float64
    ref_q, ref_k = turn(q), turn(k)
    # cos, sin and the two products are rounded once each: 3 half steps of the pair's magnitudes, then the type's own
    pair = lambda a: np.repeat(np.abs(a.astype(np.float64)).reshape(*a.shape[:3], D // 2, 2).sum(-1), 2, -1)  # noqa: E731
    turned = 4 * 2.0 ** -24 if rope else 0.0
    tol_q = turned * pair(q) + (HALF[act] if rope else 0.0) * np.abs(ref_q)
    assert np.all(np.abs(got_q.double().cpu().numpy() - ref_q) <= tol_q + 1e-30)
    done = op.append(kc, ks, ref_k, table, start, n)
    op.append(vc, vs, v.astype(np.float64), table, start, n)
    written = np.zeros((n_blocks, bs), bool)
    for p in done:
        written[p] = True
    if not codes:
        for got, ref, old, exact in ((kp, kc, before[0], not rope), (vp, vc, before[1], True)):
            got = got.double().cpu().numpy()
            assert np.array_equal(got[~written], old[~written])
            tol = 0.0 if exact else HALF[act] * np.abs(ref) + turned * 2 * np.max(np.abs(x))
            assert np.all(np.abs(got - ref)[written] <= (tol if exact else tol[written]))
        return
    assert np.array_equal(kp.scales.cpu().numpy(), ks) and np.array_equal(vp.scales.cpu().numpy(), vs)
    assert np.array_equal(codes_of(vp), vc)  # no rotation: the same codes
    gk = codes_of(kp)
    assert np.array_equal(gk[~written], kc[~written])  # the rows that were rounded again, and those left alone
    # a rotated key off by `turned` may round to the other neighbour: half a
    # step (2^-4 of the value, 2^-10 of the scale below the normal values)
    val, at = nm.e4m3fn_decode(gk) * ks[:, None, :, None], nm.e4m3fn_decode(kc) * ks[:, None, :, None]
    flips = gk != kc
    assert np.all(np.abs(val - at)[flips] <= 2 * np.maximum(2.0 ** -4 * np.abs(at), 2.0 ** -10 * ks[:, None, :, None] + 0 * at)[flips] * 1.07)
    assert flips.mean() <= 1e-4 + 2 / flips.size


APPENDS = [
    # B, S, H, Hkv, D, bs, start, lens
    (2, 1, 4, 2, 16, 4, [10, 3], None),
    (3, 1, 8, 1, 64, 16, [0, 15, 16], None),
    (5, 1, 32, 8, 128, 16, [0, 1, 15, 31, 4097], [1, 1, 0, 1, 1]),
    (1, 37, 4, 4, 32, 16, [5], None),
    (3, 70, 6, 2, 128, 32, [0, 31, 50], [70, 1, 33]),
    (2, 9, 4, 2, 16, 1, [0, 7], [9, 4]),
    (2, 150, 2, 1, 128, 100, [3, 99], [150, 120]),
    (1, 300, 2, 1, 128, 256, [200], None),
    (1, 700, 1, 1, 16, 640, [639], None),
    (2, 3, 1, 1, 128, 7, [2000000, 1 << 20], None),
]


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("pool", ["e4m3", "same"])
@pytest.mark.parametrize("B,S,H,Hkv,D,bs,start,lens", APPENDS)
def test_append(fm, act, pool, B, S, H, Hkv, D, bs, start, lens):
    rng = np.random.default_rng(B * S + D + bs)
    far = max(start) > 100000  # the tables would be long: only the pages at the new tokens exist
    per = (max(start) + S - 1) // bs + 1
    near = (min(start) if far else 0) // bs
    used = 3 if far else per
    table = np.full((B, per), -1)
    order = rng.permutation(B * used)
    for b in range(B):
        first = start[b] // bs if far else near
        n = min(used, per - first)
        table[b, first : first + n] = order[b * used : b * used + n]
    check_append(fm, rng, act, pool, B, S, H, Hkv, D, bs, start, lens, table, B * used, fused=S % 2 == 1)


def test_append_without_rotation_and_other_frequencies(fm):
    rng = np.random.default_rng(3)
    table = rng.permutation(8).reshape(2, 4)
    check_append(fm, rng, "bf16", "e4m3", 2, 5, 4, 2, 64, 8, [6, 20], [5, 3], table, 8, rope=False)
    check_append(fm, rng, "f32", "e4m3", 2, 5, 4, 2, 64, 8, [6, 20], None, table, 8, base=500000.0, fscale=0.25)


def test_append_bad_pages_and_positions_are_skipped(fm):
    """Entries outside the pool, positions past the table and before the sequence."""
    rng = np.random.default_rng(4)
    table = np.array([[0, 9, 2, -1], [3, 4, 1 << 30, 5], [6, 7, 8, 1]])
    for pool in ("e4m3", "same"):
        check_append(fm, rng, "bf16", pool, 3, 14, 2, 1, 32, 4, [1, 5, -3], None, table, 9)


def test_append_last_of_a_shared_page_wins(fm):
    rng = np.random.default_rng(5)
    table = np.array([[0, 1, 2], [3, 1, 4], [5, 6, 5]])
    for pool in ("e4m3", "same"):
        check_append(fm, rng, "f32", pool, 3, 6, 2, 1, 16, 2, [0, 1, 0], [6, 3, 6], table, 7)


def test_append_what_is_not_finite(fm):
    codes, scales = np.zeros((2, 4, 1, 16), np.uint8), np.ones((2, 1), np.float32)
    kp, vp = gpu_pool(fm, codes, scales), gpu_pool(fm, codes, scales)
    x = torch.ones(1, 2, 1, 16, device="cuda")
    x[0, 0, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1e-42])
    fm.kvcache_append(kp, vp, 0, x, x, dev(np.array([[[1]]], np.int32)), dev(np.array([0], np.int32)), rope=False)
    v = vp.dequantize()[1].cpu()
    assert torch.isnan(v[0, 0, :3]).all() and v[0, 0, 3] == 0 and torch.all(v[0, 0, 4:] == 1) and torch.all(v[1] == 1)
    zero = torch.zeros(1, 1, 1, 16, device="cuda")  # nothing but zeros: the least scale, which the next append grows
    fm.kvcache_append(kp, vp, 0, zero, zero, dev(np.array([[[0]]], np.int32)), dev(np.array([0], np.int32)))
    assert vp.scales[0, 0].item() == 2.0 ** -126
    fm.kvcache_append(kp, vp, 0, zero + 1e-3, zero + 1e-3, dev(np.array([[[0]]], np.int32)),
                      dev(np.array([1], np.int32)), rope=False)
    v = vp.dequantize()[0, :2, 0, 0].cpu()
    assert v[0] == 0 and abs(v[1] - 1e-3) <= 2.0 ** -4 * 1e-3


def test_append_in_place_views_and_pools_of_bytes(fm):
    """q_out = q, other strides and orders than contiguous, uint8 pools, NumPy inputs."""
    rng = np.random.default_rng(6)
    x = rng.standard_normal((2, 3, 4, 32)).astype(np.float32)
    table, start = dev(np.array([[[0, 1], [2, 3]]], np.int32)), np.array([3, 0], np.int64)

    def run(q, k, **kw):
        kp, vp = (fm.QuantizedKVPool(torch.zeros(4, 4, 4, 32, dtype=torch.uint8, device="cuda"),
                                     torch.zeros(4, 4, device="cuda")) for _ in range(2))
        out = fm.kvcache_append(kp, vp, 0, k, k, table, start, q=q, **kw)
        return out, kp

    want, wk = run(dev(x), dev(x))
    got, gk = run(x, x)
    assert isinstance(got, np.ndarray) and np.array_equal(got, want.cpu().numpy())
    assert torch.equal(gk.data, wk.data) and torch.equal(gk.scales, wk.scales)
    odd = torch.zeros(1 + x.size, device="cuda")[1:].view(x.shape).copy_(dev(x))  # 4-byte aligned
    turned = dev(x.transpose(2, 0, 3, 1)).permute(1, 3, 0, 2)
    for k in (odd, turned):
        q = k.clone() if k is odd else turned.clone(memory_format=torch.preserve_format)
        got, gk = run(q, k, q_out=q)
        assert got is q and torch.equal(q, want) and torch.equal(gk.data, wk.data)


# ---------------------------------------------------------------- attention
def check_attention(fm, rng, act, B, S, H, Hkv, D, bs, context, lens, causal=True, scale=None, max_context=None,
                    table=None, n_blocks=None, wide=False, **kw):
    max_context = max(context) if max_context is None else max_context
    per = max(1, -(-max(context) // bs)) if table is None else table.shape[1]
    if table is None:
        n_blocks = B * per + 2
        table = rng.permutation(n_blocks)[: B * per].reshape(B, per)
    (kc, ks), (vc, vs) = (random_pool(rng, n_blocks, bs, Hkv, D) for _ in range(2))
    q = rounded(rng.standard_normal((B, S, H, D)), act)
    n = np.full(B, S) if lens is None else np.asarray(lens)
    for b in range(B):
        q[b, n[b]:] = np.nan  # padding is not read
    if wide:  # the tokens lie in wider rows
        rows = torch.full((B, S, H + 3, D), float("nan"), device="cuda", dtype=DT[act])
        rows[:, :, 1 : H + 1] = dev(q, act)
        qd = rows[:, :, 1 : H + 1]
    else:
        qd = dev(q, act)
    ref, parts = op.attention(np.nan_to_num(q), op.values(kc, ks), op.values(vc, vs), table, context, max_context, n,
                              causal, scale)
    out = torch.full((B, S, H, D), 7.0, device="cuda", dtype=DT[act])
    tables = np.stack([np.full_like(table, -1), table]).astype(np.int32)
    cl = np.stack([np.zeros(B, np.int32), np.asarray(context, np.int32)])
    got = fm.attention_paged(qd, gpu_pool(fm, kc, ks), gpu_pool(fm, vc, vs), 1, dev(tables), dev(cl), max_context,
                             seq_lens=None if lens is None else dev(np.asarray(lens, np.int32)), causal=causal,
                             scale=scale, out=out, **kw)
    assert got is out
    err = np.abs(got.double().cpu().numpy() - ref)
    tol = op.attention_tolerance(ref, parts, D, act)
    bad = ~(err <= tol)
    assert not bad.any(), (f"{bad.sum()} of {bad.size} outside; first {np.argwhere(bad)[0]}, "
                           f"worst {np.nanmax(err / tol):.2f} of the tolerance, nan {np.isnan(err).sum()}")


# contexts at the edges of 16, 32, 64, 128, 256 and 512 positions
EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 511, 512, 513, 700]


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("H,Hkv,D,bs", [(4, 2, 16, 4), (1, 1, 32, 16), (8, 1, 64, 16), (6, 2, 64, 7), (8, 2, 128, 16),
                                        (8, 1, 128, 64), (16, 1, 128, 1), (20, 1, 128, 100), (2, 2, 128, 32)])
def test_decode_edges(fm, act, H, Hkv, D, bs):
    rng = np.random.default_rng(H * D + bs)
    check_attention(fm, rng, act, len(EDGES), 1, H, Hkv, D, bs, EDGES, None)


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("B,S,H,Hkv,D,bs,context,lens,causal", [
    (3, 2, 8, 2, 128, 16, [2, 65, 300], None, True),
    (3, 5, 4, 1, 64, 16, [3, 64, 129], [5, 4, 0], True),   # contexts shorter than the tokens, no tokens at all
    (2, 7, 4, 2, 16, 3, [7, 50], [7, 2], True),
    (4, 33, 4, 1, 128, 16, [33, 64, 31, 500], None, True),
    (2, 64, 2, 2, 64, 32, [64, 200], [64, 63], True),
    (2, 130, 4, 1, 128, 16, [130, 257], [130, 129], True),
    (1, 257, 3, 1, 128, 100, [257], None, True),
    (2, 66, 8, 4, 128, 16, [200, 66], [66, 1], False),
    (2, 40, 4, 2, 64, 5, [10, 90], None, False),
    (3, 17, 4, 2, 32, 16, [17, 40, 300], [17, 16, 3], True),
])
def test_prompts(fm, act, B, S, H, Hkv, D, bs, context, lens, causal):
    rng = np.random.default_rng(B * S + D + bs)
    check_attention(fm, rng, act, B, S, H, Hkv, D, bs, context, lens, causal, wide=S % 2 == 1)


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("S,context", [(1, 9001), (3, 8192), (20, 5000), (100, 3001)])
def test_long_contexts(fm, act, S, context):
    """Few rows: the context is cut over blocks, whose results are joined."""
    rng = np.random.default_rng(S)
    check_attention(fm, rng, act, 2, S, 8, 2, 128, 16, [context, context // 3], None)


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("S,D", [(1, 128), (40, 64), (150, 128)])
def test_bad_pages_short_tables_and_cut_contexts(fm, act, S, D):
    """Entries outside the pool and positions past the table are zeros; a
    context longer than max_context_len is cut, positions counted on."""
    rng = np.random.default_rng(S + D)
    table = rng.permutation(40).reshape(2, 20)
    table[0, 3], table[0, 7], table[1, 0], table[1, 19] = -1, 40, 1 << 30, -(1 << 31)
    check_attention(fm, rng, act, 2, S, 4, 1, D, 16, [320, 330], None, table=table, n_blocks=40)
    check_attention(fm, rng, act, 2, S, 4, 1, D, 16, [320, 300], None, table=table, n_blocks=40, max_context=200)
    check_attention(fm, rng, act, 2, S, 4, 1, D, 16, [320, 300], None, False, 0.5, table=table, n_blocks=40,
                    max_context=200)


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("S,D,bs", [(3, 128, 16), (3, 16, 4), (40, 64, 16), (70, 128, 16), (140, 128, 64)])
def test_what_is_masked_has_no_influence(fm, act, S, D, bs):
    """Keys, values and scales that are NaN, infinite or the type's largest, at
    the positions behind the context, and at positions that only later tokens
    attend: those tokens are NaN, the earlier ones exact."""
    rng = np.random.default_rng(S)
    H, Hkv, B = 4, 2, 2
    context = [S + 21, S]
    per = -(-max(context) // bs) + 1
    n_blocks = B * per
    table = rng.permutation(n_blocks).reshape(B, per)
    (kc, ks), (vc, vs) = (random_pool(rng, n_blocks, bs, Hkv, D) for _ in range(2))
    q = rounded(rng.standard_normal((B, S, H, D)), act)
    for b in range(B):  # behind the context
        for j in range(context[b], per * bs):
            kc[table[b, j // bs], j % bs] = vc[table[b, j // bs], j % bs] = 0x7F
        for lp in range(-(-context[b] // bs), per):
            ks[table[b, lp]], vs[table[b, lp]] = np.nan, np.inf
    pools = lambda: (gpu_pool(fm, kc, ks), gpu_pool(fm, vc, vs))  # noqa: E731
    args = (1, dev(np.stack([table, table]).astype(np.int32)), dev(np.stack([context, context]).astype(np.int32)), per * bs)
    want, parts = op.attention(q, op.values(kc, ks), op.values(vc, vs), table, context, per * bs, [S, S])
    tol = op.attention_tolerance(want, parts, D, act)
    got = fm.attention_paged(dev(q, act), *pools(), *args).double().cpu().numpy()
    assert np.all(np.abs(got - want) <= tol)
    # sequence 0: the value of its last-but-one position NaN (of K/V head 0, dimension 5), K of its last position NaN
    j = context[0] - 2
    vc[table[0, j // bs], j % bs, 0, 5] = 0xFF
    j += 1
    kc[table[0, j // bs], j % bs, 1, 3] = 0x7F
    bad = fm.attention_paged(dev(q, act), *pools(), *args).double().cpu().numpy()
    nan = np.zeros(want.shape, bool)
    nan[0, S - 2 :, :2, 5] = True
    nan[0, S - 1, 2:, :] = True
    assert np.array_equal(np.isnan(bad), nan)
    assert np.all((np.abs(bad - want) <= tol)[~nan])


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("S", [1, 6, 90])
def test_scores_and_weights_of_extreme_size(fm, act, S):
    """One position of all the weight beside thousands of tiny ones, weights
    that all but vanish, and pages whose scales are far apart."""
    rng = np.random.default_rng(S)
    H, Hkv, D, bs, ctx = 4, 1, 64, 16, 1500
    per = -(-ctx // bs)
    (kc, ks), (vc, vs) = (random_pool(rng, per, bs, Hkv, D) for _ in range(2))
    table = np.arange(per)[None]
    q = rounded(rng.standard_normal((1, S, H, D)), act)
    cases = {"far scales": (ks, np.exp2(rng.integers(-30, 30, vs.shape)).astype(np.float32)),
             "sharp": (ks * 40, vs), "flat": (ks * 2.0 ** -20, vs)}
    for name, (k2, v2) in cases.items():
        got = fm.attention_paged(dev(q, act), gpu_pool(fm, kc, k2), gpu_pool(fm, vc, v2), 0,
                                 dev(table[None].astype(np.int32)), dev(np.array([[ctx]], np.int32)), ctx)
        ref, parts = op.attention(q, op.values(kc, k2), op.values(vc, v2), table, [ctx], ctx, [S])
        err = np.abs(got.double().cpu().numpy() - ref)
        assert np.all(err <= op.attention_tolerance(ref, parts, D, act)), name
    # a sink: position 0 takes about half of the weight, the others a few 2^-12 each
    kc[:] = 0
    kc[0, 0, 0, 0] = nm.e4m3fn_encode(np.float32(1.0))
    k2 = np.ones_like(ks)
    q[:] = 0
    q[..., 0] = rounded(np.log(1500.0) * D ** 0.5, act)
    got = fm.attention_paged(dev(q, act), gpu_pool(fm, kc, k2), gpu_pool(fm, vc, vs), 0,
                             dev(table[None].astype(np.int32)), dev(np.array([[ctx]], np.int32)), ctx)
    ref, parts = op.attention(q, op.values(kc, k2), op.values(vc, vs), table, [ctx], ctx, [S])
    assert np.all(np.abs(got.double().cpu().numpy() - ref) <= op.attention_tolerance(ref, parts, D, act))


def test_queries_that_are_not_finite_stay_in_their_rows(fm):
    rng = np.random.default_rng(9)
    for S in (2, 70):
        (kc, ks), (vc, vs) = (random_pool(rng, 8, 16, 1, 128) for _ in range(2))
        q = rounded(rng.standard_normal((1, S, 4, 128)), "bf16")
        args = (gpu_pool(fm, kc, ks), gpu_pool(fm, vc, vs), 0, dev(np.arange(8)[None, None].astype(np.int32)),
                dev(np.array([[120]], np.int32)), 120)
        good = fm.attention_paged(dev(q, "bf16"), *args)
        q[0, 1, 2, 7], q[0, 0, 1, 3] = np.inf, np.nan
        bad = fm.attention_paged(dev(q, "bf16"), *args)
        assert torch.isnan(bad[0, 1, 2]).all() and torch.isnan(bad[0, 0, 1]).all()
        keep = torch.ones(S, 4, dtype=torch.bool, device="cuda")
        keep[1, 2] = keep[0, 1] = False
        assert torch.equal(bad[0][keep], good[0][keep])


# ---------------------------------------------------------------- many rows
def many(B, S, H, context):
    """A max_context_len for which the call is one of many (row, position)
    pairs, whatever the contexts: the kernel is chosen by it."""
    return max(max(context), (16 << 20) // (B * S * H))


@pytest.mark.parametrize("pow2", [True, False])
@pytest.mark.parametrize("B,S,H,Hkv,D,bs,context,lens,causal", [
    (2, 32, 1, 1, 128, 16, [32, 77], None, True),
    (3, 33, 4, 1, 128, 16, [33, 64, 31], [33, 20, 33], True),  # a context shorter than its tokens
    (2, 64, 2, 2, 64, 32, [64, 200], [64, 63], True),
    (2, 130, 4, 1, 128, 16, [130, 257], [130, 129], True),
    (1, 257, 3, 1, 128, 100, [257], None, True),
    (2, 66, 8, 4, 128, 4, [200, 66], [66, 1], False),
    (2, 40, 4, 2, 64, 5, [130, 90], [40, 0], False),
    (1, 70, 20, 2, 64, 1, [515], None, True),
    (3, 48, 6, 2, 128, 64, [48, 640, 1000], [48, 16, 3], True),
])
def test_many_rows(fm, pow2, B, S, H, Hkv, D, bs, context, lens, causal, monkeypatch):
    """Row tiles of 128 at their edges, scales that are powers of two and not."""
    rng = np.random.default_rng(B * S + D + bs)
    if pow2:
        pool = random_pool
        monkeypatch.setattr(__import__(__name__), "random_pool",
                            lambda *a: (lambda c, s: (c, np.exp2(np.round(np.log2(s))).astype(np.float32)))(*pool(*a)))
    check_attention(fm, rng, "bf16", B, S, H, Hkv, D, bs, context, lens, causal, wide=S % 2 == 1,
                    max_context=many(B, S, H, context))


@pytest.mark.parametrize("B,S,H,Hkv,D,context", [(1, 100, 8, 2, 128, 3001), (2, 200, 4, 1, 64, 1500), (9, 256, 32, 4, 128, 300)])
def test_many_rows_long_contexts(fm, B, S, H, Hkv, D, context):
    rng = np.random.default_rng(S)
    contexts = [context - 7 * b for b in range(B)]
    check_attention(fm, rng, "bf16", B, S, H, Hkv, D, 16, contexts, None,
                    max_context=max(context, (13 << 20) // (B * S * H)))


def test_many_rows_bad_pages_and_cut_contexts(fm):
    rng = np.random.default_rng(21)
    S, H = 150, 4
    table = rng.permutation(40).reshape(2, 20)
    table[0, 3], table[0, 7], table[1, 0], table[1, 19] = -1, 40, 1 << 30, -(1 << 31)
    table[1, 8:16] = 77  # a whole tile of zeros
    for causal in (True, False):
        check_attention(fm, rng, "bf16", 2, S, H, 1, 128, 16, [320, 330], None, causal, table=table, n_blocks=40,
                        max_context=16 << 15)
        check_attention(fm, rng, "bf16", 2, S, H, 1, 64, 16, [16 << 15, 300], None, causal, 0.5, table=table,
                        n_blocks=40, max_context=16 << 10)


@pytest.mark.parametrize("S,D,bs", [(40, 64, 16), (70, 128, 16), (140, 128, 64), (33, 128, 3)])
def test_many_rows_what_is_masked_has_no_influence(fm, S, D, bs, monkeypatch):
    real = fm.attention_paged
    monkeypatch.setattr(fm, "attention_paged",
                        lambda q, k, v, layer, bt, cl, n, **kw: real(q, k, v, layer, bt, cl, 16 << 15, **kw))
    test_what_is_masked_has_no_influence(fm, "bf16", S, D, bs)


def test_many_rows_extreme_sizes_and_queries(fm, monkeypatch):
    real = fm.attention_paged
    monkeypatch.setattr(fm, "attention_paged",
                        lambda q, k, v, layer, bt, cl, n, **kw: real(q, k, v, layer, bt, cl, 16 << 16, **kw))
    test_scores_and_weights_of_extreme_size(fm, "bf16", 90)
    test_queries_that_are_not_finite_stay_in_their_rows(fm)


@pytest.mark.parametrize("D,S,B", [(128, 70, 1), (64, 70, 1), (128, 256, 10)])
def test_many_rows_maximum_is_raised_late(fm, D, S, B):
    """Scales that are powers of two, and scores that outgrow all before them
    in the first and the second half of a tile, in later tiles, by little and
    by far; and codes that are NaN, for the rows that attend them."""
    rng = np.random.default_rng(D + S)
    H, Hkv, bs, ctx = 8, 4, 16, 900
    per = -(-ctx // bs)
    table = rng.permutation(B * per).reshape(B, per)
    (kc, ks), (vc, vs) = (random_pool(rng, B * per, bs, Hkv, D) for _ in range(2))
    ks, vs = (np.exp2(np.round(np.log2(s))).astype(np.float32) for s in (ks, vs))
    for b in range(B):
        for position, grow in ((130, 2), (200, 8), (390, 3), (450, 64), (520, 8)):
            kc[table[b, position // bs], position % bs] = 0x70  # 128 in every dimension
            ks[table[b, position // bs]] = 2.0 ** -12 * grow
    q = rounded(rng.uniform(0.1, 1, (B, S, H, D)), "bf16")
    limit = max(ctx, (13 << 20) // (B * S * H))
    lens, dt = np.full((1, B), ctx, np.int32), dev(table[None].astype(np.int32))
    call = lambda: fm.attention_paged(dev(q, "bf16"), gpu_pool(fm, kc, ks), gpu_pool(fm, vc, vs), 0, dt, dev(lens),  # noqa: E731
                                      limit).double().cpu().numpy()
    got = call()
    ref, parts = op.attention(q, op.values(kc, ks), op.values(vc, vs), table, lens[0], limit, np.full(B, S))
    assert np.all(np.abs(got - ref) <= op.attention_tolerance(ref, parts, D, "bf16"))
    for j, h, d in ((140, 1, 5), (200, 0, D - 1), (700, 3, 0)):
        vc[table[0, j // bs], j % bs, h, d] = 0xFF
    hit = np.zeros((S, H, D), bool)  # token s attends positions to ctx - S + s
    for j, h, d in ((140, 1, 5), (200, 0, D - 1), (700, 3, 0)):
        hit[max(0, j - ctx + S) :, h * (H // Hkv) : (h + 1) * (H // Hkv), d] = True
    new = call()
    assert np.isnan(new[0][hit]).all() and np.array_equal(new[0][~hit], got[0][~hit])
    assert np.array_equal(new[1:], got[1:])


@pytest.mark.parametrize("low", [3.0, 8.0, 14.0, 40.0, 400.0])
@pytest.mark.parametrize("D", [64, 128])
def test_many_rows_scores_far_below_zero(fm, D, low):
    """Scales that are powers of two, and scores of about -low: in all
    positions, in the first tile alone, and in all but the last tokens'."""
    rng = np.random.default_rng(int(low))
    B, S, H, Hkv, bs, ctx = 1, 64, 4, 1, 16, 640
    per = ctx // bs
    table = rng.permutation(per)[None]
    (_, ks), (vc, vs) = (random_pool(rng, per, bs, Hkv, D) for _ in range(2))
    vs = np.exp2(np.round(np.log2(vs))).astype(np.float32)
    q = rounded(rng.uniform(0.5, 1.5, (B, S, H, D)), "bf16")
    limit, dt = (13 << 20) // (B * S * H), dev(table[None].astype(np.int32))
    for span in ((0, ctx), (0, 128), (0, 600), (64, 200)):
        want = rng.standard_normal((ctx, Hkv, D)) * 0.5
        want[span[0] : span[1]] -= low * D ** -0.5
        ks[:] = 2.0 ** np.ceil(np.log2((low * D ** -0.5 + 3) / 448))
        kc = np.zeros((per, bs, Hkv, D), np.uint8)
        kc[table[0]] = nm.e4m3fn_encode(want.reshape(per, bs, Hkv, D) / ks[0, 0])
        got = fm.attention_paged(dev(q, "bf16"), gpu_pool(fm, kc, ks), gpu_pool(fm, vc, vs), 0, dt,
                                 dev(np.array([[ctx]], np.int32)), limit).double().cpu().numpy()
        ref, parts = op.attention(q, op.values(kc, ks), op.values(vc, vs), table, [ctx], limit, [S])
        assert np.all(np.abs(got - ref) <= op.attention_tolerance(ref, parts, D, "bf16")), span


def test_pools_of_more_than_32_bits(fm):
    """Pages past 4 GiB of a pool: appended to, and attended by one token, by
    many, and by a decode step."""
    rng = np.random.default_rng(41)
    H, Hkv, D, bs, used = 16, 8, 128, 16, 30
    n_blocks = (1 << 18) + used  # of 16 KiB
    first = n_blocks - used
    pools, small = [], []
    for _ in range(2):
        c, s = random_pool(rng, used, bs, Hkv, D)
        p = fm.QuantizedKVPool(torch.empty((n_blocks, bs, Hkv, D), dtype=torch.uint8, device="cuda"),
                               torch.empty((n_blocks, Hkv), device="cuda"))
        p.data[first:], p.scales[first:] = dev(c), dev(s)
        pools.append(p)
        small.append(fm.QuantizedKVPool(dev(c), dev(s)))
    table = rng.permutation(used).reshape(1, 1, used)
    far, near = dev((table + first).astype(np.int32)), dev(table.astype(np.int32))
    x = dev(rng.standard_normal((1, 60, H + 2 * Hkv, D)), "bf16")
    start, context = dev(np.array([405], np.int32)), dev(np.array([[465]], np.int32))
    blk, _ = block(fm, rng, "bf16", H, Hkv, D)
    step = dev(rng.standard_normal((1, H * D)), "bf16")

    def run(p, bt):
        q, k, v = x.split([H, Hkv, Hkv], dim=2)
        q = fm.kvcache_append(*p, 0, k, v, bt, start, q=q)
        out = [q, fm.attention_paged(q[:, -1:], *p, 0, bt, context, 480), fm.attention_paged(q, *p, 0, bt, context, 480),
               fm.attention_paged(q, *p, 0, bt, context, 1 << 15)]  # the kernel for many rows
        return out + list(blk.paged(step, context[0].long(), *p, 0, bt, context, 465, bt[0, :, 29], context[0] % bs))

    assert all(torch.equal(a, b) for a, b in zip(run(pools, far), run(small, near)))
    for p, s in zip(pools, small):
        assert torch.equal(p.data[first:], s.data) and torch.equal(p.scales[first:], s.scales)


# ---------------------------------------------------------------- a run of both
@pytest.mark.parametrize("act", ["bf16", "f32"])
def test_prompt_then_decode(fm, act):
    """Prompts of unequal length appended and attended, then decode steps, each
    through append and attention, against attention over the pools' values."""
    rng = np.random.default_rng(11)
    B, H, Hkv, D, bs, steps = 3, 4, 2, 64, 16, 4
    lens = np.array([37, 16, 5])
    S = int(lens.max())
    per = -(-(S + steps) // bs)
    table = rng.permutation(B * per).reshape(B, per)
    td = dev(table[None].astype(np.int32))
    kp, vp = (fm.QuantizedKVPool.zeros(B * per, bs, Hkv, D) for _ in range(2))
    at = np.zeros(B, np.int64)
    for step in range(steps + 1):
        n = lens if step == 0 else np.ones(B, np.int64)
        s = int(n.max())
        x = [rounded(rng.standard_normal((B, s, h, D)), act) for h in (H, Hkv, Hkv)]
        q = fm.kvcache_append(kp, vp, 0, dev(x[1], act), dev(x[2], act), td, dev(at.astype(np.int32)),
                              seq_lens=dev(n.astype(np.int32)), q=dev(x[0], act))
        at = at + n
        got = fm.attention_paged(q, kp, vp, 0, td, dev(at[None].astype(np.int32)), int(at.max()),
                                 seq_lens=dev(n.astype(np.int32)))
        values = [op.values(codes_of(p), p.scales.cpu().numpy()) for p in (kp, vp)]
        ref, parts = op.attention(q.double().cpu().numpy(), *values, table, at, int(at.max()), n)
        err = np.abs(got.double().cpu().numpy() - ref)
        assert np.all(err <= op.attention_tolerance(ref, parts, D, act)), step
        # and the values themselves stand within half a code step of what was appended
        for b in range(B):
            for i in range(int(n[b])):
                j = int(at[b] - n[b]) + i
                v = values[1][table[b, j // bs], j % bs]
                scale = vp.scales.cpu().numpy()[table[b, j // bs]][:, None]
                assert np.all(np.abs(v - x[2][b, i]) <= 2.0 ** -4 * np.abs(x[2][b, i]) + 2.0 ** -10 * scale)


# ---------------------------------------------------------------- the decode step
def block(fm, rng, act, H, Hkv, D):
    n, nkv = H * D, Hkv * D
    w = [rounded(rng.standard_normal(s) / np.sqrt(n), act) for s in ((n, n), (n, nkv), (n, nkv), (n, n))]
    b = [(rng.standard_normal(m) * 0.1).astype(np.float32) for m in (n, nkv, nkv, n)]
    blk = fm.AttentionBlockDecode(*(dev(x, act) for x in w), *(dev(x) for x in b), use_bias=True, n_head=H,
                                  n_head_kv=Hkv, n_embd=n, act_dtype=DT[act])
    return blk, [*w, *b, True, H, Hkv, n]


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("H,Hkv,D,bs,context,max_ctx", [
    (4, 2, 16, 4, [10, 3, 0], 12),
    (8, 1, 32, 16, [1, 64, 65], 65),
    (4, 4, 64, 32, [700, 31, 2, 300], 500),  # cut, and positions of zeros
    (8, 2, 128, 16, [5000, 4999, 17], 5000),  # a dozen splits and more
    (16, 8, 64, 16, [40] * 130, 40),  # one split
    (4, 2, 128, 16, [0, 0], 0),
])
def test_decode_step(fm, act, H, Hkv, D, bs, context, max_ctx):
    """The decode step over codes: against the 64-bit one over the codes'
    values, at the tolerances of the step over plain pools (which leave room
    for the bf16 query and weights: 2^-8 of a score and of a weight, averaged
    over the positions); what it appends bit for bit as the append does."""
    rng = np.random.default_rng(H * D + len(context))
    B, per = len(context), -(-(max(context) + 1) // bs)
    n_blocks = B * per
    table = rng.permutation(n_blocks).reshape(B, per)
    slot = table[np.arange(B), np.asarray(context) // bs].copy()
    table[0, (context[0] + 1) // bs // 2] = -5  # rows of zeros
    if B > 3:
        slot[1] = n_blocks  # nowhere
    row = np.asarray(context) % bs
    (kc, ks), (vc, vs) = (random_pool(rng, n_blocks, bs, Hkv, D) for _ in range(2))
    blk, args = block(fm, rng, act, H, Hkv, D)
    x, nw = rounded(rng.standard_normal((B, H * D)), act), rounded(rng.uniform(0.5, 1.5, H * D), act)
    pos = np.asarray(context, np.int64)
    tables, lens = (np.stack([np.full_like(t, 9 * n_blocks), t]).astype(np.int32) for t in (table, np.asarray(context)))
    kf, vf = op.values(kc, ks), op.values(vc, vs)
    good = np.where((tables >= 0) & (tables < n_blocks), tables, n_blocks)
    paging = (1, good, lens, max_ctx, np.full(B, n_blocks), row)
    rtol = 1e-4 if act == "f32" else 2e-2
    for sublayer in (False, True):
        kp, vp = gpu_pool(fm, kc, ks), gpu_pool(fm, vc, vs)
        call = (kp, vp, 1, dev(tables), dev(lens), max_ctx, dev(slot.astype(np.int32)), dev(row.astype(np.int32)))
        if sublayer:
            out, k_new, v_new = blk.paged_sublayer(dev(x, act), dev(nw, act), 1e-5, dev(pos), *call)
            ref = oa.attention_sublayer_decode_paged(x, nw, 1e-5, pos, kf, vf, *paging, *args)
        else:
            out, k_new, v_new = blk.paged(dev(x, act), dev(pos), *call)
            ref = oa.attention_decode_paged(x, pos, kf, vf, *paging, *args)
        for got, want in zip((out, k_new, v_new), ref):
            assert_close_rms(got.float().cpu().numpy(), want, rtol)
        codes = [a.copy() for a in (kc, ks, vc, vs)]
        for (c, s), new in ((codes[:2], k_new), (codes[2:], v_new)):
            op.append(c, s, new[:, None].double().cpu().numpy(), slot[:, None], row, np.ones(B))
        for got, want in zip((codes_of(kp), kp.scales.cpu().numpy(), codes_of(vp), vp.scales.cpu().numpy()), codes):
            assert np.array_equal(got, want)


def test_decode_step_is_append_and_attention_of_codes(fm):
    """Where the new token's key and value are codes exactly, the step over a
    full context attends what append and attention do: weights of zero but for
    the query's and small integers for the values."""
    H, Hkv, D, bs, ctx = 2, 1, 64, 16, 37
    n = H * D
    zero, eye = torch.zeros(n, n, device="cuda"), torch.eye(n, device="cuda")
    blk = fm.AttentionBlockDecode(zero, zero[:, :D].contiguous(), eye[:, :D].contiguous(), eye, n_head=H, n_head_kv=Hkv, n_embd=n,
                                  act_dtype=torch.float32)
    pools = [[fm.QuantizedKVPool.zeros(4, bs, Hkv, D) for _ in range(2)] for _ in range(2)]
    table = dev(np.array([[[2, 0, 3]]], np.int32))
    x = torch.randint(-8, 9, (ctx + 1, n), device="cuda").float()
    kv = torch.zeros(1, ctx, Hkv, D, device="cuda"), x[:ctx, :D].reshape(1, ctx, Hkv, D).contiguous()
    for p in pools:
        fm.kvcache_append(*p, 0, *kv, table, dev(np.zeros(1, np.int32)))
    out, k_new, v_new = blk.paged(x[ctx:], dev(np.array([ctx])), *pools[0], 0, table, dev(np.array([[ctx]], np.int32)), ctx,
                                  dev(np.array([3], np.int32)), dev(np.array([5], np.int32)))
    q = fm.kvcache_append(*pools[1], 0, k_new[:, None], v_new[:, None], table, dev(np.array([ctx], np.int32)),
                          q=torch.zeros(1, 1, H, D, device="cuda"), rope=False)
    ref = fm.attention_paged(q, *pools[1], 0, table, dev(np.array([[ctx + 1]], np.int32)), ctx + 1)
    assert all(torch.equal(a.data.view(torch.uint8), b.data.view(torch.uint8)) and torch.equal(a.scales, b.scales)
               for a, b in zip(*pools))
    # all scores are 0: the mean of integers, two roundings and a product each
    mean = x[:, :D].double().mean(0).repeat(H)
    for got in (out, ref.reshape(1, n)):
        assert (got.double() - mean).abs().max() <= 8 * 2.0 ** -22


def test_decode_step_captured(fm):
    rng = np.random.default_rng(31)
    B, H, Hkv, D, bs, ctx = 3, 8, 2, 128, 16, 900
    blk, _ = block(fm, rng, "bf16", H, Hkv, D)
    per = ctx // bs + 1
    table = dev(rng.permutation(B * per).reshape(1, B, per).astype(np.int32))
    cl = dev(np.array([[ctx, 500, 16]], np.int32))
    slot = table[0].gather(1, (cl[0] // bs).long()[:, None])[:, 0].contiguous()
    start = [random_pool(rng, B * per, bs, Hkv, D) for _ in range(2)]
    x = torch.randn(B, H * D, device="cuda").bfloat16()
    pools = [gpu_pool(fm, *s) for s in start]
    call = lambda p, x: blk.paged(x, cl[0].long(), *p, 0, table, cl, ctx, slot, cl[0] % bs)[0]  # noqa: E731
    call(pools, x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call(pools, x)
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        mine = [gpu_pool(fm, *s) for s in start]
        for p, m in zip(pools, mine):
            p.data.copy_(m.data)
            p.scales.copy_(m.scales)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(mine, x))
        assert all(torch.equal(p.data.view(torch.uint8), m.data.view(torch.uint8)) and torch.equal(p.scales, m.scales)
                   for p, m in zip(pools, mine))


def test_decode_step_arguments(fm):
    blk, _ = block(fm, np.random.default_rng(0), "f32", 4, 2, 16)
    kp, vp = (fm.QuantizedKVPool.zeros(4, 4, 2, 16) for _ in range(2))
    x, pos, bt = torch.zeros(1, 64, device="cuda"), dev(np.zeros(1, np.int64)), dev(np.zeros((1, 1, 1), np.int32))
    one = dev(np.zeros(1, np.int32))
    for exc, k, v in [(ValueError, kp, vp.dequantize()), (ValueError, kp.dequantize(), vp), (ValueError, kp, kp),
                      (ValueError, *(fm.QuantizedKVPool.zeros(4, 4, 1, 16) for _ in range(2))),
                      (TypeError, fm.QuantizedKVPool(kp.data.float(), kp.scales), vp),
                      (ValueError, fm.QuantizedKVPool(kp.data, kp.scales[:2]), vp)]:
        with pytest.raises(exc):
            blk.paged(x, pos, k, v, 0, bt, bt[0], 4, one, one)
    with pytest.raises(ValueError):
        blk.paged(x, pos, kp, vp, 0, bt, bt[0], 2 ** 31 - 4096, one, one)
    out, k_new, _ = blk.paged(x[:0], pos[:0], kp, vp, 0, bt[:, :0], bt[0, :0].view(1, 0), 4, one[:0], one[:0])
    assert out.shape == (0, 64) and k_new.shape == (0, 2, 16)


def test_captured_and_replayed(fm):
    """Append and attention in a graph, replayed with new inputs and eager work
    in between, bit for bit the eager calls; two graphs share no workspace."""
    rng = np.random.default_rng(12)
    B, H, Hkv, D, bs, ctx = 4, 8, 2, 128, 16, 1400
    per = -(-ctx // bs)
    table = dev(rng.permutation(B * per).reshape(1, B, per).astype(np.int32))
    fresh = lambda: [gpu_pool(fm, *random_pool(np.random.default_rng(1), B * per, bs, Hkv, D)) for _ in range(2)]  # noqa: E731
    cl = dev(np.array([[ctx, 900, 65, 1]], np.int32))
    start = (cl[0] - 1).contiguous()
    x = torch.randn(B, 1, H + 2 * Hkv, D, device="cuda").bfloat16()

    def step(pools, x):
        q, k, v = x.split([H, Hkv, Hkv], dim=2)
        q = fm.kvcache_append(*pools, 0, k, v, table, start, q=q)
        return fm.attention_paged(q, *pools, 0, table, cl, ctx)

    step(fresh(), x)
    graphs = []
    for _ in range(2):
        pools, xs = fresh(), x.clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(pools, xs)
        graphs.append((g, pools, xs, out))
    for i in range(3):
        new = [torch.randn_like(x) for _ in graphs]
        for (g, pools, xs, out), n in zip(graphs, new):
            for p, f in zip(pools, fresh()):
                p.data.copy_(f.data)
                p.scales.copy_(f.scales)
            xs.copy_(n)
        torch.cuda.synchronize()
        side = [torch.cuda.Stream() for _ in graphs]
        for (g, *_), s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (g, pools, xs, out), n in zip(graphs, new):
            mine = fresh()
            assert torch.equal(out, step(mine, n)), i
            assert all(torch.equal(p.data.view(torch.uint8), m.data.view(torch.uint8)) and torch.equal(p.scales, m.scales)
                       for p, m in zip(pools, mine))


def test_arguments(fm):
    kp, vp = (fm.QuantizedKVPool.zeros(4, 4, 2, 16) for _ in range(2))
    x = torch.zeros(1, 2, 2, 16, device="cuda")
    q = torch.zeros(1, 2, 4, 16, device="cuda")
    bt, st, cl = dev(np.zeros((1, 1, 1), np.int32)), dev(np.zeros(1, np.int32)), dev(np.full((1, 1), 2, np.int32))
    assert kp.shape == (4, 4, 2, 16) and not kp.dequantize().any()
    ok = fm.kvcache_append(kp, vp, 0, x, x, bt, st)
    assert ok is None
    for exc, call in [
        (TypeError, lambda: fm.kvcache_append(kp, vp, 0, x.half(), x, bt, st)),
        (ValueError, lambda: fm.kvcache_append(kp, vp, 0, x.bfloat16(), x, bt, st)),
        (ValueError, lambda: fm.kvcache_append(kp, kp, 0, x, x, bt, st)),
        (ValueError, lambda: fm.kvcache_append(kp, vp.dequantize(), 0, x, x, bt, st)),
        (TypeError, lambda: fm.kvcache_append(kp.dequantize().bfloat16(), vp.dequantize().bfloat16(), 0, x, x, bt, st)),
        (TypeError, lambda: fm.kvcache_append(kp.data.cpu(), vp, 0, x, x, bt, st)),
        (TypeError, lambda: fm.kvcache_append(kp.data.transpose(0, 1), vp, 0, x, x, bt, st)),
        (TypeError, lambda: fm.kvcache_append(fm.QuantizedKVPool(kp.data, kp.scales.half()), vp, 0, x, x, bt, st)),
        (ValueError, lambda: fm.kvcache_append(fm.QuantizedKVPool(kp.data, kp.scales[:3]), vp, 0, x, x, bt, st)),
        (ValueError, lambda: fm.kvcache_append(kp, vp, 0, x[..., :8], x, bt, st)),
        (ValueError, lambda: fm.kvcache_append(kp, vp, 0, x[:, :1], x, bt, st)),
        (ValueError, lambda: fm.kvcache_append(kp, vp, 1, x, x, bt, st)),
        (ValueError, lambda: fm.kvcache_append(kp, vp, 0, x, x, bt[0], st)),
        (TypeError, lambda: fm.kvcache_append(kp, vp, 0, x, x, bt.float(), st)),
        (ValueError, lambda: fm.kvcache_append(kp, vp, 0, x, x, bt, dev(np.zeros(2, np.int32)))),
        (ValueError, lambda: fm.kvcache_append(kp, vp, 0, x, x, bt, st, seq_lens=bt)),
        (ValueError, lambda: fm.kvcache_append(kp, vp, 0, x, x, bt, st, q=q[:, :1])),
        (ValueError, lambda: fm.kvcache_append(kp, vp, 0, x, x, bt, st, q=q.bfloat16())),
        (ValueError, lambda: fm.kvcache_append(kp, vp, 0, x, x, bt, st, q_out=q)),
        (ValueError, lambda: fm.kvcache_append(kp, vp, 0, x, x, bt, st, q=q, q_out=q[:, :, :2])),
        (ValueError, lambda: fm.kvcache_append(kp, vp, 0, x, x, bt, st, rope_freq_base=0.0)),
        (TypeError, lambda: fm.attention_paged(q, kp.dequantize(), vp, 0, bt, cl, 2)),
        (TypeError, lambda: fm.attention_paged(q.half(), kp, vp, 0, bt, cl, 2)),
        (ValueError, lambda: fm.attention_paged(q[:, :, :3], kp, vp, 0, bt, cl, 2)),
        (ValueError, lambda: fm.attention_paged(q[0], kp, vp, 0, bt, cl, 2)),
        (ValueError, lambda: fm.attention_paged(q, kp, vp, 0, bt, st, 2)),
        (ValueError, lambda: fm.attention_paged(q, kp, vp, 0, bt, cl, -1)),
        (ValueError, lambda: fm.attention_paged(q, kp, vp, 0, bt, cl, 2, scale=0.0)),
        (ValueError, lambda: fm.attention_paged(q, kp, vp, 0, bt, cl, 2, out=q[:, :1])),
        (ValueError, lambda: fm.attention_paged(q, kp, vp, 0, bt, cl, 2, out=torch.zeros_like(q).transpose(0, 1))),
    ]:
        with pytest.raises(exc):
            call()
    empty = fm.attention_paged(q[:, :0], kp, vp, 0, bt, cl, 2)
    assert empty.shape == (1, 0, 4, 16)
    assert fm.attention_paged(q, kp, vp, 0, bt, cl, 0).abs().max() == 0
