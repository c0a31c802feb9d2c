"""The paged cache of e4m3 codes and the attention over it, in 64 bits (test
infrastructure only).  No counterpart in the reference, whose cache holds fp32
(components/kvcache/kvcache.mlir) and whose RoPE this follows
(components/position/rope.mlir:38-104).
"""

from __future__ import annotations

import numpy as np

from .numerics import e4m3fn_decode, e4m3fn_encode


def rope(x, positions, freq_base=10000.0, freq_scale=1.0):
    """Pairs (2i, 2i + 1) of x [n, heads, D] turned by position * freq_scale / freq_base^(2i / D)."""
    x = np.asarray(x, np.float64)
    D = x.shape[-1]
    angle = np.asarray(positions, np.float64)[:, None] * freq_scale / freq_base ** (np.arange(0, D, 2) / D)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    out = np.empty_like(x)
    out[..., 0::2] = x[..., 0::2] * c - x[..., 1::2] * s
    out[..., 1::2] = x[..., 0::2] * s + x[..., 1::2] * c
    return out


def pow2_scale(a):
    """Least power of two s with a <= 448 s, from 2^-126 on."""
    s = 2.0 ** -126
    while a > 448.0 * s and s < 2.0 ** 126:
        s *= 2.0
    return s


def append(pool, scales, x, table, start, seq_lens):
    """New rows x [batch, seq_len, n_head_kv, D] (64 bits) into a pool's pages,
    in place.  pool: float64 values and scales None, or uint8 codes and
    float32 scales [n_blocks, n_head_kv].  Returns {(page, row)} written."""
    n_blocks, bs = pool.shape[:2]
    jobs = {}  # page -> its last append
    for b in range(x.shape[0]):
        for s in range(max(0, min(int(seq_lens[b]), x.shape[1]))):
            lp, r = divmod(int(start[b]) + s, bs)
            if 0 <= lp < table.shape[1] and 0 <= table[b, lp] < n_blocks:
                job = jobs.get(int(table[b, lp]))
                if job is None or job[:2] != (b, lp):
                    job = jobs[int(table[b, lp])] = (b, lp, r, [])
                job[3].append(x[b, s])
    done = set()
    for page, (_, _, r0, rows) in jobs.items():
        new = np.stack(rows)
        done.update((page, r0 + i) for i in range(len(rows)))
        if scales is None:
            pool[page, r0 : r0 + len(rows)] = new
            continue
        for h in range(new.shape[1]):
            a = np.abs(new[:, h])
            s = pow2_scale(np.max(a[np.isfinite(a)], initial=0.0))
            if r0 > 0:
                old = float(scales[page, h])
                if s > old:
                    pool[page, :r0, h] = e4m3fn_encode(e4m3fn_decode(pool[page, :r0, h]) * np.float32(old / s))
                else:
                    s = old
            y = new[:, h] / s
            pool[page, r0 : r0 + len(rows), h] = np.where(np.isfinite(y), e4m3fn_encode(np.nan_to_num(y)), 0x7F)
            scales[page, h] = s
    return done


def values(codes, scales):
    """decode(codes) * scales, 64 bits; a zero page behind the pool's last."""
    v = e4m3fn_decode(codes).astype(np.float64) * scales.astype(np.float64)[:, None, :, None]
    return np.concatenate([v, np.zeros((1,) + v.shape[1:])])


def attention(q, k, v, table, context_lens, max_context_len, seq_lens, causal=True, scale=None):
    """(out [batch, seq_len, n_head, D], parts) in 64 bits; k, v: pools of
    values with a zero page behind the last.  parts: per output, (sum of
    softmax |V|, sum |V| / n, largest sum |q K| of a score, positions), for tolerances."""
    q = np.asarray(q, np.float64)
    B, S, H, D = q.shape
    n_blocks, bs, Hkv = k.shape[0] - 1, k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = np.zeros_like(q)
    mag, prod, count = np.zeros_like(q), np.zeros((B, S, H, 1)), np.zeros((B, S, H, 1))
    for b in range(B):
        n = max(0, min(int(seq_lens[b]), S))
        ctx = max(0, int(context_lens[b]))
        c = min(ctx, max_context_len)
        j = np.arange(c)
        lp = j // bs
        page = np.where(lp < table.shape[1], table[b, np.minimum(lp, table.shape[1] - 1)], -1)
        page = np.where((page >= 0) & (page < n_blocks), page, n_blocks)
        kb, vb = k[page, j % bs], v[page, j % bs]  # [c, Hkv, D]
        for s in range(n):
            e = min(c, ctx - n + s + 1) if causal else c
            if e <= 0:
                continue
            for g in range(Hkv):
                h = slice(g * (H // Hkv), (g + 1) * (H // Hkv))
                sc = q[b, s, h] @ kb[:e, g].T * scale
                w = np.exp(sc - sc.max(axis=1, keepdims=True))
                w /= w.sum(axis=1, keepdims=True)
                out[b, s, h] = w @ vb[:e, g]
                mag[b, s, h] = w @ np.abs(vb[:e, g])
                prod[b, s, h, 0] = (np.abs(q[b, s, h]) @ np.abs(kb[:e, g]).T).max(axis=1) * scale
                count[b, s, h] = e
    return out, (mag, prod, count)


def attention_tolerance(out, parts, D, act):
    """How far a kernel's output may be from ``out``.

    u is half a step of the arithmetic: 2^-24.  A score is a sum of D
    products, exact or rounded once, then scaled (three factors): off by at
    most (D + 4) u of the sum of the products' magnitudes.  bf16 queries may
    be carried as two e4m3 terms under a power of two: exact from 2^-2 of
    the scale up, within 2^-10 of it below, which is 2^-17 of the row's
    largest value; against the products' magnitudes, D 2^-17 at most.  exp adds
    2^-22.  A weight off by a factor (1 + e) moves the output by at most 2 e
    times the softmax-weighted |V|; its own sum is n terms.  bf16: the
    unnormalised weights are rounded to bf16, in the numerator alone (2^-8, so
    2^-9 in e).  The output is rounded once."""
    mag, prod, count = parts
    u = 2.0 ** -24
    half = {"f32": u, "bf16": 2.0 ** -8}[act]
    e = (D + 4) * u * prod + 2.0 ** -22 + (count + 8) * u
    if act == "bf16":
        e = e + D * 2.0 ** -17 * prod / D ** 0.5 + 2.0 ** -9
    return 2 * e * mag + half * np.abs(out) + 1e-30
