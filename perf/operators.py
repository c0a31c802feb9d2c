"""The paged K/V cache's append and the attention that reads a cache held in 8 bits.

Each case is one call on data that is already on the GPU: ``kvcache_append``
(the new tokens' keys rotated and written, with the values, into their pages;
the queries rotated on the way) and ``attention_paged`` (one or more new tokens
of each sequence over e4m3 pages with a scale for each page and head).

``listed()`` holds the named cases, ``draw(rng)`` one more of the same ranges.
``prepare`` makes the inputs, ``run`` is one call: the plain form in elementary
torch operations, or the package's entry point where ``own`` is true; ``exact``
is the same result in 64 bits.
"""

from __future__ import annotations

import functools
import importlib
import math

import torch

own = False

# name: query heads, K/V heads, head size
HEADS = {"toy": (4, 2, 16), "small": (4, 2, 128), "mqa": (8, 1, 64), "mixtral": (32, 8, 128)}

TORCH = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
BYTES = {"bf16": 2, "f32": 4, "e4m3": 1}
FREQ_BASE = 10000.0
LAYER, LAYERS = 1, 2  # the tables hold two layers' pages; the call is the second's


def _append(name, heads, batch, seq, start, ragged, block_size, act="bf16", pool="e4m3"):
    return {"name": name, "kind": "append", "heads": heads, "batch": batch, "seq": seq, "start": start,
            "ragged": ragged, "block_size": block_size, "act": act, "pool": pool}


def _attention(name, heads, batch, seq, context, ragged, block_size, act="bf16", causal=True):
    return {"name": name, "kind": "attention", "heads": heads, "batch": batch, "seq": seq, "context": context,
            "ragged": ragged, "block_size": block_size, "act": act, "causal": causal}


def listed():
    return [
        # The toy model's decode step in its own type: two tokens, nothing but latency.
        _append("append-toy-f32-2", "toy", 2, 1, 10, False, 4, act="f32"),
        # A wide decode batch: one token of each of 61 sequences, most of them inside a page.
        _append("append-decode-61", "mixtral", 61, 1, 1000, True, 16),
        # Chunks of prompts of unequal length behind cached ones, into a pool of the activations' type.
        _append("append-bf16-pool-4x509", "mixtral", 4, 509, 300, True, 16, pool="bf16"),
        # A batch of whole prompts into empty pages.
        _append("append-prompts-4x2048", "mixtral", 4, 2048, 0, False, 32),
        # The toy model's decode step: a handful of positions.
        _attention("attention-toy-f32-2", "toy", 2, 1, 10, False, 4, act="f32"),
        # One user's decode step behind a long context.
        _attention("attention-decode-1x8192", "mixtral", 1, 1, 8192, False, 16),
        # A decode batch of equal sequences.
        _attention("attention-decode-16x4096", "mixtral", 16, 1, 4096, False, 16),
        # A wide decode batch of shorter sequences of unequal length.
        _attention("attention-decode-61x1000", "mixtral", 61, 1, 1000, True, 16),
        # Prompts in the reference's type, of lengths that divide nothing.
        _attention("attention-f32-3x701", "mixtral", 3, 701, 701, True, 16, act="f32"),
        # A batch of prompts of unequal length.
        _attention("attention-prompts-4x1021", "mixtral", 4, 1021, 1021, True, 16),
        # A chunk of a long prompt: few rows, long context.
        _attention("attention-chunk-256-16384", "mixtral", 1, 256, 16384, False, 16),
        # A whole long prompt: the matrix cores' work.
        _attention("attention-prompt-1x8192", "mixtral", 1, 8192, 8192, False, 32),
    ]


def _log_int(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    heads = rng.choice(["mixtral", "mixtral", "small", "mqa", "toy"])
    act = rng.choice(["bf16", "bf16", "f32"])
    block_size = rng.choice([4, 16, 16, 32, 64])
    ragged = rng.random() < 0.6
    if rng.random() < 0.4:
        batch = _log_int(rng, 1, 128)
        seq = 1 if rng.random() < 0.4 else _log_int(rng, 1, max(1, (8192 if act == "bf16" else 4096) // batch))
        c = _append("", heads, batch, seq, _log_int(rng, 1, max(1, min(4096, 65536 // batch))), ragged, block_size,
                    act=act, pool=rng.choice(["e4m3", "e4m3", act]))
    elif rng.random() < 0.5:  # decode, or a few speculated tokens
        batch = _log_int(rng, 1, 128)
        seq = rng.choice([1, 1, 1, 2, 3, 5])
        c = _attention("", heads, batch, seq, _log_int(rng, seq, max(8, min(32768, 65536 // batch))), ragged,
                       block_size, act=act, causal=rng.random() < 0.9)
    else:  # prompts and chunks of prompts
        batch = _log_int(rng, 1, 8)
        seq = _log_int(rng, 6, (4096 if act == "bf16" else 1024) // batch)
        context = seq if rng.random() < 0.5 else _log_int(rng, seq, max(seq, min(16384, 4096 * 4096 // (batch * seq))))
        c = _attention("", heads, batch, seq, context, ragged, block_size, act=act, causal=rng.random() < 0.8)
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs
def _pow2_scale(amax):
    """Least power of two s with amax / s <= 448, the largest e4m3 value (2^-126 for 0)."""
    m, e = torch.frexp(amax / 448.0)
    e = torch.where(m > 0.5, e, e - 1).clamp(-126, 126)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), torch.full_like(amax, 2.0 ** -126))


def _paged(g, pages, block_size, n_kv, dim, dtype):
    """A pool [pages, block_size, n_kv, dim] of normal values, whose size differs by head and a little by page."""
    x = torch.empty((pages, block_size, n_kv, dim), device="cuda").normal_(generator=g)
    x *= torch.empty((pages, 1, n_kv, 1), device="cuda").uniform_(0.6, 1.6, generator=g)
    if dtype != torch.float8_e4m3fn:
        return x.to(dtype), None
    scale = _pow2_scale(x.abs().amax(dim=(1, 3)))
    return (x / scale[:, None, :, None]).to(dtype), scale


def prepare(case, seed):
    H, Hkv, D = HEADS[case["heads"]]
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dt, B, S, bs = TORCH[case["act"]], case["batch"], case["seq"], case["block_size"]

    def lengths(lo, hi):
        n = torch.full((B,), hi, dtype=torch.int32, device="cuda")
        if case["ragged"]:
            n = torch.randint(lo, hi + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
            n[0] = hi
        return n

    seq_lens = lengths(max(1, S // 2), S)
    if case["kind"] == "append":
        start = lengths(case["start"] // 2, case["start"])
        reach = case["start"] + S
        pool = TORCH[case["pool"]]
    else:
        # a context holds its new tokens
        context = torch.maximum(lengths(max(1, case["context"] // 2), case["context"]), seq_lens)
        reach = case["context"]
        pool = torch.float8_e4m3fn
    per = -(-reach // bs)
    tables = torch.randperm(LAYERS * B * per, generator=g, device="cuda").to(torch.int32).view(LAYERS, B, per)
    k, k_scales = _paged(g, LAYERS * B * per, bs, Hkv, D, pool)
    v, v_scales = _paged(g, LAYERS * B * per, bs, Hkv, D, pool)
    s = {"kind": case["kind"], "k": k, "v": v, "k_scales": k_scales, "v_scales": v_scales, "tables": tables,
         "seq_lens": seq_lens if case["ragged"] and S > 1 else None}
    if case["kind"] == "append":
        # one row per token holds q | k | v, as a fused projection leaves them
        rows = torch.empty((B, S, (H + 2 * Hkv) * D), device="cuda").normal_(generator=g).to(dt)
        q, kn, vn = rows.split([H * D, Hkv * D, Hkv * D], dim=2)
        s.update(q=q.unflatten(2, (H, D)), k_new=kn.unflatten(2, (Hkv, D)), v_new=vn.unflatten(2, (Hkv, D)),
                 start=start)
    else:
        s.update(q=torch.empty((B, S, H, D), device="cuda").normal_(generator=g).to(dt),
                 context_lens=context.expand(LAYERS, B).contiguous(), max_context=case["context"],
                 causal=case["causal"])
    return s


# ---------------------------------------------------------------- the calls
@functools.lru_cache(maxsize=None)
def _package():
    return importlib.import_module("frank-models_amd")


def _own_append(s):
    fm = _package()
    k, v = s["k"], s["v"]
    if s["k_scales"] is not None:
        k, v = fm.QuantizedKVPool(k, s["k_scales"]), fm.QuantizedKVPool(v, s["v_scales"])
    q = fm.kvcache_append(k, v, LAYER, s["k_new"], s["v_new"], s["tables"], s["start"], seq_lens=s["seq_lens"],
                          q=s["q"], rope_freq_base=FREQ_BASE)
    return {"q": q, "k": s["k"], "v": s["v"], "k_scales": s["k_scales"], "v_scales": s["v_scales"]}


def _own_attention(s):
    fm = _package()
    return fm.attention_paged(s["q"], fm.QuantizedKVPool(s["k"], s["k_scales"]),
                              fm.QuantizedKVPool(s["v"], s["v_scales"]), LAYER, s["tables"], s["context_lens"],
                              s["max_context"], seq_lens=s["seq_lens"], causal=s["causal"])


def _rotate(x, positions):
    """Pairs (2i, 2i + 1) of x [B, S, heads, D] turned by position / base^(2i / D): angles in 64 bits, the rest in 32."""
    D = x.shape[-1]
    freq = FREQ_BASE ** (-torch.arange(0, D, 2, dtype=torch.float64, device=x.device) / D)
    angle = positions.double()[:, :, None, None] * freq
    c, n = angle.cos().float(), angle.sin().float()
    x0, x1 = x[..., 0::2].float(), x[..., 1::2].float()
    return torch.stack([x0 * c - x1 * n, x0 * n + x1 * c], dim=-1).flatten(-2)


def _write(pool, scales, x, table, start, lens):
    """The new rows x [B, S, n_kv, D] (32 bits) into their pages, in place."""
    B, S, n_kv, D = x.shape
    bs = pool.shape[1]
    # a padding token stands for its sequence's last one, which is then written more than once
    s = torch.minimum(torch.arange(S, device=x.device)[None], lens[:, None].long() - 1)
    x = x.gather(1, s[:, :, None, None].expand_as(x))
    t = start[:, None].long() + s
    page = table.long().gather(1, t // bs)
    row = (page * bs + t % bs).flatten()
    if scales is None:
        pool.view(-1, n_kv, D)[row] = x.flatten(0, 1).to(pool.dtype)
        return
    codes = pool.view(torch.uint8)
    # the page that each sequence stops in keeps its scale or grows it, with its earlier rows; later pages begin anew
    first, old = page[:, 0], (start % bs)[:, None].long()
    kept = torch.where(old > 0, scales[first], torch.zeros_like(scales[first]))
    largest = torch.zeros_like(scales).index_reduce_(0, page.flatten(), x.abs().amax(dim=3).flatten(0, 1), "amax")
    grown = torch.maximum(_pow2_scale(largest[first]), kept)
    before = codes[first].view(pool.dtype).float() * (scales[first] / grown)[:, None, :, None]
    live = torch.arange(bs, device=x.device)[None, :, None, None] < old[:, :, None, None]
    codes[first] = torch.where(live, before.to(pool.dtype).view(torch.uint8), codes[first])
    scales[page.flatten()] = _pow2_scale(largest)[page.flatten()]
    scales[first] = grown
    codes.view(-1, n_kv, D)[row] = (x.flatten(0, 1) / scales[page.flatten()][:, :, None]).to(pool.dtype).view(torch.uint8)


def _plain_append(s):
    B, S = s["q"].shape[:2]
    positions = s["start"][:, None] + torch.arange(S, device=s["q"].device)[None]
    lens = s["seq_lens"] if s["seq_lens"] is not None else torch.full_like(s["start"], S)
    q = _rotate(s["q"], positions).to(s["q"].dtype)
    table = s["tables"][LAYER]
    _write(s["k"], s["k_scales"], _rotate(s["k_new"], positions), table, s["start"], lens)
    _write(s["v"], s["v_scales"], s["v_new"].float(), table, s["start"], lens)
    return {"q": q, "k": s["k"], "v": s["v"], "k_scales": s["k_scales"], "v_scales": s["v_scales"]}


def _gathered(pool, scales, table, n):
    """The first n positions' rows of each sequence, [B, n_kv, n, D] in 32 bits."""
    B, pages = table.shape
    t = table.long()
    x = pool.view(torch.uint8)[t].view(pool.dtype).float() * scales[t][:, :, None, :, None]
    return x.flatten(1, 2)[:, :n].transpose(1, 2).contiguous()


def _plain_attention(s):
    q, table, n = s["q"], s["tables"][LAYER], s["max_context"]
    B, S, H, D = q.shape
    k, v = _gathered(s["k"], s["k_scales"], table, n), _gathered(s["v"], s["v_scales"], table, n)
    n_kv = k.shape[1]
    context = s["context_lens"][LAYER].long()
    lens = s["seq_lens"].long() if s["seq_lens"] is not None else torch.full_like(context, S)
    rows = q.float().unflatten(2, (n_kv, H // n_kv)).permute(0, 2, 3, 1, 4).reshape(B, n_kv, H // n_kv * S, D)
    score = (rows @ k.transpose(2, 3).contiguous()).mul_(D ** -0.5).unflatten(2, (H // n_kv, S))
    i, j = torch.arange(S, device=q.device), torch.arange(n, device=q.device)
    position = (context - lens)[:, None] + i[None]
    attends = (j < context[:, None, None]) & (i[None, :, None] < lens[:, None, None])
    if s["causal"]:
        attends &= j <= position[:, :, None]
    score.masked_fill_(~attends[:, None, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    weight = score.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = weight.sum(dim=-1, keepdim=True)
    out = (weight.flatten(2, 3) @ v).unflatten(2, (H // n_kv, S)) / torch.where(total > 0, total, torch.ones_like(total))
    return out.permute(0, 3, 1, 2, 4).reshape(B, S, H, D).to(q.dtype)


def run(state):
    if own:
        return _own_append(state) if state["kind"] == "append" else _own_attention(state)
    return _plain_append(state) if state["kind"] == "append" else _plain_attention(state)


# ---------------------------------------------------------------- what a call cannot do without
def work(case):
    H, Hkv, D = HEADS[case["heads"]]
    B, S, a = case["batch"], case["seq"], BYTES[case["act"]]
    mean = lambda n: 0.75 * n if case["ragged"] and n > 1 else float(n)  # noqa: E731  (expected length)
    if case["kind"] == "append":
        tokens = B * mean(S)
        return {"bytes": B * S * 2 * H * D * a + tokens * 2 * Hkv * D * (a + BYTES[case["pool"]]),
                "flops": 3.0 * (B * S * H + tokens * Hkv) * D}
    n, c = mean(S), max(mean(S), mean(case["context"]))
    pairs = n * (c - (n - 1) / 2) if case["causal"] else n * c
    return {"bytes": B * (2 * c * Hkv * (D + 4 / case["block_size"]) + 2 * n * H * D * a),
            "flops": 4.0 * B * pairs * H * D}


# ---------------------------------------------------------------- 64-bit results
def _rope64(x, t):
    """x [n, heads, D] at positions t [n], in 64 bits."""
    D = x.shape[-1]
    z = torch.view_as_complex(x.double().unflatten(-1, (D // 2, 2)).contiguous())
    angle = t.double()[:, None] * FREQ_BASE ** (-2.0 * torch.arange(D // 2, dtype=torch.float64, device=x.device) / D)
    return torch.view_as_real(z * torch.polar(torch.ones_like(angle), angle)[:, None]).flatten(-2)


def _e4m3(x):
    """The e4m3 value next to x (ties to the even one), |x| <= 448, as a 64-bit number."""
    e = torch.frexp(x).exponent.double() - 1
    step = torch.exp2(e.clamp_min(-6) - 3)
    return torch.round(x / step) * step


def _scale64(a):
    e = torch.ceil(torch.log2(a / 448.0))
    e = torch.where(torch.exp2(e - 1) * 448.0 >= a, e - 1, e)
    e = torch.where(torch.exp2(e) * 448.0 < a, e + 1, e)
    return torch.where(a > 0, torch.exp2(e.clamp(-126, 126)), torch.full_like(a, 2.0 ** -126))


def _exact_append(case, seed):
    s = prepare(case, seed)
    B, S = s["q"].shape[:2]
    bs, e4m3 = case["block_size"], s["k_scales"] is not None
    start = s["start"].tolist()
    lens = [S] * B if s["seq_lens"] is None else s["seq_lens"].tolist()
    out = {"q": torch.stack([_rope64(s["q"][b], start[b] + torch.arange(S, device="cuda")) for b in range(B)])}
    pools = {"k": s["k"].double(), "v": s["v"].double()}
    scales = {n: s[n + "_scales"].double() if e4m3 else None for n in pools}
    for b in range(B):
        t = start[b] + torch.arange(lens[b], device="cuda")
        pages = s["tables"][LAYER, b].long()
        for n in pools:
            x = s[n + "_new"][b, : lens[b]].double()
            x = _rope64(x, t) if n == "k" else x
            if not e4m3:
                pools[n][pages[t // bs], t % bs] = x
                continue
            for lp in range(start[b] // bs, (start[b] + lens[b] - 1) // bs + 1):
                lo, hi = max(start[b], lp * bs), min(start[b] + lens[b], (lp + 1) * bs)
                r0, p = lo - lp * bs, pages[lp]
                new = x[lo - start[b] : hi - start[b]]
                scale = _scale64(new.abs().amax(dim=(0, 2)))
                if r0 > 0:
                    scale = torch.maximum(scale, scales[n][p])
                    pools[n][p, :r0] = _e4m3(pools[n][p, :r0] * (scales[n][p] / scale)[None, :, None])
                pools[n][p, r0 : r0 + hi - lo] = _e4m3(new / scale[None, :, None])
                scales[n][p] = scale
    return {**out, **pools, "k_scales": scales["k"], "v_scales": scales["v"]}


def _exact_attention(case, seed):
    s = prepare(case, seed)
    H, Hkv, D = HEADS[case["heads"]]
    B, S = s["q"].shape[:2]
    out = torch.zeros((B, S, H, D), dtype=torch.float64, device="cuda")
    lens = [S] * B if s["seq_lens"] is None else s["seq_lens"].tolist()
    for b, c in enumerate(s["context_lens"][LAYER].tolist()):
        pages, m = s["tables"][LAYER, b].long(), lens[b]
        k, v = ((s[n].view(torch.uint8)[pages].view(s[n].dtype).double() * s[n + "_scales"].double()[pages][:, None, :, None])
                .flatten(0, 1)[:c] for n in "kv")
        hidden = torch.arange(c, device="cuda")[None] > (c - m + torch.arange(m, device="cuda"))[:, None]
        for h in range(H):
            score = s["q"][b, :m, h].double() @ k[:, h // (H // Hkv)].T.contiguous() / math.sqrt(D)
            if case["causal"]:
                score[hidden] = -math.inf
            out[b, :m, h] = torch.softmax(score, dim=1) @ v[:, h // (H // Hkv)].contiguous()
    return out


def exact(case, seed):
    """What ``run`` returns on ``prepare(case, seed)``'s inputs, in 64 bits."""
    return _exact_append(case, seed) if case["kind"] == "append" else _exact_attention(case, seed)
