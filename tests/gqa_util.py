"""Plain 64-bit forms of the operators of a paged cache of ordinary heads (include/gqa_attn.h), on the CPU, and caches to run them on."""
import math

import torch

PAGE = 128


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make_cache(gen, n_pages, heads, width, dtype, layout="cells", fill=None):
    """[n_pages, 128, heads, width]; every row that no test writes holds `fill` (NaN: a result that depends on it shows)."""
    shape = (n_pages, PAGE, heads, width) if layout == "cells" else (n_pages, heads, PAGE, width)
    t = torch.randn(shape, generator=gen).to(dtype) if fill is None else torch.full(shape, fill, dtype=dtype)
    return t if layout == "cells" else t.transpose(1, 2)


def make_table(gen, lens, width, n_pages):
    """Distinct shuffled pages for what the lengths need, 0 elsewhere."""
    ids = torch.randperm(n_pages, generator=gen).tolist()
    bt = torch.zeros((len(lens), width), dtype=torch.int32)
    for b, n in enumerate(lens):
        for j in range((max(n, 0) + PAGE - 1) // PAGE):
            bt[b, j] = ids.pop()
    return bt


def rows_of(cache, bt, b, first, last):
    """Rows first .. last - 1 of sequence b: [rows, heads, width] float64."""
    at = torch.arange(first, last)
    return cache[bt[b].long()[at // PAGE], at % PAGE].double()


def span(n, cap, window):
    n = min(max(n, 0), cap)
    return (max(0, n - window) if window else 0), n


def attn(q, k_cache, v_cache, bt, lens, scale, softcap=0.0, window=0, mask=None, n_pages=None):
    """out [n_seq, heads, dv], weights [n_seq, kv heads, width * 128] and the bound of either's error in f32 (see below), in float64."""
    n_seq, heads, dk = q.shape
    kv_heads = k_cache.shape[2]
    dv = v_cache.shape[3] if v_cache is not None else 0
    group, cap = heads // kv_heads, bt.shape[1] * PAGE
    out, off = torch.zeros((n_seq, heads, dv), dtype=torch.float64), torch.zeros((n_seq, heads, dv), dtype=torch.float64)
    weights, w_off = (torch.zeros((n_seq, kv_heads, cap), dtype=torch.float64) for _ in range(2))
    for b in range(n_seq):
        first, last = span(int(lens[b]), cap, window)
        at = torch.arange(first, last)
        ok = (bt[b].long()[at // PAGE] >= 0) & (bt[b].long()[at // PAGE] < k_cache.shape[0])
        add = torch.zeros(len(at), dtype=torch.float64)
        if mask is not None:
            ok &= at < mask.shape[1]
            at_m = at.clamp(max=mask.shape[1] - 1)
            add = mask[b, at_m].double()
            ok &= add != float("-inf")
        at, add = at[ok], add[ok]
        if not len(at):
            continue
        page, row = bt[b].long()[at // PAGE], at % PAGE
        for g in range(kv_heads):
            k = k_cache[page, row, g].double()
            qg = q[b, g * group:(g + 1) * group].double()
            s = qg @ k.T * scale
            size = (qg.abs() @ k.abs().T).amax(1) * abs(scale)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            s = s + add
            p = torch.softmax(s, 1)
            # f32: a dot of dk products is off by at most dk 2^-24 of the sum of their sizes, the cap by 2^-20 of itself (one exp2, one
            # reciprocal), what is added by 2^-24 of the sum's size; the softmax turns a score's error into twice that of its weights
            ds = dk * 2.0 ** -24 * size + softcap * 2.0 ** -20 + 2.0 ** -22 * s.abs().amax(1)
            rel = 2 * ds + 2.0 ** -20
            weights[b, g, at] = p.sum(0)
            w_off[b, g, at] = (p * rel[:, None]).sum(0)
            if dv:
                v = v_cache[page, row, g].double()
                out[b, g * group:(g + 1) * group] = p @ v
                # P as two 16-bit halves: 2^-16 of it at most; the sum over the rows: 2^-24 an addition
                off[b, g * group:(g + 1) * group] = (p @ v.abs()) * (rel + 2.0 ** -16 + len(at) * 2.0 ** -24)[:, None]
    return out, off, weights, w_off


def heads(x, weight, eps, pos, n_dims, mode, n_ctx_orig=0, freq_base=10000.0, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0,
          freq_factors=None):
    """Normed and rotated rows [tokens, heads, dk] and the bound of their error in f32, in float64."""
    x = x.double()
    dk = x.shape[-1]
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    out, size = x.clone(), x.abs()
    mag = attn_factor * (1 + 0.1 * math.log(1 / freq_scale)) if ext_factor else attn_factor
    lo = hi = 0
    if ext_factor:
        lo = max(0, math.floor(n_dims * math.log(n_ctx_orig / (beta_fast * 2 * math.pi)) / (2 * math.log(freq_base))))
        hi = min(n_dims - 1, math.ceil(n_dims * math.log(n_ctx_orig / (beta_slow * 2 * math.pi)) / (2 * math.log(freq_base))))
    for i in range(n_dims // 2):
        a, b = (i, i + n_dims // 2) if mode == 2 else (2 * i, 2 * i + 1)
        scale = freq_scale
        if ext_factor:
            mix = (1 - min(1.0, max(0.0, (i - lo) / max(0.001, hi - lo)))) * ext_factor
            scale = scale * (1 - mix) + mix
        t = pos.double()[:, None] * scale * freq_base ** (-2.0 * i / n_dims) / (float(freq_factors[i]) if freq_factors is not None else 1.0)
        c, s = torch.cos(t) * mag, torch.sin(t) * mag
        out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
        size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * mag
    # f32: the sum of dk squares by dk 2^-24 (half of that in its root), four roundings of a normed value, sine and cosine 2^-22 each with the
    # fraction of the turn, two roundings of the rotation
    return out, size * (dk * 2.0 ** -25 + 2.0 ** -20)


def evict(weights, bt, lens, k_cache, v_cache, n_keep, n_sink, n_recent):
    """(kept, new_lens, weights, k_cache, v_cache) after the eviction, by ranking."""
    n_seq, kv_heads, cap = weights.shape
    k_new, v_new = k_cache.clone(), v_cache.clone() if v_cache is not None else None
    kept = torch.full((n_seq, kv_heads, n_keep), -1, dtype=torch.int32)
    out = torch.zeros_like(weights)
    new_lens = torch.zeros(n_seq, dtype=torch.int32)
    for b in range(n_seq):
        n = min(max(int(lens[b]), 0), cap)
        new_lens[b] = min(n, n_keep)
        for h in range(kv_heads):
            rows = torch.arange(n)
            if n > n_keep:
                middle = rows[n_sink:n - n_recent]
                w = weights[b, h, middle]
                nan = torch.isnan(w)                                          # below -inf itself
                order = torch.argsort(torch.where(nan, float("-inf"), w), descending=True, stable=True)
                order = order[torch.argsort(nan[order].int(), stable=True)]
                rows = torch.cat((rows[:n_sink], middle[order[:n_keep - n_sink - n_recent]].sort().values, rows[n - n_recent:]))
            kept[b, h, :len(rows)] = rows.int()
            out[b, h, :len(rows)] = weights[b, h, rows]
            to = torch.arange(len(rows))
            page = lambda i: bt[b].long()[i // PAGE]
            there = (page(rows) >= 0) & (page(rows) < k_cache.shape[0]) & (page(to) >= 0) & (page(to) < k_cache.shape[0])
            rows, to = rows[there], to[there]
            k_new[page(to), to % PAGE, h] = k_cache[page(rows), rows % PAGE, h]
            if v_new is not None:
                v_new[page(to), to % PAGE, h] = v_cache[page(rows), rows % PAGE, h]
    return kept, new_lens, out, k_new, v_new


def bits(t):
    """Equal bits, NaN included."""
    return t.contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32, 8: torch.int64}[t.element_size()])
