"""Plain 64-bit forms of attention of many query rows over the same keys (include/gqa_batch.h), on the CPU."""
import torch

from tests import gqa_util as R

PAGE = R.PAGE


def attend(q, k, v, first, last, scale, softcap=0.0, add=None):
    """q [n_q, heads, dk] over k, v [n, kv_heads, width], query j seeing rows first[j] .. last[j] - 1; add [n] (or [n_q, n]): a mask's numbers or None.
    Returns out and the bound of its error before the result's own rounding, [n_q, heads, dv] in float64."""
    n_q, heads, dk = q.shape
    n, kv_heads, dv = v.shape
    group = heads // kv_heads
    out, off = (torch.zeros((n_q, heads, dv), dtype=torch.float64) for _ in range(2))
    if n == 0 or n_q == 0:
        return out, off
    i = torch.arange(n)[None]
    see = (i >= first[:, None]) & (i < last[:, None])
    add = torch.zeros((n_q, n), dtype=torch.float64) if add is None else add.double().expand(n_q, n)
    see = see & (add != float("-inf"))
    add = torch.where(see, add, 0.0)
    live = see.any(1)
    step = R.half_step(q.dtype)
    # what nobody sees may hold anything
    seen = see.any(0)
    for g in range(kv_heads):
        kk, vv = (torch.where(seen[:, None], x[:, g].double(), 0.0) for x in (k, v))
        for h in range(g * group, (g + 1) * group):
            x = q[:, h].double()
            s = x @ kk.T * scale
            size = (torch.where(see, x.abs() @ kk.abs().T, 0.0)).amax(1) * abs(scale)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            s = torch.where(see, s + add, float("-inf"))
            p = torch.softmax(s, 1)
            p[~live] = 0.0
            top = torch.where(see, s.abs(), 0.0).amax(1)
            # f32: a dot of dk products is off by at most dk 2^-24 of the sum of their sizes, the cap by 2^-20 of itself, what is added by 2^-22 of
            # the sum's size; the softmax turns a score's error into twice that of its weights
            ds = dk * 2.0 ** -24 * size + softcap * 2.0 ** -20 + 2.0 ** -22 * top
            # a weight is rounded to the type (half a step of it; f16: no finer than 2^-36 of the largest) after its sum is taken; the
            # sum over the rows: 2^-24 an addition, and as much for those of the weights
            rel = 2 * ds + 2.0 ** -20 + step + 2 * n * 2.0 ** -24
            out[:, h] = p @ vv
            off[:, h] = (p @ vv.abs()) * rel[:, None] + n * 2.0 ** -36 * vv.abs().amax()
    return out, off


def prompt(q, k_cache, v_cache, bt, lens, starts, scale, softcap=0.0, window=0, causal=True, mask=None):
    """out, off [n_tok, heads, dv]; rows of tokens of no sequence: NaN."""
    n_tok, heads, _ = q.shape
    cap = bt.shape[1] * PAGE
    out, off = (torch.full((n_tok, heads, v_cache.shape[3]), float("nan"), dtype=torch.float64) for _ in range(2))
    for b in range(bt.shape[0]):
        a, e = int(starts[b]), int(starts[b + 1])
        n = min(max(int(lens[b]), 0), cap)
        at = torch.arange(n)
        page = bt[b].long()[at // PAGE]
        ok = (page >= 0) & (page < k_cache.shape[0])
        add = torch.zeros(n, dtype=torch.float64)
        if mask is not None:
            w = min(mask.shape[1], n)
            add = torch.full((n,), float("-inf"), dtype=torch.float64)
            add[:w] = mask[b, :w].double()
        add[~ok] = float("-inf")
        page = torch.where(ok, page, 0)
        last = (n - (e - a) + torch.arange(e - a) + 1).clamp(0, n) if causal else torch.full((e - a,), n)
        first = (last - window).clamp(min=0) if window else torch.zeros_like(last)
        out[a:e], off[a:e] = attend(q[a:e], k_cache[page, at % PAGE], v_cache[page, at % PAGE], first, last, scale, softcap, add)
    return out, off


def cross(q, k, v, starts, lens, scale, softcap=0.0, mask=None, kv_starts=None):
    """k, v [n_seq, n, heads, width], or packed with kv_starts."""
    n_tok, heads, _ = q.shape
    out, off = (torch.full((n_tok, heads, v.shape[-1]), float("nan"), dtype=torch.float64) for _ in range(2))
    for b in range(len(starts) - 1):
        a, e = int(starts[b]), int(starts[b + 1])
        kb, vb = (x[b] if kv_starts is None else x[min(max(int(kv_starts[b]), 0), x.shape[0]):] for x in (k, v))
        if kv_starts is not None and not 0 <= int(kv_starts[b]) <= k.shape[0]:
            kb, vb = kb[:0], vb[:0]
        n = min(max(int(lens[b]), 0), kb.shape[0])
        add = None
        if mask is not None:
            w = min(mask.shape[1], n)
            add = torch.full((n,), float("-inf"), dtype=torch.float64)
            add[:w] = mask[b, :w].double()
        last = torch.full((e - a,), n)
        out[a:e], off[a:e] = attend(q[a:e], kb[:n], vb[:n], torch.zeros_like(last), last, scale, softcap, add)
    return out, off
