"""Attention in which a row of keys serves many queries, as measurable cases: what a serving loop over caches of ordinary heads does besides the
attention of one new token a sequence.

    prompt  attention of many new tokens of every sequence (a prompt, a chunk of one, draft tokens to verify) over its pages, each token up to itself
    cross   attention of a decoder's tokens to an encoder's states, which have a length of their own and lie in one piece, padded or packed
    prefix  attention of one new token of every sequence where groups of sequences share their first rows: those are read once a group

A paged cache is a tensor [pages, 128, KV heads, width], stored rows first ("cells") or heads first inside a page ("heads").
"""
import math

import torch

own = False

PAGE = 128
DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16}
LOWEST_COST = 4096   # bytes: an empty pass


def _prompt(name, n_seq, heads, kv_heads, dk, dv, kv, q_lo, q_hi, past_lo, past_hi, layout="cells", window=0, softcap=0.0, mask=False):
    """q_lo .. q_hi new tokens a sequence behind past_lo .. past_hi cached rows."""
    c = dict(op="prompt", n_seq=n_seq, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv, kv=kv, q_lo=q_lo, q_hi=q_hi, past_lo=past_lo, past_hi=past_hi, layout=layout, window=window,
             softcap=softcap, mask=mask)
    return dict(c, name=name) if name else c


def _cross(name, n_seq, heads, kv_heads, dk, dv, kv, q_lo, q_hi, lo, hi, packed=False, softcap=0.0, mask=False):
    """q_lo .. q_hi tokens a sequence over lo .. hi states, which are packed one sequence behind the other or padded to the longest."""
    c = dict(op="cross", n_seq=n_seq, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv, kv=kv, q_lo=q_lo, q_hi=q_hi, lo=lo, hi=hi, packed=packed, softcap=softcap, mask=mask)
    return dict(c, name=name) if name else c


def _prefix(name, n_seq, n_prefix, alone, heads, kv_heads, dk, dv, kv, p_lo, p_hi, lo, hi, layout="cells", softcap=0.0, mask=False):
    """n_prefix groups of sequences that share p_lo .. p_hi rows and have lo .. hi of their own; the last `alone` sequences share nothing."""
    c = dict(op="prefix", n_seq=n_seq, n_prefix=n_prefix, alone=alone, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv, kv=kv, p_lo=p_lo, p_hi=p_hi, lo=lo, hi=hi, layout=layout, softcap=softcap,
             mask=mask)
    return dict(c, name=name) if name else c


def listed():
    return [
        # eight draft tokens of one user verified behind 4000 rows, 32 query heads on 8 KV heads: latency
        _prompt("prompt_1x8_past4k_bf16", 1, 32, 8, 128, 128, "bf16", 8, 8, 4000, 4000),
        # a batch of four fresh prompts of ordinary lengths
        _prompt("prompt_4x2k_bf16", 4, 32, 8, 128, 128, "bf16", 1500, 2048, 0, 0),
        # chunks of 512 tokens of eight users behind contexts of up to 16384 rows, heads of 64, a cache stored heads first
        _prompt("prompt_8x512_past16k_f16", 8, 16, 4, 64, 64, "f16", 512, 512, 5000, 16384, layout="heads"),
        # two long prompts of heads that each have their own keys, 192 wide, values 128 wide; a mask hides padding in front
        _prompt("prompt_2x4k_192_mask_bf16", 2, 16, 16, 192, 128, "bf16", 3500, 4096, 0, 0, mask=True),
        # windows of 1024 rows and capped scores, heads of 256
        _prompt("prompt_6x700_window_cap_f16", 6, 16, 4, 256, 256, "f16", 300, 700, 100, 4000, window=1024, softcap=50.0),
        # one user's document of 16384 tokens in one go: the largest
        _prompt("prompt_1x16k_bf16", 1, 32, 8, 128, 128, "bf16", 16384, 16384, 0, 0),
        # the next token of 16 users over 1500 encoder states, each head with keys of its own
        _cross("cross_16x1_1500_f16", 16, 16, 16, 64, 64, "f16", 1, 1, 1500, 1500),
        # texts of up to 448 tokens over ragged encoder states, padded, a mask over some of them
        _cross("cross_8x448_ragged_mask_bf16", 8, 16, 16, 64, 64, "bf16", 100, 448, 300, 1500, mask=True),
        # grouped heads, long inputs packed one behind the other
        _cross("cross_3x1k_8k_packed_bf16", 3, 32, 8, 128, 128, "bf16", 600, 1024, 3000, 8192, packed=True),
        # a full server whose 32 users share a system prompt of 8192 rows
        _prefix("prefix_32_8k_bf16", 32, 1, 0, 32, 8, 128, 128, "bf16", 8192, 8192, 10, 700),
        # four groups of users and some without one, heads of 64, a cache stored heads first
        _prefix("prefix_60_in_4_f16", 60, 4, 7, 16, 4, 64, 64, "f16", 1000, 5000, 1, 2000, layout="heads"),
        # five answers sampled from one context of 100000 rows
        _prefix("prefix_5_100k_bf16", 5, 1, 0, 32, 8, 128, 128, "bf16", 100000, 100000, 1, 300),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


SHAPES = [(32, 8, 128, 128), (16, 4, 64, 64), (16, 16, 192, 128), (16, 4, 256, 256), (28, 4, 128, 128), (64, 2, 128, 128), (7, 7, 64, 64)]


def draw(rng):
    kv = rng.choice(["bf16", "f16"])
    heads, kv_heads, dk, dv = rng.choice(SHAPES)
    softcap, mask = rng.choice([0.0, 0.0, 30.0]), rng.random() < 0.25
    op = rng.choice(["prompt", "cross", "prefix"])
    layout = rng.choice(["cells", "heads"])
    pairs = (1 << 31) // heads                  # (query, key) pairs of all sequences: at the widest heads the largest listed case's work
    if op == "prefix":
        n_seq = _log(rng, 1, 96)
        n_prefix = rng.randrange(1, min(n_seq, 6) + 1)
        alone = rng.randrange(0, n_seq - n_prefix + 1) if rng.random() < 0.4 else 0
        hi = _log(rng, 1, 4000)
        p_hi = _log(rng, 60, min(100000, (1 << 22) // (n_seq * kv_heads)))
        return _prefix(None, n_seq, n_prefix, alone, heads, kv_heads, dk, dv, kv, max(1, int(p_hi * rng.uniform(0.3, 1.0))), p_hi, max(1, int(hi * rng.uniform(0.1, 1.0))), hi, layout, softcap, mask)
    n_seq = _log(rng, 1, 32)
    q_hi = 1 if op == "cross" and rng.random() < 0.3 else _log(rng, 1, min(6000, math.isqrt(pairs // n_seq)))
    q_lo = max(1, int(q_hi * rng.uniform(0.1, 1.0)))
    room = min(40000, max(16, pairs // (n_seq * q_hi)), (1 << 21) // (n_seq * kv_heads))
    if op == "cross":
        hi = _log(rng, 16, room)
        return _cross(None, n_seq, heads, kv_heads, dk, dv, kv, q_lo, q_hi, max(1, int(hi * rng.uniform(0.1, 1.0))), hi, rng.random() < 0.5, softcap, mask)
    past_hi = rng.choice([0, _log(rng, 1, max(1, room - q_hi))]) if room > q_hi else 0
    return _prompt(None, n_seq, heads, kv_heads, dk, dv, kv, q_lo, q_hi, int(past_hi * rng.uniform(0.1, 1.0)), past_hi, layout, rng.choice([0, 0, 0, 1 + (q_hi + past_hi) // 3]), softcap, mask)


# ---------------------------------------------------------------- inputs

def _between(gen, dev, lo, hi, n):
    """n lengths, the first of them the longest, so that the widths of tables do not depend on the seed."""
    x = torch.randint(lo, hi + 1, (n,), generator=gen, device=dev)
    x[0] = hi
    return x


def _between_of_one_sum(gen, dev, lo, hi, n):
    """The same for lengths whose sum does not depend on the seed: pairs that lie as far above lo as below hi."""
    off = torch.randint(0, hi - lo + 1, ((n - 1) // 2,), generator=gen, device=dev)
    middle = off.new_full(((n - 1) % 2,), (lo + hi) // 2)
    return torch.cat((off.new_full((1,), hi), lo + off, hi - off, middle))


def _values(gen, dev, shape, dtype):
    return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32 if math.prod(shape) < (1 << 25) else dtype).to(dtype)


def _cache(gen, dev, n_pages, heads, width, dtype, layout):
    """[pages, 128, heads, width], rows or heads outermost inside a page."""
    t = _values(gen, dev, (n_pages, PAGE, heads, width) if layout == "cells" else (n_pages, heads, PAGE, width), dtype)
    return t if layout == "cells" else t.transpose(1, 2)


def _starts(n):
    return torch.nn.functional.pad(torch.cumsum(n, 0), (1, 0)).to(torch.int32)


def _mask(gen, dev, n_seq, n, pad_hi):
    """Padding in front, of another length for every sequence, and a few rows struck out further on."""
    pad = torch.randint(0, max(1, pad_hi), (n_seq, 1), generator=gen, device=dev)
    out = (torch.arange(n, device=dev)[None] < pad) | (torch.rand((n_seq, n), generator=gen, device=dev) < 0.02)
    return torch.where(out, float("-inf"), 0.0).to(torch.float16)


def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    kv = DTYPE[c["kv"]]
    s = dict(c)
    s["scale"] = 1.0 / math.sqrt(c["dk"])
    n_seq = c["n_seq"]
    if c["op"] == "prefix":
        n_prefix, in_groups = c["n_prefix"], n_seq - c["alone"]
        # groups of sequences that lie side by side in the batch, of odd sizes
        cuts = 1 + torch.randperm(in_groups - 1, generator=gen, device=dev)[:n_prefix - 1].sort().values
        s["prefix_starts"] = torch.cat((cuts.new_zeros(1), cuts, cuts.new_full((1,), in_groups))).to(torch.int32)
        s["prefix_lens"] = _between(gen, dev, c["p_lo"], c["p_hi"], n_prefix).to(torch.int32)
        mine = _between(gen, dev, c["lo"], c["hi"], n_seq)
        group = torch.searchsorted(s["prefix_starts"][1:].contiguous(), torch.arange(n_seq, device=dev, dtype=torch.int32), right=True)
        shared = torch.nn.functional.pad(s["prefix_lens"], (0, 1))[group].long()
        s["seq_lens"] = (mine + shared).to(torch.int32)
        # whole pages of the shared rows are the same pages; a page that begins with shared rows is each sequence's own copy of them
        width, per = (c["p_hi"] + c["hi"] + PAGE - 1) // PAGE, (c["hi"] + 2 * PAGE - 2) // PAGE
        whole = c["p_hi"] // PAGE
        n_pages = n_prefix * whole + n_seq * per
        ids = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32)
        j = torch.arange(width, device=dev)[None]
        full = (shared // PAGE)[:, None]
        at = torch.where(j < full, group[:, None] * whole + j, n_prefix * whole + torch.arange(n_seq, device=dev)[:, None] * per + (j - full).clamp(max=per - 1))
        used = j * PAGE < s["seq_lens"][:, None]
        s["block_table"] = torch.where(used, ids[torch.where(used, at, 0)], 0).to(torch.int32).contiguous()
        s["k_cache"] = _cache(gen, dev, n_pages, c["kv_heads"], c["dk"], kv, c["layout"])
        s["v_cache"] = _cache(gen, dev, n_pages, c["kv_heads"], c["dv"], kv, c["layout"])
        first = torch.nn.functional.pad(s["prefix_starts"][:-1], (0, 1))[group].long()
        edge = (shared // PAGE).clamp(max=width - 1)
        row = torch.arange(PAGE, device=dev)
        b, i = torch.nonzero((row[None] < (shared % PAGE)[:, None]) & (group < n_prefix)[:, None], as_tuple=True)
        for cache in (s["k_cache"], s["v_cache"]):
            cache[s["block_table"][b, edge[b]].long(), i] = cache[s["block_table"][first[b], edge[b]].long(), i]
        s["q"] = _values(gen, dev, (n_seq, c["heads"], c["dk"]), kv)
        s["row_mask"] = _mask(gen, dev, n_seq, width * PAGE, c["lo"]) if c["mask"] else None
        return s
    n_q = _between_of_one_sum(gen, dev, c["q_lo"], c["q_hi"], n_seq)
    s["q_starts"] = _starts(n_q)
    n_tok = int(s["q_starts"][-1])
    s["q"] = _values(gen, dev, (n_tok, c["heads"], c["dk"]), kv)
    if c["op"] == "prompt":
        s["seq_lens"] = (n_q + _between(gen, dev, c["past_lo"], c["past_hi"], n_seq)).to(torch.int32)
        width = (c["q_hi"] + c["past_hi"] + PAGE - 1) // PAGE
        n_pages = n_seq * width
        ids = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32).view(n_seq, width)
        s["block_table"] = torch.where(torch.arange(width, device=dev)[None] * PAGE < s["seq_lens"][:, None], ids, 0).to(torch.int32).contiguous()
        s["k_cache"] = _cache(gen, dev, n_pages, c["kv_heads"], c["dk"], kv, c["layout"])
        s["v_cache"] = _cache(gen, dev, n_pages, c["kv_heads"], c["dv"], kv, c["layout"])
        s["row_mask"] = _mask(gen, dev, n_seq, width * PAGE, (c["q_lo"] + c["past_lo"]) // 2) if c["mask"] else None
        return s
    n_kv = _between(gen, dev, c["lo"], c["hi"], n_seq)
    s["kv_lens"] = n_kv.to(torch.int32)
    s["kv_starts"] = _starts(n_kv) if c["packed"] else None
    shape = (int(n_kv.sum()),) if c["packed"] else (n_seq, c["hi"])
    s["k"] = _values(gen, dev, shape + (c["kv_heads"], c["dk"]), kv)
    s["v"] = _values(gen, dev, shape + (c["kv_heads"], c["dv"]), kv)
    s["row_mask"] = _mask(gen, dev, n_seq, c["hi"], c["lo"] // 2) if c["mask"] else None
    return s


# ---------------------------------------------------------------- the operators

def run(state):
    return {"prompt": _run_prompt, "cross": _run_cross, "prefix": _run_prefix}[state["op"]](state)


def _attend(s, q, k, v, visible):
    """q [n_seq, n_q, heads, dk] over k, v [n_seq, n, kv_heads, width]; visible [n_seq or 1, n_q or 1, n]: [n_seq, n_q, heads, dv] in 32 bits."""
    n_seq, n_q, heads, dk = q.shape
    kv_heads = s["kv_heads"]
    group = heads // kv_heads
    q = q.float().view(n_seq, n_q, kv_heads, group, dk).permute(0, 2, 1, 3, 4).reshape(n_seq, kv_heads, n_q * group, dk)
    score = torch.matmul(q, k.float().permute(0, 2, 3, 1).contiguous()).mul_(s["scale"]).view(n_seq, kv_heads, n_q, group, -1)
    if s["softcap"]:
        score = score.div_(s["softcap"]).tanh_().mul_(s["softcap"])
    if s["row_mask"] is not None:
        score = score.add_(s["row_mask"].float()[:, None, None, None])
    score = score.masked_fill_(~visible[:, None, :, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_min(1e-38))
    out = torch.matmul(p.view(n_seq, kv_heads, n_q * group, -1), v.float().permute(0, 2, 1, 3).contiguous())
    return out.view(n_seq, kv_heads, n_q, group, -1).permute(0, 2, 1, 3, 4).reshape(n_seq, n_q, heads, -1)


def _rows(s):
    """Row number of every key a sequence may have [1, n] and its page [n_seq, n]."""
    t = torch.arange(s["block_table"].shape[1] * PAGE, device=s["block_table"].device)[None]
    return t, s["block_table"].long().repeat_interleave(PAGE, 1)


def _padded(s):
    """The queries [n_seq, q_hi, heads, dk], how many each sequence has [n_seq, 1], and, to go back, the place (sequence, number) of every token."""
    starts = s["q_starts"].long()
    n_q = (starts[1:] - starts[:-1])[:, None]
    at = starts[:-1, None] + torch.arange(s["q_hi"], device=starts.device)[None]
    q = s["q"][at.clamp(max=s["q"].shape[0] - 1)]
    tok = torch.arange(s["q"].shape[0], device=starts.device)
    b = torch.searchsorted(starts[1:].contiguous(), tok, right=True)
    return q, n_q, (b, tok - starts[b])


def _run_prompt(s):
    if own:
        import jittorinfer_amd as J
        return J.gqa_prompt_attn(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["seq_lens"], s["q_starts"], scale=s["scale"], logit_softcap=s["softcap"], window=s["window"],
                                 mask=s["row_mask"])
    t, page = _rows(s)
    q, n_q, back = _padded(s)
    k, v = s["k_cache"][page, t % PAGE], s["v_cache"][page, t % PAGE]
    # token j of a sequence's new ones is its row lens - n_q + j, and sees what is there up to itself
    last = (s["seq_lens"].long()[:, None] - n_q + torch.arange(q.shape[1], device=q.device)[None])[..., None]
    visible = t[None] <= last
    if s["window"]:
        visible = visible & (t[None] > last - s["window"])
    return _attend(s, q, k, v, visible)[back].to(s["q"].dtype)


def _run_cross(s):
    if own:
        import jittorinfer_amd as J
        if s["packed"]:
            return J.gqa_cross_attn(s["q"], s["k"], s["v"], q_starts=s["q_starts"] if s["q_hi"] > 1 else None, kv_starts=s["kv_starts"], scale=s["scale"], logit_softcap=s["softcap"], mask=s["row_mask"])
        return J.gqa_cross_attn(s["q"], s["k"], s["v"], q_starts=s["q_starts"] if s["q_hi"] > 1 else None, kv_lens=s["kv_lens"], scale=s["scale"], logit_softcap=s["softcap"], mask=s["row_mask"])
    q, _, back = _padded(s)
    k, v = s["k"], s["v"]
    t = torch.arange(s["hi"], device=q.device)[None]
    if s["packed"]:
        at = (s["kv_starts"].long()[:-1, None] + t).clamp(max=k.shape[0] - 1)
        k, v = k[at], v[at]
    return _attend(s, q, k, v, (t < s["kv_lens"][:, None])[:, None])[back].to(s["q"].dtype)


def _run_prefix(s):
    if own:
        import jittorinfer_amd as J
        return J.gqa_prefix_attn(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["seq_lens"], s["prefix_starts"], s["prefix_lens"], scale=s["scale"], logit_softcap=s["softcap"],
                                 mask=s["row_mask"])
    t, page = _rows(s)
    k, v = s["k_cache"][page, t % PAGE], s["v_cache"][page, t % PAGE]
    return _attend(s, s["q"][:, None], k, v, (t < s["seq_lens"][:, None])[:, None])[:, 0].to(s["q"].dtype)


# ---------------------------------------------------------------- what a pass cannot do without

def _mean(lo, hi, n):
    """Of n lengths between lo and hi, the first of them hi (the seed makes the others)."""
    return (hi + (n - 1) * (lo + hi) / 2) / n


def work(case):
    c = case
    e = 2
    row = c["kv_heads"] * (c["dk"] + c["dv"]) * e
    pair = 2 * c["heads"] * (c["dk"] + c["dv"])
    token = c["heads"] * (c["dk"] + c["dv"]) * e
    if c["op"] == "prefix":
        mine, shared = _mean(c["lo"], c["hi"], c["n_seq"]), _mean(c["p_lo"], c["p_hi"], c["n_prefix"])
        seen = c["n_seq"] * mine + (c["n_seq"] - c["alone"]) * shared
        rows = c["n_seq"] * mine + c["n_prefix"] * shared
        return {"bytes": rows * row + c["n_seq"] * token + (seen * 2 if c["mask"] else 0) + LOWEST_COST, "flops": seen * pair}
    n_q = _mean(c["q_lo"], c["q_hi"], c["n_seq"])
    if c["op"] == "cross":
        n = _mean(c["lo"], c["hi"], c["n_seq"])
        return {"bytes": c["n_seq"] * (n * row + n_q * token + (n * 2 if c["mask"] else 0)) + LOWEST_COST, "flops": c["n_seq"] * n_q * n * pair}
    past = _mean(c["past_lo"], c["past_hi"], c["n_seq"])
    w = c["window"]
    keys = min(past, w) + n_q if w else past + n_q
    # of n_q queries the j-th sees past + j + 1 rows, or the window
    seen = n_q * past + n_q * (n_q + 1) / 2
    if w:
        ramp = min(n_q, max(0.0, w - past))      # queries that see less than the window
        seen = ramp * past + ramp * (ramp + 1) / 2 + (n_q - ramp) * min(w, past + n_q)
    return {"bytes": c["n_seq"] * (keys * row + n_q * token + (keys * 2 if c["mask"] else 0)) + LOWEST_COST, "flops": c["n_seq"] * seen * pair}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    heads, group = s["heads"], s["heads"] // s["kv_heads"]
    out = torch.zeros((s["q"].shape[0], heads, s["dv"]), dtype=torch.float64, device=s["q"].device)
    for b in range(s["n_seq"]):
        if s["op"] == "prefix":
            first, n_q = b, 1
        else:
            first, end = (int(x) for x in s["q_starts"][b:b + 2])
            n_q = end - first
        if s["op"] == "cross":
            n = int(s["kv_lens"][b])
            k_all, v_all = (x[int(s["kv_starts"][b]):][:n] if s["packed"] else x[b, :n] for x in (s["k"], s["v"]))
        else:
            n = int(s["seq_lens"][b])
            at = torch.arange(n, device=out.device)
            page = s["block_table"][b].long()[at // PAGE]
            k_all, v_all = s["k_cache"][page, at % PAGE], s["v_cache"][page, at % PAGE]
        # queries in pieces, so that a piece's scores stay small
        step = max(1, (1 << 25) // max(1, n))
        for j0 in range(0, n_q, step):
            j = torch.arange(j0, min(n_q, j0 + step), device=out.device)
            see = torch.ones((len(j), n), dtype=torch.bool, device=out.device)
            if s["op"] == "prompt":
                me = n - n_q + j[:, None]
                see = torch.arange(n, device=out.device)[None] <= me
                if s["window"]:
                    see &= torch.arange(n, device=out.device)[None] + s["window"] > me
            for g in range(s["kv_heads"]):
                k, v = k_all[:, g].double(), v_all[:, g].double()
                for h in range(g * group, (g + 1) * group):
                    x = (s["q"][first + j, h].double() @ k.T.contiguous()) * s["scale"]
                    if s["softcap"]:
                        x = torch.tanh(x / s["softcap"]) * s["softcap"]
                    if s["row_mask"] is not None:
                        x = x + s["row_mask"][b, :n].double()
                    x = torch.where(see, x, float("-inf"))
                    out[first + j, h] = torch.softmax(x, 1).nan_to_num(0.0) @ v      # no row left: no weight anywhere
    return out
