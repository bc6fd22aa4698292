"""The operators of a paged key-value cache of ordinary attention heads, as measurable cases.

A model whose layers keep keys and values per head (grouped queries, one KV head for a group of query heads; a key head as wide as its
value head, or 192 against 128 as DeepSeek-V2 has them without the absorbed form) serves its tokens with three calls:

    norm_rope  the RMS norms of every head's query and key, their rotation, and the write of the new keys and values into the cache
    attn       attention of one new token of every sequence over its pages, optionally adding up the weight every cached row received;
               over a latent cache (rows of 576, one KV head) the weights alone
    evict      rows of little accumulated weight leave the cache: the rows kept move up, in order, in the pages the sequence has

Pages hold 128 rows; a cache is a tensor [pages, 128, KV heads, width], stored rows first ("cells") or heads first inside a page ("heads").
"""
import math

import torch

own = False

PAGE = 128
DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
YARN = dict(n_ctx_orig=4096, freq_scale=0.025, ext_factor=1.0, attn_factor=0.8)   # as DeepSeek-V2 configures it
EPS = 1e-6
LOWEST_COST = 4096   # bytes: an empty pass


def _norm_rope(name, n_tok, n_seq, heads, kv_heads, dk, dv, src, kv, mode, n_dims, past, yarn=False, norm=True, layout="cells"):
    c = dict(op="norm_rope", n_tok=n_tok, n_seq=n_seq, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv, src=src, kv=kv, mode=mode, n_dims=n_dims, past=past, yarn=yarn,
             norm=norm, layout=layout)
    return dict(c, name=name) if name else c


def _attn(name, n_seq, heads, kv_heads, dk, dv, kv, lo, hi, layout="cells", window=0, softcap=0.0, mask=False, weights=False):
    c = dict(op="attn", n_seq=n_seq, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv, kv=kv, lo=lo, hi=hi, layout=layout, window=window, softcap=softcap, mask=mask, weights=weights)
    return dict(c, name=name) if name else c


def _evict(name, n_seq, kv_heads, dk, dv, kv, lo, hi, keep, sink, recent, layout="cells"):
    c = dict(op="evict", n_seq=n_seq, kv_heads=kv_heads, dk=dk, dv=dv, kv=kv, lo=lo, hi=hi, keep=keep, sink=sink, recent=recent, layout=layout)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user's next token, 32 query heads on 8 KV heads: latency only
        _norm_rope("norm_rope_1_bf16", 1, 1, 32, 8, 128, 128, "bf16", "bf16", 2, 128, 4000),
        # a decode batch of 64 users from f32 activations, heads of 64, an f16 cache stored heads first
        _norm_rope("norm_rope_64_f32_f16", 64, 64, 16, 4, 64, 64, "f32", "f16", 2, 64, 1000, layout="heads"),
        # prompts of 8 users, ragged, together 8111 tokens; every head rotated in half of its channels with adjacent pairs and YaRN
        _norm_rope("norm_rope_8111_bf16", 8111, 8, 32, 8, 128, 128, "bf16", "bf16", 0, 64, 100000, yarn=True),
        # one user of 32 query heads on 8 KV heads, 1024 tokens: the smallest step
        _attn("attn_1x1k_bf16", 1, 32, 8, 128, 128, "bf16", 1024, 1024),
        # a full server: 32 users, contexts of 700 to 8192 tokens
        _attn("attn_32_ragged_bf16", 32, 32, 8, 128, 128, "bf16", 700, 8192),
        # one user deep in a long context of the other type
        _attn("attn_1x128k_f16", 1, 32, 8, 128, 128, "f16", 131001, 131001, layout="heads"),
        # 16 heads that each have their own keys, 192 wide, values 128 wide, and the sum of the weights for a later eviction; a mask hides padding
        _attn("attn_8x4k_192_weights_bf16", 8, 16, 16, 192, 128, "bf16", 3500, 4096, mask=True, weights=True),
        # 16 users with a window of 1024 rows and capped scores, heads of 256
        _attn("attn_16_window_cap_f16", 16, 16, 4, 256, 256, "f16", 900, 6000, window=1024, softcap=50.0),
        # what every row of a latent cache of 8 users received from 128 heads: the score of an eviction
        _attn("weights_8x8k_latent_bf16", 8, 128, 1, 576, 0, "bf16", 5000, 8192, weights=True),
        # one user's cache of 8192 rows is cut to 4096
        _evict("evict_1x8k_bf16", 1, 8, 128, 128, "bf16", 8192, 8192, 4096, 4, 512),
        # 32 users of ragged lengths, some of them short enough to stay as they are
        _evict("evict_32_ragged_f16", 32, 8, 128, 128, "f16", 1500, 8192, 2048, 16, 256, layout="heads"),
        # a latent cache of one long context
        _evict("evict_2x100k_latent_bf16", 2, 1, 576, 0, "bf16", 99000, 100001, 40000, 4, 1000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kv = rng.choice(["bf16", "f16"])
    layout = rng.choice(["cells", "heads"])
    op = rng.choice(["norm_rope", "attn", "attn", "evict"])
    if op == "evict":
        kv_heads, dk, dv = rng.choice([(8, 128, 128), (4, 64, 64), (16, 192, 128), (2, 256, 256), (1, 576, 0)])
        n_seq = _log(rng, 1, 48)
        hi = _log(rng, 300, min(100000, (1 << 28) // (n_seq * kv_heads * (dk + dv) * 2)))
        lo = max(1, int(hi * rng.uniform(0.2, 1.0)))
        keep = max(48, int(hi * rng.uniform(0.2, 0.8)))
        return _evict(None, n_seq, kv_heads, dk, dv, kv, lo, hi, keep, rng.randrange(0, 17), rng.randrange(0, keep - 32), layout)
    heads, kv_heads, dk, dv = rng.choice([(32, 8, 128, 128), (16, 4, 64, 64), (16, 16, 192, 128), (16, 4, 256, 256), (28, 4, 128, 128), (64, 2, 128, 128), (7, 7, 64, 64)])
    if op == "norm_rope":
        n_tok = _log(rng, 1, 8000)
        n_seq = min(n_tok, rng.randrange(1, 65))
        mode = rng.choice([0, 2])
        return _norm_rope(None, n_tok, n_seq, heads, kv_heads, dk, dv, rng.choice(["f32", kv]), kv, mode, rng.choice([dk, dk // 2]), _log(rng, 1, 130000), rng.random() < 0.3, rng.random() < 0.8, layout)
    weights = rng.random() < 0.3
    if weights and rng.random() < 0.3:
        heads, kv_heads, dk, dv = rng.choice([(128, 1, 576, 0), (16, 1, 576, 0)])
    n_seq = _log(rng, 1, 64)
    hi = _log(rng, 40, min(131072, (1 << 29) // (n_seq * kv_heads * (dk + dv) * 2 + (n_seq * heads * 16 if weights else 0))))
    lo = max(1, int(hi * rng.uniform(0.1, 1.0)))
    return _attn(None, n_seq, heads, kv_heads, dk, dv, kv, lo, hi, layout, rng.choice([0, 0, 0, 1 + hi // 3]), rng.choice([0.0, 0.0, 30.0]), rng.random() < 0.25, weights)


# ---------------------------------------------------------------- inputs

def _lens(c, gen, dev):
    n = torch.randint(c["lo"], c["hi"] + 1, (c["n_seq"],), generator=gen, device=dev)
    n[0] = c["hi"]   # the longest, so that the block table's width does not depend on the seed
    return n.to(torch.int32)


def _cache(gen, dev, n_pages, heads, width, dtype, layout):
    """[pages, 128, heads, width], rows or heads outermost inside a page."""
    shape = (n_pages, PAGE, heads, width) if layout == "cells" else (n_pages, heads, PAGE, width)
    t = torch.randn(shape, generator=gen, device=dev, dtype=torch.float32 if width * heads * n_pages < (1 << 18) else dtype).to(dtype)
    return t if layout == "cells" else t.transpose(1, 2)


def _table(gen, dev, lens, hi):
    """A block table over shuffled pages, unused entries 0, and how many pages the pool has."""
    width = (hi + PAGE - 1) // PAGE
    n_pages = lens.shape[0] * width
    ids = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32).view(lens.shape[0], width)
    used = torch.arange(width, device=dev)[None] * PAGE < lens[:, None]
    return torch.where(used, ids, torch.zeros_like(ids)).contiguous(), n_pages


def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    kv = DTYPE[c["kv"]]
    s = dict(c)
    if c["op"] == "norm_rope":
        src = DTYPE[c["src"]]
        # the projections' output: q, k and v side by side, the heads' rows views of it
        nq, nk = c["heads"] * c["dk"], c["kv_heads"] * c["dk"]
        qkv = (torch.randn((c["n_tok"], nq + nk + c["kv_heads"] * c["dv"]), generator=gen, device=dev) * 2.0).to(src)
        s["q"] = qkv[:, :nq].view(c["n_tok"], c["heads"], c["dk"])
        s["k"] = qkv[:, nq:nq + nk].view(c["n_tok"], c["kv_heads"], c["dk"])
        s["v"] = qkv[:, nq + nk:].view(c["n_tok"], c["kv_heads"], c["dv"])
        s["wq"], s["wk"] = ((1.0 + 0.2 * torch.randn((c["dk"],), generator=gen, device=dev)) if c["norm"] else None for _ in range(2))
        # every sequence gets its share of the tokens, behind `past` cached positions (whole pages of them stay out of this pool)
        at = torch.arange(c["n_tok"], device=dev)
        s["seq_ids"] = (at * c["n_seq"] // c["n_tok"]).to(torch.int32)
        first = (torch.arange(c["n_seq"], device=dev) * c["n_tok"] + c["n_seq"] - 1) // c["n_seq"]
        within = at - first[s["seq_ids"].long()]
        s["pos"] = (within + c["past"]).to(torch.int32)
        s["slots"] = (within + c["past"] % PAGE).to(torch.int32)
        longest = (c["n_tok"] + c["n_seq"] - 1) // c["n_seq"] + c["past"] % PAGE
        s["block_table"], n_pages = _table(gen, dev, torch.full((c["n_seq"],), longest, device=dev), longest)
        s["k_cache"] = _cache(gen, dev, n_pages, c["kv_heads"], c["dk"], kv, c["layout"])
        s["v_cache"] = _cache(gen, dev, n_pages, c["kv_heads"], c["dv"], kv, c["layout"])
        s["rope"] = dict(n_dims=c["n_dims"], mode=c["mode"], freq_base=10000.0, **(YARN if c["yarn"] else {}))
        return s
    s["seq_lens"] = _lens(c, gen, dev)
    s["block_table"], n_pages = _table(gen, dev, s["seq_lens"], c["hi"])
    s["k_cache"] = _cache(gen, dev, n_pages, c["kv_heads"], c["dk"], kv, c["layout"])
    s["v_cache"] = _cache(gen, dev, n_pages, c["kv_heads"], c["dv"], kv, c["layout"]) if c["dv"] else None
    n_max = s["block_table"].shape[1] * PAGE
    if c["op"] == "attn":
        s["q"] = torch.randn((c["n_seq"], c["heads"], c["dk"]), generator=gen, device=dev).to(kv)
        s["scale"] = 1.0 / math.sqrt(192.0 if c["dk"] == 576 else c["dk"])
        if c["mask"]:
            # left padding of another length for every sequence, and a few rows struck out further on
            pad = torch.randint(0, max(1, c["lo"] // 2), (c["n_seq"], 1), generator=gen, device=dev)
            out = (torch.arange(n_max, device=dev)[None] < pad) | (torch.rand((c["n_seq"], n_max), generator=gen, device=dev) < 0.02)
            s["row_mask"] = torch.where(out, float("-inf"), 0.0).to(torch.float16)
        else:
            s["row_mask"] = None
        s["sums"] = torch.rand((c["n_seq"], c["kv_heads"], n_max), generator=gen, device=dev) if c["weights"] else None
    else:
        # accumulated weights are heavy-tailed; rows no query has looked at yet hold exact zeros
        w = torch.exp(2.0 * torch.randn((c["n_seq"], c["kv_heads"], n_max), generator=gen, device=dev))
        s["sums"] = torch.where(torch.rand(w.shape, generator=gen, device=dev) < 0.05, torch.zeros_like(w), w)
    return s


# ---------------------------------------------------------------- the operators

def run(state):
    return {"norm_rope": _run_norm_rope, "attn": _run_attn, "evict": _run_evict}[state["op"]](state)


def _angles(r, pos):
    """The rotation's angles [tokens, n_dims / 2] in 64 bits, and the magnitude scale: ggml_rope_ext's definition, YaRN included."""
    n, base = r["n_dims"], r["freq_base"]
    pair = torch.arange(n // 2, device=pos.device, dtype=torch.float64)
    freq = base ** (-2.0 * pair / n)
    scale, ext, mag = r.get("freq_scale", 1.0), r.get("ext_factor", 0.0), r.get("attn_factor", 1.0)
    if ext:
        start, end = (n * math.log(r["n_ctx_orig"] / (beta * 2 * math.pi)) / (2 * math.log(base)) for beta in (32.0, 1.0))
        start, end = max(0.0, math.floor(start)), min(n - 1.0, math.ceil(end))
        mix = (1.0 - ((pair - start) / max(0.001, end - start)).clamp(0.0, 1.0)) * ext
        freq = freq * (scale * (1.0 - mix) + mix)
        mag = mag * (1.0 + 0.1 * math.log(1.0 / scale))
    else:
        freq = freq * scale
    return pos.double()[:, None] * freq, mag


def _normed_rotated(x, w, r, pos):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    angle, mag = _angles(r, pos)
    cos, sin = (torch.cos(angle) * mag).float()[:, None], (torch.sin(angle) * mag).float()[:, None]
    n = r["n_dims"]
    a, b = (x[..., :n // 2], x[..., n // 2:n]) if r["mode"] == 2 else (x[..., 0:n:2], x[..., 1:n:2])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat((ra, rb), -1) if r["mode"] == 2 else torch.stack((ra, rb), -1).flatten(-2)
    return torch.cat((turned, x[..., n:]), -1)


def _run_norm_rope(s):
    if own:
        import jittorinfer_amd as J
        q = J.gqa_norm_rope(s["q"], s["k"], s["v"], s["pos"], q_weight=s["wq"], k_weight=s["wk"], eps=EPS, k_cache=s["k_cache"], v_cache=s["v_cache"],
                            block_table=s["block_table"], seq_ids=s["seq_ids"], slots=s["slots"], **s["rope"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    kv = s["k_cache"].dtype
    q = _normed_rotated(s["q"], s["wq"], s["rope"], s["pos"]).to(kv)
    slots = s["slots"].long()
    page = s["block_table"][s["seq_ids"].long(), slots // PAGE].long()
    s["k_cache"][page, slots % PAGE] = _normed_rotated(s["k"], s["wk"], s["rope"], s["pos"]).to(kv)
    s["v_cache"][page, slots % PAGE] = s["v"].to(kv)
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _rows(s):
    """Row number of every key a sequence may have [1, n], its page [n_seq, n], and which of them attend."""
    table, lens = s["block_table"], s["seq_lens"][:, None]
    t = torch.arange(table.shape[1] * PAGE, device=table.device)[None]
    live = t < lens
    if s.get("window"):
        live = live & (t >= lens - s["window"])
    return t, table.long().repeat_interleave(PAGE, 1), live


def _run_attn(s):
    if own:
        import jittorinfer_amd as J
        out = J.gqa_attn(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["seq_lens"], scale=s["scale"], logit_softcap=s["softcap"], window=s["window"],
                         mask=s["row_mask"], weights=s["sums"])
        return {"out": out if s["dv"] else None, "weights": s["sums"]}
    t, page, live = _rows(s)
    n_seq, kv_heads = s["n_seq"], s["kv_heads"]
    k = s["k_cache"][page, t % PAGE].transpose(1, 2).float()                     # [n_seq, kv_heads, n, dk]
    q = s["q"].float().view(n_seq, kv_heads, -1, s["dk"])
    score = torch.matmul(q, k.transpose(2, 3)) * s["scale"]                      # [n_seq, kv_heads, group, n]
    if s["softcap"]:
        score = s["softcap"] * torch.tanh(score / s["softcap"])
    if s["row_mask"] is not None:
        score = score + s["row_mask"].float()[:, None, None]
    score = torch.where(live[:, None, None], score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-38)
    if s["sums"] is not None:
        s["sums"] += p.sum(2)
    if not s["dv"]:
        return {"out": None, "weights": s["sums"]}
    v = s["v_cache"][page, t % PAGE].transpose(1, 2).float()
    out = torch.matmul(p, v).reshape(n_seq, s["heads"], s["dv"]).to(s["q"].dtype)
    return {"out": out, "weights": s["sums"]}


def _run_evict(s):
    if own:
        import jittorinfer_amd as J
        kept, lens, sums = J.gqa_evict(s["sums"], s["block_table"], s["seq_lens"], s["k_cache"], s["v_cache"], n_keep=s["keep"], n_sink=s["sink"], n_recent=s["recent"])
        return {"kept": kept, "lens": lens, "weights": sums, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    t, page, live = _rows(s)
    n_seq, kv_heads, n = s["sums"].shape
    lens = s["seq_lens"][:, None]
    keep = min(s["keep"], n)
    # the first and the last rows stay whatever their weight; among equals the lower row stays
    held = (t < s["sink"]) | (t >= lens - s["recent"])
    key = torch.where(held[:, None], float("inf"), s["sums"])
    key = torch.where(live[:, None], key, float("-inf"))
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.sort(best, dim=-1).values                                       # in the order of the rows
    new_lens = torch.minimum(s["seq_lens"], torch.full_like(s["seq_lens"], keep))
    slot = torch.arange(keep, device=kept.device)
    stays = slot[None] < new_lens[:, None]
    kept = torch.where(lens[:, None] <= keep, slot[None, None], kept)
    sums = torch.zeros_like(s["sums"])
    sums[..., :keep] = torch.where(stays[:, None], torch.gather(s["sums"], 2, kept), 0.0)
    # rows that move: to a slot of the same sequence from a later row
    b, h, i = torch.nonzero(stays[:, None] & (kept != slot), as_tuple=True)
    src = kept[b, h, i]
    table = s["block_table"].long()
    to, by = table[b, i // PAGE], table[b, src // PAGE]
    s["k_cache"][to, i % PAGE, h] = s["k_cache"][by, src % PAGE, h]
    if s["v_cache"] is not None:
        s["v_cache"][to, i % PAGE, h] = s["v_cache"][by, src % PAGE, h]
    kept = torch.where(stays[:, None], kept, -1)
    if keep < s["keep"]:
        kept = torch.nn.functional.pad(kept, (0, s["keep"] - keep), value=-1)
    return {"kept": kept.to(torch.int32), "lens": new_lens, "weights": sums, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    e = 2
    row = c["kv_heads"] * (c["dk"] + c["dv"]) * e
    if c["op"] == "norm_rope":
        heads = c["heads"] * c["dk"] + c["kv_heads"] * (c["dk"] + c["dv"])
        src = {"f32": 4, "bf16": 2, "f16": 2}[c["src"]]
        return {"bytes": c["n_tok"] * (heads * (src + e) + 12) + LOWEST_COST, "flops": c["n_tok"] * heads * 8}
    # sequences are as long as the seed makes them: the mean
    mean = (c["hi"] + (c["n_seq"] - 1) * (c["lo"] + c["hi"]) / 2) / c["n_seq"]
    if c["op"] == "attn":
        keys = min(mean, c["window"]) if c["window"] else mean
        moved = keys * row + c["heads"] * (c["dk"] + c["dv"]) * e + (keys * 2 if c["mask"] else 0) + (keys * c["kv_heads"] * 8 if c["weights"] else 0)
        return {"bytes": c["n_seq"] * moved + LOWEST_COST, "flops": c["n_seq"] * keys * c["heads"] * 2 * (c["dk"] + c["dv"])}
    kept = min(c["keep"], mean)
    shut = (c["keep"] - c["lo"]) / (c["hi"] - c["lo"]) if c["hi"] > c["lo"] else 0.0     # the share of sequences that stay as they are
    moving = (1.0 - min(1.0, max(0.0, shut))) * max(0, kept - c["sink"])
    width = (c["hi"] + PAGE - 1) // PAGE * PAGE
    return {"bytes": c["n_seq"] * (moving * row * 2 + c["kv_heads"] * (mean * 4 + kept * 4 + width * 4)) + LOWEST_COST, "flops": c["n_seq"] * c["kv_heads"] * mean}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"norm_rope": _exact_norm_rope, "attn": _exact_attn, "evict": _exact_evict}[case["op"]](s)


def _exact_heads(x, w, r, pos):
    """Channel by channel as complex numbers: a rotated pair is its number times e^(i angle)."""
    x = x.double()
    if w is not None:
        x = w.double() * x / torch.sqrt(torch.sum(x ** 2, -1, keepdim=True) / x.shape[-1] + EPS)
    n, base, half = r["n_dims"], r["freq_base"], r["n_dims"] // 2
    first = list(range(half)) if r["mode"] == 2 else list(range(0, n, 2))
    step = half if r["mode"] == 2 else 1
    out = x.clone()
    mag = r.get("attn_factor", 1.0)
    if r.get("ext_factor", 0.0):
        mag *= 1.0 + 0.1 * math.log(1.0 / r["freq_scale"])
    for i, at in enumerate(first):
        turn = r.get("freq_scale", 1.0)
        if r.get("ext_factor", 0.0):
            lo = max(0, math.floor(n * math.log(r["n_ctx_orig"] / (64 * math.pi)) / (2 * math.log(base))))
            hi = min(n - 1, math.ceil(n * math.log(r["n_ctx_orig"] / (2 * math.pi)) / (2 * math.log(base))))
            mix = (1.0 - min(1.0, max(0.0, (i - lo) / max(0.001, hi - lo)))) * r["ext_factor"]
            turn = turn * (1.0 - mix) + mix
        angle = pos.double() * (turn * base ** (-2.0 * i / n))
        z = torch.complex(x[..., at], x[..., at + step]) * (mag * torch.polar(torch.ones_like(angle), angle))[:, None]
        out[..., at], out[..., at + step] = z.real, z.imag
    return out


def _exact_norm_rope(s):
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    k = _exact_heads(s["k"], s["wk"], s["rope"], s["pos"])
    for b in range(s["n_seq"]):
        mine = torch.nonzero(s["seq_ids"] == b)[:, 0]
        slot = s["slots"][mine].long()
        page = s["block_table"][b].long()[slot // PAGE]
        k_cache[page, slot % PAGE] = k[mine]
        v_cache[page, slot % PAGE] = s["v"][mine].double()
    return {"q": _exact_heads(s["q"], s["wq"], s["rope"], s["pos"]), "k_cache": k_cache, "v_cache": v_cache}


def _exact_attn(s):
    group = s["heads"] // s["kv_heads"]
    out = torch.zeros((s["n_seq"], s["heads"], s["dv"]), dtype=torch.float64, device=s["q"].device)
    sums = s["sums"].double() if s["sums"] is not None else None
    for b, n in enumerate(s["seq_lens"].tolist()):
        first = max(0, n - s["window"]) if s["window"] else 0
        at = torch.arange(first, n, device=out.device)
        page = s["block_table"][b].long()[at // PAGE]
        for g in range(s["kv_heads"]):
            k = s["k_cache"][page, at % PAGE, g].double()
            score = k @ s["q"][b, g * group:(g + 1) * group].double().T.contiguous() * s["scale"]    # [keys, group]
            if s["softcap"]:
                score = torch.tanh(score / s["softcap"]) * s["softcap"]
            if s["row_mask"] is not None:
                score = score + s["row_mask"][b, at].double()[:, None]
            p = torch.softmax(score, 0).nan_to_num(0.0)      # no row left by the mask: no weight anywhere
            if sums is not None:
                sums[b, g, at] += p.sum(1)
            if s["dv"]:
                out[b, g * group:(g + 1) * group] = p.T.contiguous() @ s["v_cache"][page, at % PAGE, g].double()
    return {"out": out if s["dv"] else None, "weights": sums}


def _exact_evict(s):
    """Kept rows by ranking: a row stays when fewer than the free places go to rows of more weight, or of the same weight and a lower number."""
    k_cache, v_cache = s["k_cache"].clone(), s["v_cache"].clone() if s["v_cache"] is not None else None
    sums = torch.zeros_like(s["sums"])
    for b, n in enumerate(s["seq_lens"].tolist()):
        table = s["block_table"][b].long()
        for h in range(s["kv_heads"]):
            rows = torch.arange(n, device=sums.device)
            if n > s["keep"]:
                first, last = min(s["sink"], n), max(min(s["sink"], n), n - s["recent"])
                w = s["sums"][b, h, first:last].double()
                places = max(0, s["keep"] - first - (n - last))
                order = torch.argsort(-w, stable=True)[:places]
                rows = torch.cat((rows[:first], rows[first:last][order].sort().values, rows[last:]))
            to = torch.arange(rows.shape[0], device=sums.device)
            k_cache[table[to // PAGE], to % PAGE, h] = s["k_cache"][table[rows // PAGE], rows % PAGE, h]
            if v_cache is not None:
                v_cache[table[to // PAGE], to % PAGE, h] = s["v_cache"][table[rows // PAGE], rows % PAGE, h]
            sums[b, h, to] = s["sums"][b, h, rows]
    return {"kept": None, "lens": None, "weights": sums, "k_cache": k_cache, "v_cache": v_cache}
