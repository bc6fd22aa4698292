"""The paged cache of ordinary heads on the GPU, at its edges: weights bit by bit, caps of any size, streams of the caller, and shapes that only one rule reaches."""
import math

import pytest
import torch

from tests import gqa_util as R
from tests.test_gqa_gpu import BF16, F16, F32, WIDTHS, _attn_case, _check_attn, _check_evict, _check_rows, _near

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -24


def _exact_scores_case(n, width, heads, kv_heads, dk, dv, dtype, seed=0, step=-1 / 64):
    """One sequence whose scores are known exactly (a query of one 1, keys of one number t = j * step, j <= 60, scale 1), whose row i has its weight to itself in column
    i of dv or fewer: V is one-hot, so a result is the sum of few weights and nothing else."""
    gen = torch.Generator().manual_seed(seed)
    q, k, v, bt, lens = _attn_case(seed, [n], width, heads, kv_heads, dk, dv, dtype)
    at = torch.arange(n)
    page, row = bt[0].long()[at // 128], at % 128
    t = torch.randint(0 if step < 0 else -60, 61, (n,), generator=gen).double() * step
    q.zero_()
    q[..., 0] = 1
    k[page, row] = 0
    k[page, row, :, 0] = t.to(dtype)[:, None]
    if dv:
        v[page, row] = 0
        v[page, row, :, at % dv] = 1
    return q, k, v, bt, lens, t


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dk,dv", WIDTHS)
@pytest.mark.parametrize("heads,kv_heads,width", [(4, 2, 2), (8, 8, 256), (40, 2, 1024)])     # one block of heads, four KV heads a workgroup, two blocks
@pytest.mark.parametrize("n", [64, 128, 250])
def test_attn_weights_of_single_rows(gpu, dtype, dk, dv, heads, kv_heads, width, n):
    """Every weight as the second product takes it, in an f32 result: 32-bit rounding, not that of 16-bit parts."""
    import jittorinfer_amd as J
    q, k, v, bt, lens, t = _exact_scores_case(n, width, heads, kv_heads, dk, dv, dtype)
    p = torch.softmax(t, 0)
    want = torch.zeros(dv, dtype=torch.float64).index_add_(0, torch.arange(n) % dv, p)
    got = J.gqa_attn(*(x.to(gpu) for x in (q, k, v, bt, lens)), scale=1.0, out=torch.empty((1, heads, dv), dtype=F32, device=gpu)).cpu().double()
    # Beside the heaviest column, so that the sum's own roundings cancel.  |t| < 1: its log2 form and its distance to the maximum are three roundings of less than 2,
    # exp2 is off by 2 half steps; the weight's parts by 2^-22; joins, reciprocal and product by 2 half steps each, a column of several rows by 1 each; in either
    got, want = got / got[..., want.argmax()][..., None], want / want.max()
    rel = 2 * ((3 * 2 + 2) * EPS32 + 2.0 ** -22 + (6 + math.ceil(n / dv)) * EPS32)
    assert n > 128 or rel < 2.0 ** -18.6               # (weights as two bf16 parts are off by 2^-17.5)
    bad = (got - want).abs() > rel * want
    assert not bad.any(), "%d of %d, worst %.3g of its bound" % (int(bad.sum()), bad.numel(), float(((got - want).abs() / (rel * want).clamp_min(1e-300)).max()))


CAPS = [1e-38, 1e-3, 0.5, 5.0, 20.0, 50.0, 1e3, 1e6, 1e7, 1e8, 1e30, 3e38]


@pytest.mark.parametrize("dk,dv", [(64, 64), (576, 0)])
@pytest.mark.parametrize("step", [1 / 64, 1 / 8])
@pytest.mark.parametrize("cap", CAPS)
def test_attn_softcap_of_any_size(gpu, cap, step, dk, dv):
    """A cap far above the scores leaves them as they are, one far below makes them equal: weights within 32-bit rounding of c tanh(s / c) for all of them."""
    import jittorinfer_amd as J
    n, heads = 64, 2
    q, k, v, bt, lens, t = _exact_scores_case(n, 2, heads, 1, dk, dv, BF16, step=step)
    s = cap * torch.tanh(t / cap)
    p = torch.softmax(s, 0)
    sums = torch.zeros((1, 1, 256), device=gpu)
    out = torch.empty((1, heads, dv), dtype=F32, device=gpu) if dv else None
    J.gqa_attn(*(x.to(gpu) if x is not None else None for x in (q, k, v, bt, lens)), scale=1.0, logit_softcap=cap, weights=sums, out=out)
    # a capped score is off by 2^-21 of itself (a quotient's reciprocal and exp2 are 2 half steps each, four products and sums), its log2 form and the distance to the
    # maximum by three half steps more; twice, in the weight and in the one it is compared with; exp2, parts, sum over two heads, joins as above
    size = float(s.abs().max())
    rel = 2 * (size * (8 + 2 * 3) + 2 + 4 + 7 + 2) * EPS32
    for what, got in (("weights", sums[0, 0, :n]), ("out", out[0])) if dv else (("weights", sums[0, 0, :n]),):
        got = got.cpu().double()
        got = got / got[..., p.argmax()][..., None]
        bad = (got - p / p.max()).abs() > rel * p / p.max()
        assert not bad.any(), "%s: %d of %d, worst %.3g of its bound" % (what, int(bad.sum()), bad.numel(), float(((got - p / p.max()).abs() / (rel * p / p.max())).max()))
    assert abs(float(sums.double().sum()) - heads) < heads * (n + 10) * EPS32 and (sums[0, 0, n:] == 0).all()


@pytest.mark.parametrize("scale", [-0.125, 1e-6, 30.0])
def test_attn_softcap_with_other_scales(gpu, scale):
    """Scores of either sign from a negative scale, all far below the cap, and all at it."""
    import jittorinfer_amd as J
    q, k, v, bt, lens = _attn_case(50, [200, 1], 2, 4, 2, 64, 64, F16)
    out, off, w, w_off = R.attn(q, k, v, bt, lens.tolist(), scale, 30.0)
    sums = torch.zeros((2, 2, 256), device=gpu)
    got = J.gqa_attn(*(x.to(gpu) for x in (q, k, v, bt, lens)), scale=scale, logit_softcap=30.0, weights=sums)
    _near(got, out, off, F16)
    _near(sums, w, w_off, F32)


def test_scratch_of_another_stream_is_not_this_ones(gpu):
    """A stream's first area is no block that the allocator keeps for work queued on the current stream."""
    from jittorinfer_amd import capi
    size = 96 << 20
    side = torch.cuda.Stream()
    old = torch.empty(size, dtype=torch.uint8, device=gpu)
    held = old.data_ptr()
    del old                                                           # free again, to the current stream's later work
    ws = capi._workspace(gpu, size, side.cuda_stream)
    again = torch.empty(size, dtype=torch.uint8, device=gpu)
    assert again.data_ptr() == held and ws.data_ptr() != held
    capi.release_workspaces(side.cuda_stream, gpu)


def test_forked_branches_of_one_capture(gpu):
    """Calls on the current stream and, through stream=, on a side stream of the same capture run side by side at every replay: neither uses the other's scratch."""
    import jittorinfer_amd as J
    cases = [[t.to(gpu) for t in _attn_case(51 + i, [1024, 600, 1000, 128 + i], 8, 8, 2, 128, 128, BF16)] for i in range(4)]
    want = [J.gqa_attn(*c, scale=0.1) for c in cases]
    outs = [torch.empty_like(w) for w in want]
    sums = [torch.zeros((4, 2, 1024), device=gpu) for _ in cases]
    want_sums = [torch.zeros_like(s) for s in sums]
    for c, s in zip(cases, want_sums):
        J.gqa_attn(*c, scale=0.1, weights=s)
    cut = _evict_on(gpu, 60)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fork = torch.cuda.Event()
        fork.record()
        side.wait_event(fork)
        for i, c in enumerate(cases):
            J.gqa_attn(*c, scale=0.1, weights=sums[i], out=outs[i], stream=side.cuda_stream if i % 2 else None)
        cut["run"](stream=side.cuda_stream)
        torch.cuda.current_stream().wait_stream(side)
    for step in range(4):
        for o, s in zip(outs, sums):
            o.fill_(float("nan"))
            s.zero_()
        cut["reset"]()
        J.gqa_attn(*cases[0], scale=0.1)                               # eager work between the replays
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)) and all(torch.equal(a, b) for a, b in zip(sums, want_sums)), step
        cut["check"]()


def _evict_on(gpu, seed):
    """An eviction with its results made ahead: run(stream=), reset() and check() against the plain form."""
    import jittorinfer_amd as J
    from tests.test_gqa_gpu import _evict_case
    w, bt, lens, k, v = _evict_case(seed, [700, 1000, 90], 8, 2, 64, 64, BF16)
    want = R.evict(w, bt, lens.tolist(), k, v, 300, 4, 30)
    d = [t.to(gpu) for t in (w, bt, lens, k, v)]
    outs = dict(weights_out=torch.empty_like(d[0]), kept=torch.empty((3, 2, 300), dtype=torch.int32, device=gpu), new_lens=torch.empty(3, dtype=torch.int32, device=gpu))

    def check():
        assert torch.equal(outs["kept"].cpu(), want[0]) and torch.equal(outs["new_lens"].cpu(), want[1]) and torch.equal(outs["weights_out"].cpu(), want[2])
        assert torch.equal(R.bits(d[3].cpu()), R.bits(want[3])) and torch.equal(R.bits(d[4].cpu()), R.bits(want[4]))
    return dict(run=lambda **kw: J.gqa_evict(*d, n_keep=300, n_sink=4, n_recent=30, **outs, **kw), check=check, reset=lambda: (d[3].copy_(k), d[4].copy_(v)))


def test_calls_on_a_captured_stream_that_is_not_the_current_one(gpu):
    """A capture on one stream, the call made while another is the current one: scratch is the graph's, not the area that eager calls of the stream share."""
    import jittorinfer_amd as J
    from jittorinfer_amd import capi
    c = [t.to(gpu) for t in _attn_case(55, [1024, 600], 8, 8, 2, 128, 128, F16)]
    want, out = J.gqa_attn(*c, scale=0.1), torch.empty((2, 8, 128), dtype=F16, device=gpu)
    inner, other = torch.cuda.Stream(), torch.cuda.Stream()
    capi.release_workspaces(inner.cuda_stream, gpu)                   # (streams come from a pool: this one may have had calls before)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=inner):
        with torch.cuda.stream(other):
            J.gqa_attn(*c, scale=0.1, out=out, stream=inner.cuda_stream)
    assert (gpu, inner.cuda_stream) not in capi._workspaces
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_side_stream_calls_without_waiting(gpu):
    """Eager calls on a side stream through stream=, ordered by events alone, while the current stream goes on allocating."""
    import jittorinfer_amd as J
    c = [t.to(gpu) for t in _attn_case(56, [1024, 600, 30], 8, 8, 2, 128, 128, BF16)]
    want = J.gqa_attn(*c, scale=0.1)
    outs = [torch.empty_like(want) for _ in range(20)]
    cuts = _evict_on(gpu, 61)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for i, out in enumerate(outs):
        J.gqa_attn(*c, scale=0.1, out=out, stream=side.cuda_stream)
        torch.full((1 << 20,), float(i), device=gpu).add_(1.0)
        assert torch.equal(J.gqa_attn(*c, scale=0.1), want)
    cuts["run"](stream=side.cuda_stream)
    side.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    cuts["check"]()


@pytest.mark.parametrize("heads,dk,dv", [(2, 32, 16), (5, 16, 16), (8, 16, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_many_heads_selected_by_several_workgroups(gpu, heads, dk, dv, in_place):
    """Block tables of more than 24576 rows with several KV heads, K and V with room between their heads and rows, weights with room between theirs; lengths that end
    inside a run of 8192, at its end, and below what is kept; sinks and recent rows that fill whole runs."""
    import jittorinfer_amd as J
    from tests.test_gqa_gpu import _evict_case
    lens, width = [33000, 24577, 16384, 9000, 100], 260
    assert len(lens) * heads <= 64                        # (as many groups as the rule takes)
    w, bt, lens, k, v = _evict_case(70 + heads, lens, width, heads, dk, dv, BF16)
    w[0, 0] = 1.0                                         # one head all ties
    gen = torch.Generator().manual_seed(heads)
    w[1, -1] = torch.randint(0, 3, (width * 128,), generator=gen).float()
    for n_keep, n_sink, n_recent in ((9000, 4, 500), (20000, 8200, 9000), (24576, 0, 0)):
        want = R.evict(w, bt, lens.tolist(), k, v, n_keep, n_sink, n_recent)
        kk = torch.full((k.shape[0], 128, heads, dk + 8), 3.0, dtype=BF16, device=gpu)
        kk[..., :dk] = k.to(gpu)
        vv = None
        if dv:
            vv = torch.full((v.shape[0], 130, heads + 1, dv), 3.0, dtype=BF16, device=gpu)
            vv[:, :128, :heads] = v.to(gpu)
        ww = torch.full((len(lens), heads + 1, width * 128 + 12), 7.0, device=gpu)
        ww[:, :heads, 4:4 + width * 128] = w.to(gpu)
        ws = ww[:, :heads, 4:4 + width * 128]
        kept, new, out = J.gqa_evict(ws, bt.to(gpu), lens.to(gpu), kk[..., :dk], vv[:, :128, :heads] if dv else None, n_keep=n_keep, n_sink=n_sink, n_recent=n_recent,
                                     weights_out=ws if in_place else None)
        torch.cuda.synchronize()
        assert torch.equal(kept.cpu(), want[0]) and torch.equal(new.cpu(), want[1]), (n_keep, n_sink)
        assert torch.equal(out.cpu(), want[2])
        assert torch.equal(kk[..., :dk].cpu(), want[3]) and (kk[..., dk:] == 3).all()
        if dv:
            assert torch.equal(vv[:, :128, :heads].cpu(), want[4]) and (vv[:, 128:] == 3).all() and (vv[:, :, heads:] == 3).all()
        assert (ww[:, heads:] == 7).all() and (ww[..., :4] == 7).all() and (ww[..., 4 + width * 128:] == 7).all()
        assert in_place or torch.equal(ws.cpu(), w)


@pytest.mark.parametrize("n_sink,n_recent", [(3000, 100), (100, 3000), (2000, 2000)])
def test_evict_in_place_of_held_rows(gpu, n_sink, n_recent):
    """Weights of rows that stay whatever they weigh move down over rows that other threads hold: one workgroup a group, one chunk and two."""
    from tests.test_gqa_gpu import _evict_case
    for width, n in ((40, 5000), (190, 24000)):
        w, bt, lens, k, _ = _evict_case(80, [n, n - 37], width, 2, 16, 0, BF16)
        for n_keep in (4000, n - 40):
            _check_evict(gpu, w, bt, lens, k, None, n_keep, n_sink, n_recent, in_place=True)


@pytest.mark.parametrize("heads", [1, 16, 40, 128])
def test_weights_of_many_pages_a_unit(gpu, heads):
    """A latent cache's running maxima and sums, handed from page to page of a unit."""
    _check_attn(gpu, *_attn_case(81, [2500, 2177, 300], 20, heads, 1, 576, 0, BF16), n_workgroups=4)


def test_evict_keeps_as_many_as_there_may_be(gpu):
    """n_keep of 2^31 - 1: nothing leaves, every place past the length is marked."""
    import jittorinfer_amd as J
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    w, n = torch.rand((1, 1, 256), device=gpu), 200
    k = torch.rand((2, 128, 1, 16), device=gpu).to(BF16)
    before = k.clone()
    kept, new, out = J.gqa_evict(w, torch.tensor([[1, 0]], dtype=torch.int32, device=gpu), torch.tensor([n], dtype=torch.int32, device=gpu), k, n_keep=2 ** 31 - 1)
    torch.cuda.synchronize()
    assert kept.shape == (1, 1, 2 ** 31 - 1) and new.tolist() == [n] and torch.equal(k, before)
    assert torch.equal(kept[0, 0, :n].cpu(), torch.arange(n, dtype=torch.int32)) and int(kept[0, 0, n:].max()) == -1 == int(kept[0, 0, n:].min())
    assert torch.equal(out[..., :n], w[..., :n]) and (out[..., n:] == 0).all()


@pytest.mark.parametrize("kind", ["spread", "late", "alternate"])
def test_evict_moves_many_segments(gpu, kind):
    """A segment a row, more of them than 63 a thread: rows that come from near and far, from the end alone, and every other one."""
    import jittorinfer_amd as J
    width, n, n_keep = 320, 40900, 33000
    gen = torch.Generator().manual_seed(82)
    w = torch.rand((1, 1, width * 128), generator=gen)
    if kind == "late":
        w[..., n - n_keep:n] += 2
    elif kind == "alternate":
        w[..., :2 * (n - n_keep):2] -= 2
    bt = torch.randperm(width, generator=gen).to(torch.int32)[None]
    # rows of 16384 bytes, 4 apart: every 4-byte number says which row and which place of it it is
    store = torch.zeros((width, 128, 1, 4097), dtype=torch.int32, device=gpu)
    k = store[..., :4096]
    row = torch.arange(width * 128, device=gpu, dtype=torch.int32)
    page = bt[0].to(gpu).long()
    def pattern(rows):
        return rows[:, None] * 4096 + torch.arange(4096, device=gpu, dtype=torch.int32)[None]
    for j in range(width):
        k[page[j], :, 0] = pattern(row[j * 128:(j + 1) * 128])
    kept, new, out = J.gqa_evict(w.to(gpu), bt.to(gpu), torch.tensor([n], dtype=torch.int32, device=gpu), k, n_keep=n_keep, n_sink=2, n_recent=10)
    key = w[0, 0, :n].clone()
    key[:2], key[n - 10:] = 9, 9
    want = torch.sort(torch.sort(key, descending=True, stable=True).indices[:n_keep]).values.to(gpu)
    assert torch.equal(kept[0, 0].long(), want) and new.tolist() == [n_keep]
    held = torch.cat((want.int(), row[n_keep:]))
    for j in range(width):
        assert torch.equal(k[page[j], :, 0], pattern(held[j * 128:(j + 1) * 128])), j
    assert (store[..., 4096] == 0).all()


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_takes_weights_as_wide_as_attention_does(gpu, in_place):
    """Sums with room for more rows than the block table has: the columns past it stay."""
    import jittorinfer_amd as J
    from tests.test_gqa_gpu import _evict_case
    w, bt, lens, k, v = _evict_case(83, [300, 384], 3, 2, 64, 64, F16)
    wide = torch.full((2, 2, 512), 7.0, device=gpu)
    wide[..., :384] = w.to(gpu)
    want = R.evict(w, bt, lens.tolist(), k, v, 140, 2, 10)
    dst = wide if in_place else torch.full((2, 2, 500), 8.0, device=gpu)
    d = [t.to(gpu) for t in (bt, lens, k, v)]
    kept, new, out = J.gqa_evict(wide, *d, n_keep=140, n_sink=2, n_recent=10, weights_out=dst)
    assert out is dst and torch.equal(kept.cpu(), want[0]) and torch.equal(dst[..., :384].cpu(), want[2]) and (dst[..., 384:] == (7 if in_place else 8)).all()
    assert torch.equal(d[2].cpu(), want[3]) and torch.equal(d[3].cpu(), want[4])
    if not in_place:
        d = [t.to(gpu) for t in (bt, lens, k, v)]
        assert J.gqa_evict(wide, *d, n_keep=140)[2].shape == (2, 2, 384)


def test_strides_of_dimensions_of_one(gpu):
    """One token, one sequence, one head, one page: where there is no next one, the stride to it is any number."""
    import jittorinfer_amd as J
    from tests.test_gqa_gpu import _evict_case
    odd = lambda t, *dims: t.as_strided(t.shape, [13 if d in dims else s for d, s in enumerate(t.stride())])
    q, k, v, bt, lens = (t.to(gpu) for t in _attn_case(90, [100], 1, 3, 1, 64, 64, BF16, spare=0, stale=0.0))
    want, sums = J.gqa_attn(q, k, v, bt, lens, scale=0.1), torch.zeros((1, 1, 128), device=gpu)
    J.gqa_attn(q, k, v, bt, lens, scale=0.1, weights=sums)
    out, got = torch.empty_like(want), torch.zeros_like(sums)
    J.gqa_attn(odd(q, 0), odd(k, 0, 2), odd(v, 0, 2), bt, lens, scale=0.1, weights=odd(got, 0, 1), out=odd(out, 0))
    assert torch.equal(out, want) and torch.equal(got, sums)
    one = q[:, :1].contiguous()
    assert torch.equal(J.gqa_attn(odd(one, 0, 1), k, v, bt, lens, scale=0.1), want[:, :1])
    pos, ids = torch.tensor([7], dtype=torch.int32, device=gpu), torch.zeros(1, dtype=torch.int32, device=gpu)
    kc, vc, kc2, vc2 = k.clone(), v.clone(), k.clone(), v.clone()
    x = torch.randn((1, 1, 64), device=gpu).to(BF16)
    rope = dict(n_dims=64, mode=2, block_table=bt, seq_ids=ids)
    want = J.gqa_norm_rope(q, x, x, pos, k_cache=kc, v_cache=vc, **rope)
    got = torch.empty_like(want)
    J.gqa_norm_rope(odd(q, 0), odd(x, 0, 1), odd(x, 0, 1), pos, k_cache=odd(kc2, 0, 2), v_cache=odd(vc2, 0, 2), q_out=odd(got, 0), **rope)
    assert torch.equal(got, want) and torch.equal(kc, kc2) and torch.equal(vc, vc2)
    w = torch.rand((1, 1, 128), device=gpu)
    kept, new, moved = J.gqa_evict(w, bt, lens, kc, vc, n_keep=30)
    kept2, new2, moved2 = J.gqa_evict(odd(w, 0, 1), bt, lens, odd(kc2, 0, 2), odd(vc2, 0, 2), n_keep=30, weights_out=odd(torch.empty_like(w), 0, 1))
    assert torch.equal(kept, kept2) and torch.equal(moved, moved2) and torch.equal(kc, kc2) and torch.equal(vc, vc2)


def _shares(call, *args, **kw):
    with pytest.raises(RuntimeError, match="share memory|failed with code -6"):
        call(*args, **kw)


def test_results_on_operands_are_refused(gpu):
    """What a call writes may not lie on what it reads; views of one buffer that share no byte may."""
    import jittorinfer_amd as J
    z = lambda *s, dtype=BF16: torch.zeros(s, dtype=dtype, device=gpu)
    i = lambda *s: z(*s, dtype=torch.int32)
    buf, kv, bt, lens = z(4, 10, 64), z(3, 128, 4, 64), i(4, 2), i(4)
    q, k, v, sums = buf[:, :4], kv[:, :, :2], kv[:, :, 2:], z(4, 2, 300, dtype=F32)
    attn = dict(q=q, k_cache=k, v_cache=v, block_table=bt, seq_lens=lens, scale=1.0)
    J.gqa_attn(**attn, out=buf[:, 4:8], weights=sums)
    for out in (q, buf[:, 1:5], buf[:, 3:7], kv[2, :16].view(4, 4, 4, 64)[:, :, 0], sums.view(torch.uint8).view(-1)[:2048].view(BF16).view(4, 4, 64)):
        _shares(J.gqa_attn, **attn, out=out, weights=sums)
    bytes_of = lambda t: t.contiguous().view(-1).view(torch.uint8)
    _shares(J.gqa_attn, **attn, weights=bytes_of(kv)[:4 * 2 * 256 * 4].view(F32).view(4, 2, 256))
    mask = z(4, 256 * 2, dtype=F16)
    wide = z(4, 2, 256, dtype=F32)
    _shares(J.gqa_attn, **attn, weights=wide, mask=wide.view(-1).view(F16)[:1024].view(4, 256))
    assert not buf.any() and not kv.any() and not mask.any()

    pos, ids = i(4), i(4)
    qkv = z(4, 12, 64)
    rows = dict(q=qkv[:, :4], k=qkv[:, 8:10], v=qkv[:, 10:], pos=pos, n_dims=64, k_cache=k, v_cache=v, block_table=bt, seq_ids=ids)
    J.gqa_norm_rope(**rows, q_out=qkv[:, 4:8])
    J.gqa_norm_rope(**rows, q_out=qkv[:, :4])
    for out in (qkv[:, 1:5], qkv[:, 5:9], qkv[:, 7:11], kv[0, :4]):
        _shares(J.gqa_norm_rope, **rows, q_out=out)
    for name, other in (("v_cache", kv[:, :, 1:3]), ("v_cache", k), ("k_cache", kv[:, :, 1:3])):
        _shares(J.gqa_norm_rope, **{**rows, name: other})

    w = z(5, 4, 256, dtype=F32)
    cut = dict(weights=w[:4, :2], block_table=bt, seq_lens=lens, k_cache=k, v_cache=v, n_keep=20)
    J.gqa_evict(**cut, weights_out=w[:4, 2:])
    J.gqa_evict(**cut, weights_out=w[:4, :2])
    for out in (w[1:5, :2], w[:4, 1:3]):
        _shares(J.gqa_evict, **cut, weights_out=out)
    both = i(4 * 2 * 20 + 4)
    J.gqa_evict(**cut, kept=both[:160].view(4, 2, 20), new_lens=both[160:])
    _shares(J.gqa_evict, **cut, kept=both[:160].view(4, 2, 20), new_lens=both[157:161])
    _shares(J.gqa_evict, **cut, new_lens=bt.view(-1)[2:6])
    _shares(J.gqa_evict, **{**cut, "v_cache": kv[:, :, 1:3]})
    _shares(J.gqa_evict, **{**cut, "k_cache": kv[:, :, 1:3]})


# ---------------------------------------------------------------- the prompt form of norms and rotation: a workgroup a token, four sets of rows ahead, from 1024 tokens on

@pytest.mark.parametrize("src,kv", [(F32, BF16), (F32, F16), (BF16, BF16), (BF16, F16), (F16, F16), (F16, BF16)])
@pytest.mark.parametrize("dk,dv", [(64, 64), (72, 40), (128, 128), (256, 256)])
def test_norm_rope_prompts(gpu, src, kv, dk, dv):
    for n_tok, n_head, n_head_kv, mode in ((1023, 4, 1, 0), (1024, 3, 2, 2), (1025, 5, 2, 0)):
        _check_rows(gpu, src, kv, n_tok, n_head, n_head_kv, dk, dv, n_dims=dk // 16 * 16, mode=mode, w_type=src, out_type=F32 if n_tok == 1024 else None, seed=dk)


@pytest.mark.parametrize("n_head,n_head_kv,dk", [(64, 2, 128), (66, 1, 128), (128, 1, 64), (39, 2, 256), (33, 8, 192), (160, 4, 64), (64, 0, 128)])
@pytest.mark.parametrize("in_place", [False, True])
def test_norm_rope_prompts_of_many_rows(gpu, n_head, n_head_kv, dk, in_place):
    """More than the four sets of rows that are under way at once; a last set that is not full, one that holds queries and keys; in place."""
    if n_head_kv:
        _check_rows(gpu, BF16, BF16, 1100, n_head, n_head_kv, dk, 64, n_dims=dk, mode=2, in_place=in_place, seed=n_head)
        _check_rows(gpu, BF16, BF16, 1030, n_head, n_head_kv, dk, 64, "heads", n_dims=32, mode=0, in_place=in_place, norm=False, seed=n_head)
    else:
        import jittorinfer_amd as J
        gen = torch.Generator().manual_seed(1)
        q, w, pos = torch.randn((1024, n_head, dk), generator=gen), torch.rand(dk, generator=gen) + 0.5, torch.arange(1024, dtype=torch.int32)
        want, off = R.heads(q, w, 1e-6, pos, dk, 2)
        d = q.to(gpu)
        got = J.gqa_norm_rope(d, None, None, pos.to(gpu), n_dims=dk, mode=2, q_weight=w.to(gpu), q_out=d if in_place else None)
        _near(got, want, off, F32)


@pytest.mark.parametrize("in_place", [False, True])
def test_norm_rope_few_tokens_of_many_rows(gpu, in_place):
    """More sets of rows than a token has workgroups (64): a workgroup takes several in turn."""
    _check_rows(gpu, BF16, BF16, 3, 600, 2, 256, 64, n_dims=256, mode=2, in_place=in_place)
    _check_rows(gpu, F32, F16, 2, 1030, 1, 128, 64, n_dims=64, mode=0, in_place=in_place)
    _check_rows(gpu, F32, BF16, 1040, 9, 3, 128, 128, n_dims=128, mode=2, in_place=in_place, past=70000)


@pytest.mark.parametrize("n_tok", [5, 1200])
@pytest.mark.parametrize("in_place", [False, True])
def test_norm_rope_of_heads_in_two_parts(gpu, n_tok, in_place):
    """Heads of 128 plain values with 64 rotated ones behind, those of the keys shared by all heads: a call for each part, on views of queries, results and cache."""
    import jittorinfer_amd as J
    from tests.test_gqa_gpu import YARN
    H, plain, turned, dv = 16, 128, 64, 128
    gen = torch.Generator().manual_seed(n_tok)
    q, kv, pe = (torch.randn(s, generator=gen).to(BF16) for s in ((n_tok, H, plain + turned), (n_tok, H, plain + dv), (n_tok, turned)))
    pos, ids = torch.arange(n_tok, dtype=torch.int32) // 2 + 3000, torch.arange(n_tok, dtype=torch.int32) % 2
    slots, width = torch.arange(n_tok, dtype=torch.int32) // 2, n_tok // 256 + 1
    bt = R.make_table(gen, [width * 128] * 2, width, 2 * width)
    kc, vc = (torch.full((2 * width, 128, H, d), 3.0, dtype=BF16, device=gpu) for d in (plain + turned, dv))
    dq, dkv, dpe = q.to(gpu), kv.to(gpu), pe.to(gpu)
    out = dq if in_place else torch.empty_like(dq)
    rope = dict(n_dims=turned, mode=0, **YARN)
    at = dict(block_table=bt.to(gpu), seq_ids=ids.to(gpu), slots=slots.to(gpu))
    J.gqa_norm_rope(dq[..., :plain], dkv[..., :plain], dkv[..., plain:], pos.to(gpu), n_dims=0, k_cache=kc[..., :plain], v_cache=vc, q_out=out[..., :plain], **at)
    J.gqa_norm_rope(dq[..., plain:], dpe[:, None].expand(n_tok, H, turned), None, pos.to(gpu), k_cache=kc[..., plain:], q_out=out[..., plain:], **rope, **at)
    want, off = R.heads(q[..., plain:], None, 0, pos, **rope)
    assert torch.equal(out[..., :plain].cpu(), q[..., :plain])
    _near(out[..., plain:], want, off, BF16)
    page, row = bt[ids.long(), slots.long() // 128].long(), slots.long() % 128
    want, off = R.heads(pe[:, None], None, 0, pos, **rope)
    got = kc.cpu()[page, row]
    assert torch.equal(got[..., :plain], kv[..., :plain]) and torch.equal(vc.cpu()[page, row], kv[..., plain:])
    _near(got[..., plain:], want.expand(n_tok, H, turned), off.expand(n_tok, H, turned), BF16)
    mark = torch.ones((2 * width, 128), dtype=torch.bool)
    mark[page, row] = False
    assert (kc.cpu()[mark] == 3).all() and (vc.cpu()[mark] == 3).all()


@pytest.mark.parametrize("n_tok", [7, 1100])
def test_norm_rope_in_a_graph_and_on_another_stream(gpu, n_tok):
    """Captured once, replayed while activations, positions and rows change under it; and launched through stream= with results of the caller's."""
    import jittorinfer_amd as J
    H, G, D, width = 6, 2, 128, n_tok // 128 + 2
    gen = torch.Generator().manual_seed(n_tok)
    wq, wk = (torch.rand(D, generator=gen) + 0.5 for _ in range(2))
    bt = R.make_table(gen, [width * 128], width, width)
    rope = dict(n_dims=D, mode=2, freq_base=10000.0)
    qkv, pos, slots = torch.empty((n_tok, H + 2 * G, D), dtype=BF16, device=gpu), torch.zeros(n_tok, dtype=torch.int32, device=gpu), torch.zeros(n_tok, dtype=torch.int32, device=gpu)
    ids, table, dwq, dwk = torch.zeros(n_tok, dtype=torch.int32, device=gpu), bt.to(gpu), wq.to(gpu), wk.to(gpu)
    kc, vc = (torch.empty((width, 128, G, D), dtype=BF16, device=gpu) for _ in range(2))
    out = torch.empty((n_tok, H, D), dtype=BF16, device=gpu)

    def call(**kw):
        J.gqa_norm_rope(qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:], pos, q_weight=dwq, k_weight=dwk, k_cache=kc, v_cache=vc, block_table=table, seq_ids=ids, slots=slots, q_out=out, **rope, **kw)
    qkv.zero_()
    torch.cuda.synchronize()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g):
        call()
    for step in range(4):
        x, p, r = torch.randn(qkv.shape, generator=gen).to(BF16), torch.arange(n_tok, dtype=torch.int32) + 5000 * step, (torch.arange(n_tok, dtype=torch.int32) + 37 * step) % (width * 128)
        qkv.copy_(x), pos.copy_(p), slots.copy_(r), kc.fill_(5.0), vc.fill_(5.0)
        torch.cuda.synchronize()
        if step < 3:
            g.replay()
        else:
            call(stream=side.cuda_stream)
        torch.cuda.synchronize()
        want, off = R.heads(x[:, :H], wq, 1e-6, p, **rope)
        _near(out, want, off, BF16, "q %d" % step)
        want, off = R.heads(x[:, H:H + G], wk, 1e-6, p, **rope)
        page, row = bt[0, r.long() // 128].long(), r.long() % 128
        _near(kc.cpu()[page, row], want, off, BF16, "k %d" % step)
        assert torch.equal(vc.cpu()[page, row], x[:, H + G:]) and int((kc != 5).any(-1).any(-1).sum()) == n_tok == int((vc != 5).any(-1).any(-1).sum())


def test_a_captured_decode_step(gpu):
    """Fill, attend with weights and cut, captured together with padding behind the last sequence, replayed for several steps beside eager calls: the same bits."""
    import jittorinfer_amd as J
    H, G, D, n_seq, width, keep = 16, 8, 128, 5, 260, 400
    gen = torch.Generator().manual_seed(91)
    bt = R.make_table(gen, [width * 128] * n_seq, width, n_seq * width + 1).to(gpu)
    k0, v0 = (torch.randn((n_seq * width + 1, 128, G, D), generator=torch.Generator(device=gpu).manual_seed(i), device=gpu, dtype=F32).to(BF16) for i in range(2))
    ids = torch.arange(n_seq, dtype=torch.int32, device=gpu)
    fresh = lambda: dict(kc=k0.clone(), vc=v0.clone(), sums=torch.zeros((n_seq, G, width * 128), device=gpu), qkv=torch.zeros((n_seq, H + 2 * G, D), dtype=BF16, device=gpu),
                         pos=torch.zeros(n_seq, dtype=torch.int32, device=gpu), slots=torch.zeros(n_seq, dtype=torch.int32, device=gpu), lens=torch.zeros(n_seq, dtype=torch.int32, device=gpu),
                         q=torch.empty((n_seq, H, D), dtype=BF16, device=gpu), out=torch.empty((n_seq, H, D), dtype=BF16, device=gpu),
                         kept=torch.empty((n_seq, G, keep), dtype=torch.int32, device=gpu), new=torch.empty(n_seq, dtype=torch.int32, device=gpu))

    def step(s):
        J.gqa_norm_rope(s["qkv"][:, :H], s["qkv"][:, H:H + G], s["qkv"][:, H + G:], s["pos"], n_dims=D, mode=2, k_cache=s["kc"], v_cache=s["vc"], block_table=bt, seq_ids=ids, slots=s["slots"], q_out=s["q"])
        J.gqa_attn(s["q"], s["kc"], s["vc"], bt, s["lens"], scale=0.09, weights=s["sums"], out=s["out"])
        J.gqa_evict(s["sums"], bt, s["lens"], s["kc"], s["vc"], n_keep=keep, n_sink=4, n_recent=60, weights_out=s["sums"], kept=s["kept"], new_lens=s["new"])
    held, eager = fresh(), fresh()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(held)
    lens = [1, 33000, 401, 700, 0]                        # the last one is padding: no row, its token's row lies outside the table
    for i in range(4):
        x = torch.randn(held["qkv"].shape, generator=gen).to(BF16)
        for s in (held, eager):
            s["qkv"].copy_(x)
            s["pos"].copy_(torch.tensor([n + 50 * i for n in lens], dtype=torch.int32))
            s["slots"].copy_(torch.tensor([n - 1 for n in lens], dtype=torch.int32))
            s["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        g.replay()
        step(eager)
        torch.cuda.synchronize()
        for name in held:
            assert torch.equal(held[name], eager[name]), (i, name)
        assert held["new"].tolist() == [min(n, keep) for n in lens] and (held["out"][4] == 0).all() and not held["sums"][4].any()
        lens = [n + 1 if n else 0 for n in held["new"].tolist()]


@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-38])
def test_norm_rope_of_tiny_rows(gpu, eps):
    """Mean squares below the smallest normal number with an eps that does not lift them: rows of unit size all the same, and zeros where eps holds them up."""
    import jittorinfer_amd as J
    gen = torch.Generator().manual_seed(92)
    size = torch.tensor([1e-18, 1e-19, 5e-20, 1.0])[:, None, None]
    q = (torch.rand((4, 3, 128), generator=gen) + 0.5) * size * torch.where(torch.rand((4, 3, 128), generator=gen) < 0.5, -1.0, 1.0)
    w, pos = torch.rand(128, generator=gen) + 0.5, torch.arange(4, dtype=torch.int32)
    want, off = R.heads(q, w, float(torch.tensor(eps, dtype=F32)), pos, 128, 2)
    # squares, their sum, mean and eps step by 2^-149 down there: three times that of the mean square, half of it in its root
    ms = (q.double() ** 2).mean(-1, keepdim=True) + eps
    off = off + want.abs().amax(-1, keepdim=True) * 2 * 1.5 * 2.0 ** -149 / ms
    got = J.gqa_norm_rope(q.to(gpu), None, None, pos.to(gpu), n_dims=128, mode=2, q_weight=w.to(gpu), eps=eps)
    _near(got, want, off, F32)
    if eps:
        assert (J.gqa_norm_rope(torch.zeros((1, 2, 128), device=gpu), None, None, pos[:1].to(gpu), n_dims=128, mode=2, q_weight=w.to(gpu), eps=eps) == 0).all()
