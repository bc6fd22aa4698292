"""The paged cache of ordinary heads on the GPU against plain forms in 64 bits (tests/gqa_util.py): attention of a new token, the pass that fills the
cache, eviction, and the three in a row."""
import math

import pytest
import torch

from tests import gqa_util as R

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
WIDTHS = [(64, 64), (128, 128), (192, 128), (256, 256)]


def _near(got, want, off, dtype, what=""):
    """Within the f32 bound plus half a step of the result's type (and of its smallest numbers)."""
    got = got.cpu().double()
    assert torch.isfinite(got).all(), "%s: %d values are not finite" % (what, int((~torch.isfinite(got)).sum()))
    tol = off + R.half_step(dtype) * want.abs() + torch.finfo(dtype).smallest_normal * R.half_step(dtype)
    bad = (got - want).abs() > tol
    assert not bad.any(), "%s: %d of %d, worst %.3g of its bound" % (what, int(bad.sum()), bad.numel(), float(((got - want).abs() / tol).max()))


def _attn_case(seed, lens, width, heads, kv_heads, dk, dv, dtype, layout="cells", spare=2, stale=float("nan")):
    """Pages hold what the lengths need and NaN everywhere else: rows behind a sequence's end, spare pages."""
    gen = torch.Generator().manual_seed(seed)
    pages = sum((max(n, 0) + 127) // 128 for n in lens) + spare
    bt = R.make_table(gen, [min(n, width * 128) for n in lens], width, pages)
    k = R.make_cache(gen, pages, kv_heads, dk, dtype, layout, fill=stale)
    v = R.make_cache(gen, pages, kv_heads, dv, dtype, layout, fill=stale) if dv else None
    for b, n in enumerate(lens):
        at = torch.arange(min(max(n, 0), width * 128))
        page = bt[b].long()[at // 128]
        k[page, at % 128] = torch.randn((len(at), kv_heads, dk), generator=gen).to(dtype)
        if dv:
            v[page, at % 128] = torch.randn((len(at), kv_heads, dv), generator=gen).to(dtype)
    q = torch.randn((len(lens), heads, dk), generator=gen).to(dtype)
    return q, k, v, bt, torch.tensor(lens, dtype=torch.int32)


def _check_attn(gpu, q, k, v, bt, lens, what="", out_type=None, weights=True, **kw):
    import jittorinfer_amd as J
    scale = 1 / math.sqrt(q.shape[2])
    out, off, w, w_off = R.attn(q.to(k.dtype), k, v, bt, lens.tolist(), scale, kw.get("logit_softcap", 0.0), kw.get("window", 0), kw.get("mask"))
    d = {n: (t.to(gpu) if isinstance(t, torch.Tensor) else t) for n, t in kw.items()}
    before = torch.rand(w.shape, generator=torch.Generator().manual_seed(1)) if weights else None
    sums = before.to(gpu) if weights else None
    dst = torch.full(out.shape, float("nan"), dtype=out_type, device=gpu) if out_type else None
    got = J.gqa_attn(q.to(gpu), k.to(gpu), v.to(gpu) if v is not None else None, bt.to(gpu), lens.to(gpu), scale=scale, weights=sums, out=dst, **d)
    torch.cuda.synchronize()
    if v is not None:
        _near(got, out, off, got.dtype, what)
    if weights:
        _near(sums, before.double() + w, w_off, F32, what + " weights")
        idle = w == 0
        assert torch.equal(sums.cpu()[idle & (w_off == 0)], before[idle & (w_off == 0)])
    return got, sums


LENS = [0, 1, 31, 32, 33, 127, 128, 129, 300, 512]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dk,dv", WIDTHS)
@pytest.mark.parametrize("layout", ["cells", "heads"])
def test_attn_widths_types_layouts(gpu, dk, dv, dtype, layout):
    _check_attn(gpu, *_attn_case(dk, LENS, 4, 8, 2, dk, dv, dtype, layout), "%s %s" % ((dk, dv), dtype))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 7), (3, 1), (16, 1), (34, 2), (32, 1), (40, 1), (66, 1), (28, 4)])
def test_attn_groups(gpu, heads, kv_heads):
    """A query head for itself, groups that fill a block of 16, that pass it, and more than the two blocks a wave holds."""
    _check_attn(gpu, *_attn_case(heads, [5, 200, 0, 129], 2, heads, kv_heads, 64, 64, BF16))
    _check_attn(gpu, *_attn_case(heads, [5, 200, 0, 129], 300, heads, kv_heads, 64, 64, BF16))       # a wide block table: two blocks of 16 a wave


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dk,dv", WIDTHS)
@pytest.mark.parametrize("heads,kv_heads,layout", [(8, 4, "cells"), (24, 8, "heads"), (64, 4, "cells")])
def test_attn_four_heads_a_workgroup(gpu, heads, kv_heads, layout, dk, dv, dtype):
    """Block tables with room for 8192 pages and more, KV heads in fours: a wave takes a head of its own; runs that end inside a page list,
    windows that begin and lengths that end inside any quarter of a page."""
    case = _attn_case(dk + heads, [0, 1, 31, 33, 64, 97, 128, 129, 300, 640], 256, heads, kv_heads, dk, dv, dtype, layout)
    _check_attn(gpu, *case)
    _check_attn(gpu, *case, window=70)
    _check_attn(gpu, *case, window=200, n_workgroups=5, logit_softcap=20.0, mask=_mask(torch.Generator().manual_seed(4), 10, 256 * 128))
    _check_attn(gpu, *case, out_type=F32, n_workgroups=3, mask=torch.zeros((10, 300), dtype=F16))


@pytest.mark.parametrize("n_workgroups", [1, 2, 3, 5, 8, 64, 4096])
def test_attn_any_number_of_workgroups(gpu, n_workgroups):
    """Runs that hold several sequences, end inside one, or are empty."""
    _check_attn(gpu, *_attn_case(3, [700, 1, 0, 0, 128, 513, 40, 0], 6, 4, 2, 128, 128, F16), n_workgroups=n_workgroups)


def test_attn_more_sequences_than_threads(gpu):
    gen = torch.Generator().manual_seed(5)
    lens = [int(x) for x in torch.randint(0, 200, (600,), generator=gen)]
    lens[:300] = [0] * 300
    _check_attn(gpu, *_attn_case(5, lens, 2, 2, 1, 64, 64, BF16))


@pytest.mark.parametrize("window", [1, 5, 100, 128, 129, 1000])
def test_attn_window(gpu, window):
    _check_attn(gpu, *_attn_case(6, [0, 1, 130, 256, 300, 511], 4, 4, 2, 128, 128, BF16), window=window)


@pytest.mark.parametrize("cap", [5.0, 50.0])
def test_attn_softcap(gpu, cap):
    _check_attn(gpu, *_attn_case(7, [1, 130, 300], 3, 4, 1, 128, 128, F16), logit_softcap=cap)


@pytest.mark.parametrize("dk,dv", [(128, 128), (256, 256)])
def test_attn_lengths_outside_the_table(gpu, dk, dv):
    """A negative length is none, one past the table's room is that room."""
    q, k, v, bt, lens = _attn_case(8, [-5, 256, 200], 2, 4, 2, dk, dv, BF16)
    lens[1] = 100000
    _check_attn(gpu, q, k, v, bt, lens)


def _mask(gen, n_seq, n):
    m = torch.zeros((n_seq, n), dtype=F16)
    m[torch.rand((n_seq, n), generator=gen) < 0.3] = float("-inf")
    return m


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attn_mask(gpu, dtype):
    """Rows struck out, a sequence without any left, values that are not 0, keys and values of struck-out rows that are NaN or infinite."""
    q, k, v, bt, lens = _attn_case(9, [300, 129, 64, 40, 1], 3, 6, 2, 64, 64, dtype)
    gen = torch.Generator().manual_seed(9)
    mask = _mask(gen, 5, 384)
    mask[2] = float("-inf")
    mask[3] = torch.randn(384, generator=gen).to(F16)
    mask[4, 0] = 0.0
    for b, n in enumerate(lens.tolist()):
        for i in torch.nonzero(mask[b, :n] == float("-inf"))[:, 0].tolist():
            k[bt[b, i // 128], i % 128] = float("nan") if i % 2 else float("inf")
            v[bt[b, i // 128], i % 128] = float("inf") if i % 3 else float("nan")
    got, _ = _check_attn(gpu, q, k, v, bt, lens, mask=mask)
    assert (got[2] == 0).all()


def test_attn_mask_of_the_lowest_value(gpu):
    """-65504 is a number: rows that carry it weigh nothing beside rows that do not, and share the weight where all carry it."""
    q, k, v, bt, lens = _attn_case(10, [200, 200], 2, 4, 2, 64, 64, BF16)
    mask = torch.zeros((2, 256), dtype=F16)
    mask[0, ::2] = -65504.0
    mask[1] = -65504.0
    _check_attn(gpu, q, k, v, bt, lens, mask=mask)


def test_attn_mask_narrower_than_the_sequences(gpu):
    """Rows past a mask's end are out; with a window in front of them nothing may be left."""
    q, k, v, bt, lens = _attn_case(11, [300, 100, 256], 3, 4, 2, 64, 64, BF16)
    _check_attn(gpu, q, k, v, bt, lens, mask=torch.zeros((3, 130), dtype=F16))
    _check_attn(gpu, q, k, v, bt, lens, mask=torch.zeros((1, 130), dtype=F16).expand(3, 130), window=60)


@pytest.mark.parametrize("value", [-1, 1000000])
def test_attn_bad_pages_count_as_masked(gpu, value):
    q, k, v, bt, lens = _attn_case(12, [300, 256, 100], 3, 4, 2, 128, 128, F16)
    k[0], v[0] = float("nan"), float("nan")      # (a bad page is read as page 0, whose rows must not show)
    keep = bt == 0
    bt[keep] = 1
    bt[0, 1] = value
    bt[1, 0] = value
    bt[2, 0] = value
    k2, v2 = k.clone(), v.clone()
    k2[1:], v2[1:] = torch.randn(k2[1:].shape).to(F16), torch.randn(v2[1:].shape).to(F16)
    got, _ = _check_attn(gpu, q, k2, v2, bt, lens)
    assert (got[2] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attn_f32_queries_and_results(gpu, dtype):
    """f32 queries are rounded to the cache's type; f32 results keep what the 16-bit ones round away."""
    q, k, v, bt, lens = _attn_case(13, [1, 77, 300], 3, 4, 2, 128, 128, dtype)
    q32 = torch.randn(q.shape, generator=torch.Generator().manual_seed(2))
    _check_attn(gpu, q32, k, v, bt, lens, out_type=F32)
    _check_attn(gpu, q32, k, v, bt, lens, out_type=dtype)
    got, _ = _check_attn(gpu, q, k, v, bt, lens, out_type=F32)
    assert got.dtype == F32


def test_attn_strided_operands(gpu):
    """Queries inside a fused projection, results inside a wider tensor, caches with room between rows, weights with room behind."""
    import jittorinfer_amd as J
    q, k, v, bt, lens = _attn_case(14, [130, 50], 2, 4, 2, 64, 64, BF16)
    scale = 0.125
    out, off, w, w_off = R.attn(q, k, v, bt, lens.tolist(), scale)
    qq = torch.randn((2, 9, 64)).to(BF16)
    qq[:, 3:7] = q
    kk, vv = torch.zeros((k.shape[0], 128, 3, 72), dtype=BF16), torch.zeros((k.shape[0], 130, 2, 64), dtype=BF16)
    kk[:, :, :2, :64], vv[:, :128] = k, v
    dst = torch.full((2, 6, 80), 7.0, dtype=BF16, device=gpu)
    sums = torch.zeros((2, 2, 300), device=gpu)
    J.gqa_attn(qq.to(gpu)[:, 3:7], kk.to(gpu)[:, :, :2, :64], vv.to(gpu)[:, :128], bt.to(gpu), lens.to(gpu), scale=scale, out=dst[:, 1:5, 8:72], weights=sums)
    _near(dst[:, 1:5, 8:72], out, off, BF16)
    _near(sums[..., :256], w, w_off, F32)
    assert (dst[:, 0] == 7).all() and (dst[:, 5] == 7).all() and (dst[:, :, :8] == 7).all() and (dst[:, :, 72:] == 7).all() and (sums[..., 256:] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads", [1, 16, 100, 130])
def test_weights_over_a_latent_cache(gpu, dtype, heads):
    q, k, _, bt, lens = _attn_case(15, [0, 1, 200, 385], 4, heads, 1, 576, 0, dtype)
    _check_attn(gpu, q, k, None, bt, lens)
    _check_attn(gpu, q, k, None, bt, lens, window=70, n_workgroups=3)
    mask = _mask(torch.Generator().manual_seed(3), 4, 512)
    _check_attn(gpu, q, k, None, bt, lens, mask=mask)


@pytest.mark.parametrize("kw", [dict(), dict(window=1500), dict(window=2100, n_workgroups=40), dict(n_workgroups=7)], ids=str)
def test_weights_of_many_rows(gpu, kw):
    """More rows than the workgroups that add them up take at once; few and many pieces to a head."""
    _check_attn(gpu, *_attn_case(30, [2500, 2177, 1, 0, 129, 2400, 300, 2499], 20, 72, 8, 64, 64, BF16), **kw)


@pytest.mark.parametrize("kw", [dict(), dict(window=5000), dict(n_workgroups=200, window=3000)], ids=str)
def test_weights_of_heads_in_many_pieces(gpu, kw):
    """Heads joined ahead of the sums: over a latent cache, and with results; sequences of one piece and of none beside them."""
    _check_attn(gpu, *_attn_case(37, [8001, 0, 100], 64, 128, 1, 576, 0, BF16), **kw)
    _check_attn(gpu, *_attn_case(38, [16000, 1], 128, 64, 1, 64, 64, F16), **kw)
    _check_attn(gpu, *_attn_case(39, [9001], 128, 40, 1, 576, 0, F16), mask=_mask(torch.Generator().manual_seed(5), 1, 9001), **kw)


@pytest.mark.parametrize("kw", [dict(), dict(n_workgroups=5)], ids=str)
def test_weights_of_groups_past_256_heads(gpu, kw):
    _check_attn(gpu, *_attn_case(31, [5, 300, 0, 129], 3, 600, 2, 64, 64, F16), **kw)
    _check_attn(gpu, *_attn_case(32, [200, 0, 385], 4, 300, 1, 576, 0, BF16), **kw)
    _check_attn(gpu, *_attn_case(33, [1400, 0, 1345] + [0, 1] * 49, 11, 300, 1, 64, 64, BF16), **kw)


@pytest.mark.parametrize("n_seq,heads", [(255, 16), (257, 16), (600, 3), (130, 130)])
def test_weights_over_many_latent_caches(gpu, n_seq, heads):
    """As many sequences (blocks of 128 heads) as workgroups, and more: runs of whole ones in turn, that leave no piece."""
    gen = torch.Generator().manual_seed(n_seq)
    lens = [int(x) for x in torch.randint(0, 200, (n_seq,), generator=gen)]
    _check_attn(gpu, *_attn_case(36, lens, 2, heads, 1, 576, 0, BF16))


def test_attn_scores_far_apart(gpu):
    """Scores that grow by hundreds along a sequence, and fall: the running maximum moves, and leaves nothing of what came before."""
    q, k, v, bt, lens = _attn_case(16, [512, 512], 4, 4, 2, 64, 64, F16)
    for b, order in enumerate((1, -1)):
        at = torch.arange(512)
        ramp = torch.linspace(0, 30, 512) if order > 0 else torch.linspace(30, 0, 512)
        k[bt[b].long()[at // 128], at % 128] = (q[b, ::2].float()[None] * ramp[:, None, None] * 0.2).to(F16)
    _check_attn(gpu, q, k, v, bt, lens)
    _check_attn(gpu, q, k, v, bt, lens, n_workgroups=2)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("above", [9.0, 11.0, 13.0, 15.0, 17.5, 22.0])
@pytest.mark.parametrize("at", [0, 777, 16383])
def test_attn_one_row_far_above_many(gpu, dtype, above, at):
    """A row with a value of 0 holds nearly all of the weight: what is left is the sum of many weights of 2^-13 to 2^-32 of the largest."""
    import jittorinfer_amd as J
    n = 16384
    gen = torch.Generator().manual_seed(34)
    q, k, v, bt, lens = _attn_case(34, [n], n // 128, 4, 2, 64, 64, dtype)
    rows = torch.arange(n)
    page, row = bt[0].long()[rows // 128], rows % 128
    q[:] = 0
    q[..., 0] = 8
    k[page, row] = 0
    k[page[at], row[at], :, 0] = above
    v[page, row] = (torch.rand((n, 2, 64), generator=gen) + 0.5).to(dtype)
    v[page[at], row[at]] = 0
    out, off, _, _ = R.attn(q, k, v, bt, [n], 1 / 8)
    # in f16 the two halves of a weight end at 2^-25, 2^-36 of the largest (2^11 at least): an error of that a row
    off = off + (n * 1.5 * 2.0 ** -36 if dtype == F16 else 0.0)
    for n_workgroups in (0, 1):
        got = J.gqa_attn(q.to(gpu), k.to(gpu), v.to(gpu), bt.to(gpu), lens.to(gpu), scale=1 / 8, n_workgroups=n_workgroups, out=torch.empty(out.shape, dtype=F32, device=gpu))
        _near(got, out, off, F32)


def test_attn_same_call_same_bits(gpu):
    import jittorinfer_amd as J
    q, k, v, bt, lens = (t.to(gpu) for t in _attn_case(17, [900, 33, 513], 8, 8, 2, 128, 128, BF16))
    runs = []
    for _ in range(3):
        sums = torch.zeros((3, 2, 1024), device=gpu)
        runs.append((J.gqa_attn(q, k, v, bt, lens, scale=0.1, weights=sums), sums))
    for out, sums in runs[1:]:
        assert torch.equal(out, runs[0][0]) and torch.equal(sums, runs[0][1])


def test_attn_pool_past_32_bits(gpu):
    """Pages whose offset in the pool passes 2^32 bytes."""
    import jittorinfer_amd as J
    n_pages = 20000                                # 8 heads x 128 x 128 rows x 2 bytes: 262144 bytes a page
    k = torch.zeros((n_pages, 128, 8, 128), dtype=BF16, device=gpu)
    v = torch.zeros((n_pages, 128, 8, 128), dtype=BF16, device=gpu)
    gen = torch.Generator().manual_seed(18)
    ids = [n_pages - 1, 17000, 3]
    bt = torch.tensor([ids], dtype=torch.int32)
    rows_k, rows_v = torch.randn((3, 128, 8, 128), generator=gen).to(BF16), torch.randn((3, 128, 8, 128), generator=gen).to(BF16)
    k[ids], v[ids] = rows_k.to(gpu), rows_v.to(gpu)
    q = torch.randn((1, 16, 128), generator=gen).to(BF16)
    out, off, _, _ = R.attn(q, rows_k, rows_v, torch.tensor([[0, 1, 2]], dtype=torch.int32), [350], 0.1)
    got = J.gqa_attn(q.to(gpu), k, v, bt.to(gpu), torch.tensor([350], dtype=torch.int32, device=gpu), scale=0.1)
    _near(got, out, off, BF16)
    # the cache write and the eviction reach the same pages
    x = torch.randn((1, 16, 128), generator=gen).to(BF16).to(gpu)
    kk, one = torch.randn((1, 8, 128), generator=gen).to(BF16).to(gpu), torch.zeros(1, dtype=torch.int32, device=gpu)
    J.gqa_norm_rope(x, kk, kk, torch.tensor([5], dtype=torch.int32, device=gpu), n_dims=0, k_cache=k, v_cache=v, block_table=bt.to(gpu), seq_ids=one)
    assert torch.equal(k[n_pages - 1, 5], kk[0]) and torch.equal(v[n_pages - 1, 5], kk[0])
    w = torch.zeros((1, 8, 384), device=gpu)
    w[..., 200:300] = 1.0
    kept, new, _ = J.gqa_evict(w, bt.to(gpu), torch.tensor([350], dtype=torch.int32, device=gpu), k, v, n_keep=100)
    assert torch.equal(kept[0, 0].cpu(), torch.arange(200, 300, dtype=torch.int32)) and int(new[0]) == 100
    assert torch.equal(k[n_pages - 1, :100].cpu(), rows_k.flatten(0, 1)[200:300]) and torch.equal(v[n_pages - 1, :100].cpu(), rows_v.flatten(0, 1)[200:300])


def test_attn_graphs(gpu):
    """Two captured graphs replayed in turn with eager calls between, lengths changing under them."""
    import jittorinfer_amd as J
    cases, graphs = [], []
    for seed, lens in ((19, [900, 33, 513]), (20, [128, 1000, 1])):
        q, k, v, bt, ln = _attn_case(seed, [1024] * 3, 8, 8, 2, 128, 128, BF16)
        cases.append([t.to(gpu) for t in (q, k, v, bt)] + [torch.tensor(lens, dtype=torch.int32, device=gpu)])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for q, k, v, bt, ln in cases:
            sums = torch.zeros((3, 2, 1024), device=gpu)
            J.gqa_attn(q, k, v, bt, ln, scale=0.1, weights=sums)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for q, k, v, bt, ln in cases:
        sums, out = torch.zeros((3, 2, 1024), device=gpu), torch.empty((3, 8, 128), dtype=BF16, device=gpu)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            J.gqa_attn(q, k, v, bt, ln, scale=0.1, weights=sums, out=out)
        graphs.append((g, out, sums))
    for step in range(4):
        for i, ((g, out, sums), (q, k, v, bt, ln)) in enumerate(zip(graphs, cases)):
            ln.copy_(torch.tensor([100 + 200 * step, 1000 - 300 * step + i, step], dtype=torch.int32))
            sums.zero_()
        streams = [torch.cuda.Stream() for _ in graphs]
        torch.cuda.synchronize()
        for (g, _, _), st in zip(graphs, streams):          # side by side
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for (g, out, sums), (q, k, v, bt, ln) in zip(graphs, cases):
            want = torch.zeros_like(sums)
            eager = J.gqa_attn(q, k, v, bt, ln, scale=0.1, weights=want)
            torch.cuda.synchronize()
            assert torch.equal(eager, out) and torch.equal(want, sums), step


@pytest.mark.parametrize("dk,dv,kv_heads", [(256, 256, 2), (576, 0, 1), (64, 64, 4)])
def test_attn_in_a_graph_widths(gpu, dk, dv, kv_heads):
    """The kernels that ask for more LDS, and the four-head one, captured before they ever ran, and replayed while lengths change."""
    import jittorinfer_amd as J
    q, k, v, bt, lens = _attn_case(dk, [1024] * 2, 8 if dk != 64 else 2200, 8, kv_heads, dk, dv, F16, stale=0.0)
    d = [t.to(gpu) if t is not None else None for t in (q, k, v, bt, lens)]
    sums = torch.zeros((2, kv_heads, bt.shape[1] * 128), device=gpu)
    out = torch.empty((2, 8, dv), dtype=F16, device=gpu) if dv else None
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        J.gqa_attn(*d, scale=0.05, weights=sums, out=out)
    for step in range(3):
        n = [1000 - 333 * step, 1 + 500 * step]
        d[4].copy_(torch.tensor(n, dtype=torch.int32))
        sums.zero_()
        g.replay()
        torch.cuda.synchronize()
        want, off, w, w_off = R.attn(q, k, v, bt, n, 0.05)
        if dv:
            _near(out, want, off, F16, str(step))
        _near(sums, w, w_off, F32, str(step))


def test_two_threads_on_one_stream(gpu):
    """Calls of two threads share their stream's scratch: the kernels of a call stay together."""
    import threading
    import jittorinfer_amd as J
    cases, want = [], []
    for seed in (60, 61):
        c = [t.to(gpu) for t in _attn_case(seed, [900, 500, 1024], 8, 8, 2, 128, 128, BF16)]
        cases.append(c)
        want.append(J.gqa_attn(*c, scale=0.1))
    torch.cuda.synchronize()
    bad = []

    def work(i):
        outs = [J.gqa_attn(*cases[i], scale=0.1) for _ in range(200)]
        torch.cuda.synchronize()
        bad.extend(1 for o in outs if not torch.equal(o, want[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_attn_on_another_stream(gpu):
    import jittorinfer_amd as J
    q, k, v, bt, lens = _attn_case(21, [300, 129], 3, 4, 2, 64, 64, BF16)
    out, off, _, _ = R.attn(q, k, v, bt, lens.tolist(), 0.1)
    d = [t.to(gpu) for t in (q, k, v, bt, lens)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    dst = torch.empty((2, 4, 64), dtype=BF16, device=gpu)
    with pytest.raises(ValueError):
        J.gqa_attn(*d, scale=0.1, stream=side.cuda_stream)
    J.gqa_attn(*d, scale=0.1, stream=side.cuda_stream, out=dst)
    side.synchronize()
    _near(dst, out, off, BF16)
    with torch.cuda.stream(side):
        got = J.gqa_attn(*d, scale=0.1)
    side.synchronize()
    assert torch.equal(got, dst)


def test_attn_empty_batch(gpu):
    import jittorinfer_amd as J
    z = lambda *s, dtype=BF16: torch.zeros(s, dtype=dtype, device=gpu)
    out = J.gqa_attn(z(0, 4, 64), z(1, 128, 2, 64), z(1, 128, 2, 64), z(0, 1, dtype=torch.int32), z(0, dtype=torch.int32), scale=1.0)
    assert out.shape == (0, 4, 64)


# ---------------------------------------------------------------- norms, rotation, cache write

YARN = dict(n_ctx_orig=4096, freq_scale=0.025, ext_factor=1.0, attn_factor=0.8)


def _check_rows(gpu, src, kv, n_tok, n_head, n_head_kv, dk, dv, layout="cells", norm=True, w_type=F32, slots=True, seed=0, out_type=None, ff=False, in_place=False, past=0, **rope):
    import jittorinfer_amd as J
    gen = torch.Generator().manual_seed(seed)
    qkv = (torch.randn((n_tok, n_head * dk + n_head_kv * (dk + dv)), generator=gen) * 3).to(src)
    cut = lambda t: (t[:, :n_head * dk].view(n_tok, n_head, dk), t[:, n_head * dk:(n_head + n_head_kv) * dk].view(n_tok, n_head_kv, dk),
                     t[:, (n_head + n_head_kv) * dk:].view(n_tok, n_head_kv, dv))
    q, k, v = cut(qkv)
    wq, wk = ((torch.randn(dk, generator=gen) * 0.2 + 1).to(w_type) if norm else None for _ in range(2))
    ids = torch.arange(n_tok, dtype=torch.int32) % 3
    within = torch.arange(n_tok, dtype=torch.int32) // 3
    pos = within + past
    width = n_tok // 3 // 128 + 1
    bt = R.make_table(gen, [width * 128] * 3, width, 3 * width + 1)
    kc, vc = (R.make_cache(gen, 3 * width + 1, n_head_kv, d, kv, layout, fill=-2.0) for d in (dk, dv))
    factors = torch.rand(rope["n_dims"] // 2, generator=gen) + 0.5 if ff else None
    d_qkv, d_kc, d_vc = qkv.to(gpu), kc.to(gpu), vc.to(gpu)
    dq, dk_, dv_ = cut(d_qkv)
    g = lambda t: t.to(gpu) if t is not None else None
    dst = dq if in_place else torch.full(q.shape, float("nan"), dtype=out_type, device=gpu) if out_type else None
    got = J.gqa_norm_rope(dq, dk_, dv_, pos.to(gpu), q_weight=g(wq), k_weight=g(wk), eps=1e-5, k_cache=d_kc, v_cache=d_vc, block_table=bt.to(gpu), seq_ids=ids.to(gpu),
                          slots=within.to(gpu) if slots else None, freq_factors=g(factors), q_out=dst, **rope)
    torch.cuda.synchronize()
    want, off = R.heads(q, wq, 1e-5, pos, freq_factors=factors, **rope)
    _near(got, want, off, got.dtype, "q")
    want_k, off_k = R.heads(k, wk, 1e-5, pos, freq_factors=factors, **rope)
    row = within if slots else pos
    at = (row < width * 128).nonzero()[:, 0]
    page, slot = bt[ids.long()[at], row.long()[at] // 128].long(), row.long()[at] % 128
    h_kc, h_vc = d_kc.cpu(), d_vc.cpu()
    _near(h_kc[page, slot], want_k[at], off_k[at], kv, "k")
    assert torch.equal(h_vc[page, slot], v[at].to(kv))
    mark = torch.ones(kc.shape[:2], dtype=torch.bool)
    mark[page, slot] = False
    assert (h_kc[mark] == -2).all() and (h_vc[mark] == -2).all()          # rows of no token keep what they held
    return got


@pytest.mark.parametrize("src,kv", [(F32, BF16), (F32, F16), (BF16, BF16), (F16, F16), (BF16, F16)])
@pytest.mark.parametrize("mode", [0, 2])
def test_norm_rope_types(gpu, src, kv, mode):
    _check_rows(gpu, src, kv, 37, 6, 2, 128, 128, n_dims=128, mode=mode)
    _check_rows(gpu, src, kv, 5, 3, 1, 128, 128, n_dims=64, mode=mode, out_type=F32, w_type=src)


@pytest.mark.parametrize("dk,dv", [(8, 8), (16, 8), (64, 64), (72, 40), (96, 96), (128, 128), (192, 128), (256, 256)])
@pytest.mark.parametrize("layout", ["cells", "heads"])
def test_norm_rope_widths(gpu, dk, dv, layout):
    for mode, n_dims in ((0, dk), (2, dk // 16 * 16), (0, 8), (0, 0)):
        _check_rows(gpu, BF16, BF16, 20, 5, 2, dk, dv, layout, n_dims=n_dims, mode=mode, seed=dk)


def test_norm_rope_without_norms_is_the_rotation(gpu):
    _check_rows(gpu, F32, BF16, 40, 4, 4, 64, 64, norm=False, n_dims=64, mode=2, out_type=F32)
    _check_rows(gpu, F32, F16, 40, 4, 4, 64, 64, norm=False, n_dims=32, mode=0, out_type=F32, ff=True)


@pytest.mark.parametrize("past", [0, 1000, 131071, 1048575, 2000000000])
def test_norm_rope_far_positions(gpu, past):
    """The angle's error does not grow with the position."""
    _check_rows(gpu, F32, BF16, 12, 2, 1, 128, 128, n_dims=128, mode=2, out_type=F32, past=past)
    _check_rows(gpu, F32, BF16, 12, 2, 1, 128, 128, n_dims=64, mode=0, out_type=F32, past=past, **YARN)


@pytest.mark.parametrize("n_tok", [1, 2, 3, 255, 1000])
def test_norm_rope_tokens(gpu, n_tok):
    _check_rows(gpu, BF16, BF16, n_tok, 32, 8, 128, 128, n_dims=128, mode=2, **YARN)


def test_norm_rope_positions_as_rows_and_rows_outside_the_table(gpu):
    _check_rows(gpu, BF16, BF16, 300, 2, 1, 64, 64, n_dims=64, mode=0, slots=False)
    _check_rows(gpu, BF16, BF16, 300, 2, 1, 64, 64, n_dims=64, mode=0, slots=False, past=60)     # the last positions have no page


def test_norm_rope_in_place(gpu):
    _check_rows(gpu, BF16, BF16, 50, 32, 8, 128, 128, n_dims=128, mode=2, in_place=True)
    _check_rows(gpu, F32, BF16, 50, 5, 1, 192, 128, n_dims=64, mode=0, in_place=True)


def test_norm_rope_queries_alone_and_keys_without_values(gpu):
    import jittorinfer_amd as J
    gen = torch.Generator().manual_seed(30)
    q, k = torch.randn((9, 4, 64), generator=gen), torch.randn((9, 2, 64), generator=gen)
    pos = torch.arange(9, dtype=torch.int32)
    want, off = R.heads(q, None, 0, pos, 64, 2)
    got = J.gqa_norm_rope(q.to(gpu), None, None, pos.to(gpu), n_dims=64, mode=2)
    _near(got, want, off, F32)
    kc, bt = torch.zeros((1, 128, 2, 64), dtype=F16, device=gpu), torch.zeros((1, 1), dtype=torch.int32, device=gpu)
    got = J.gqa_norm_rope(q.to(gpu), k.to(gpu), None, pos.to(gpu), n_dims=64, mode=2, k_cache=kc, block_table=bt, seq_ids=torch.zeros(9, dtype=torch.int32, device=gpu))
    assert got.dtype == F16
    want, off = R.heads(k, None, 0, pos, 64, 2)
    _near(kc[0, :9], want, off, F16)


@pytest.mark.parametrize("what", ["slot", "seq", "page"])
def test_norm_rope_skips_bad_rows(gpu, what):
    import jittorinfer_amd as J
    q, k = torch.randn((4, 2, 64), device=gpu), torch.randn((4, 2, 64), device=gpu)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    kc = torch.full((2, 128, 2, 64), 5.0, dtype=BF16, device=gpu)
    slots, ids, bt = i([0, 1, 2, 3]), i([0, 0, 0, 0]), i([[0, 1]])
    if what == "slot":
        slots = i([-1, 256, 2, 2147483647])
    elif what == "seq":
        ids = i([-1, 1, 0, 1000000])
    else:
        bt = i([[-1, 1]])
        slots = i([0, 5, 130, 127])
    J.gqa_norm_rope(q, k, k, i([0, 1, 2, 3]), n_dims=0, k_cache=kc, v_cache=torch.empty_like(kc), block_table=bt, seq_ids=ids, slots=slots)
    torch.cuda.synchronize()
    page, row = (1, 2) if what == "page" else (0, 2)
    assert torch.equal(kc[page, row], k[2].to(BF16))
    kc[page, row] = 5.0
    assert (kc == 5).all()


def test_norm_rope_zero_rows(gpu):
    """A row of zeros stays one: eps keeps the norm finite; infinities and NaN stay in their own row."""
    import jittorinfer_amd as J
    q = torch.randn((3, 4, 128), device=gpu)
    q[1, 2] = 0
    q[2, 0, 5] = float("nan")
    got = J.gqa_norm_rope(q, None, None, torch.arange(3, dtype=torch.int32, device=gpu), n_dims=128, mode=2, q_weight=torch.ones(128, device=gpu))
    assert (got[1, 2] == 0).all() and torch.isnan(got[2, 0]).all() and torch.isfinite(got[:2]).all() and torch.isfinite(got[2, 1:]).all()


# ---------------------------------------------------------------- eviction

def _check_evict(gpu, w, bt, lens, k, v, n_keep, n_sink=0, n_recent=0, **kw):
    import jittorinfer_amd as J
    want = R.evict(w, bt, lens.tolist(), k, v, n_keep, n_sink, n_recent)
    dk, dv, dw = k.to(gpu), v.to(gpu) if v is not None else None, w.to(gpu)
    if kw.get("in_place"):
        kw = dict(weights_out=dw)
    kept, new, out = J.gqa_evict(dw, bt.to(gpu), lens.to(gpu), dk, dv, n_keep=n_keep, n_sink=n_sink, n_recent=n_recent, **kw)
    torch.cuda.synchronize()
    assert torch.equal(kept.cpu(), want[0]) and torch.equal(new.cpu(), want[1])
    assert torch.equal(R.bits(out.cpu()), R.bits(want[2]))
    assert torch.equal(R.bits(dk.cpu()), R.bits(want[3]))
    if v is not None:
        assert torch.equal(R.bits(dv.cpu()), R.bits(want[4]))


def _evict_case(seed, lens, width, kv_heads, dk, dv, dtype, layout="cells"):
    gen = torch.Generator().manual_seed(seed)
    pages = len(lens) * width + 2
    bt = R.make_table(gen, [width * 128] * len(lens), width, pages)
    k = R.make_cache(gen, pages, kv_heads, dk, dtype, layout)
    v = R.make_cache(gen, pages, kv_heads, dv, dtype, layout) if dv else None
    w = torch.exp(2 * torch.randn((len(lens), kv_heads, width * 128), generator=gen))
    return w, bt, torch.tensor(lens, dtype=torch.int32), k, v


@pytest.mark.parametrize("layout", ["cells", "heads"])
@pytest.mark.parametrize("kv_heads,dk,dv", [(2, 64, 64), (3, 128, 128), (2, 192, 128), (1, 576, 0), (1, 256, 256)])
def test_evict_shapes(gpu, kv_heads, dk, dv, layout):
    w, bt, lens, k, v = _evict_case(dk, [0, 1, 99, 100, 101, 128, 250, 384], 3, kv_heads, dk, dv, BF16, layout)
    _check_evict(gpu, w, bt, lens, k, v, 100, 4, 20)
    _check_evict(gpu, w, bt, lens, k, v, 100, 4, 20, in_place=True)


@pytest.mark.parametrize("n_keep,n_sink,n_recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (7, 0, 0), (50, 50, 0), (50, 0, 50), (50, 25, 25), (128, 3, 3), (129, 0, 64), (383, 1, 1), (384, 0, 0), (500, 4, 4)])
def test_evict_budgets(gpu, n_keep, n_sink, n_recent):
    w, bt, lens, k, v = _evict_case(40, [384, 130, 60], 3, 2, 64, 64, F16)
    _check_evict(gpu, w, bt, lens, k, v, n_keep, n_sink, n_recent)


@pytest.mark.parametrize("kind", ["equal", "few", "zeros", "odd", "negative"])
def test_evict_ties_and_odd_weights(gpu, kind):
    """Equal weights go to the lower row; zeros of either sign are equal; NaN below everything; infinities at the ends."""
    w, bt, lens, k, v = _evict_case(41, [3000, 2500], 24, 2, 64, 64, BF16)
    gen = torch.Generator().manual_seed(41)
    if kind == "equal":
        w[:] = 0.7
    elif kind == "few":
        w = torch.randint(0, 3, w.shape, generator=gen).float()
    elif kind == "zeros":
        w = torch.where(torch.rand(w.shape, generator=gen) < 0.5, 0.0, -0.0)
    elif kind == "odd":
        r = torch.rand(w.shape, generator=gen)
        w[r < 0.3] = float("nan")
        w[(r >= 0.3) & (r < 0.4)] = float("inf")
        w[(r >= 0.4) & (r < 0.8)] = float("-inf")
        w[(r >= 0.8) & (r < 0.85)] = 1e-42
    else:
        w = -w
    _check_evict(gpu, w, bt, lens, k, v, 1000, 3, 100)
    _check_evict(gpu, w, bt, lens, k, v, 2400, 0, 0, in_place=True)


@pytest.mark.parametrize("kind", ["spread", "equal", "few", "odd"])
def test_evict_sequences_selected_by_several_workgroups(gpu, kind):
    """Block tables of more than 32768 rows: lengths that end inside a run of 8192, fill some of the runs, and are not cut at all."""
    lens = [40000, 33000, 8192, 8193, 30000, 100, 20000]
    w, bt, lens, k, _ = _evict_case(46, lens, 313, 1, 16, 0, BF16)
    gen = torch.Generator().manual_seed(46)
    if kind == "equal":
        w[:] = 2.5
    elif kind == "few":
        w = torch.randint(0, 3, w.shape, generator=gen).float()
    elif kind == "odd":
        r = torch.rand(w.shape, generator=gen)
        w[r < 0.3] = float("nan")
        w[(r >= 0.3) & (r < 0.9)] = -1.0
    _check_evict(gpu, w, bt, lens, k, None, 8000, 4, 1000)
    _check_evict(gpu, w, bt, lens, k, None, 20000, 0, 0, in_place=True)
    _check_evict(gpu, w, bt, lens, k, None, 30001, 30001, 0, in_place=True)
    _check_evict(gpu, w, bt, lens, k, None, 39999, 3, 39990)
    _check_evict(gpu, w, bt, lens, k, None, 313 * 128 + 5, 3, 4)


def test_evict_many_long_sequences(gpu):
    """So many heads that one workgroup each selects, in several chunks."""
    import jittorinfer_amd as J
    width, heads, n = 264, 1700, 33700
    gen = torch.Generator().manual_seed(47)
    w = torch.rand((1, heads, width * 128), generator=gen)
    k = torch.arange(width * 128, dtype=torch.int32).view(width, 128, 1, 1).expand(width, 128, heads, 2).contiguous()
    bt, lens = torch.arange(width, dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32)
    d = k.to(gpu)
    kept, new, out = J.gqa_evict(w.to(gpu), bt.to(gpu), lens.to(gpu), d, n_keep=20000, n_sink=2, n_recent=100)
    key = w[0, :, :n].clone()
    key[:, :2], key[:, n - 100:] = 2.0, 2.0
    want = torch.sort(torch.sort(key.to(gpu), dim=1, descending=True, stable=True).indices[:, :20000], dim=1).values
    assert torch.equal(kept[0].long(), want) and new.tolist() == [20000]
    assert torch.equal(out[0, :, :20000], torch.gather(w[0].to(gpu), 1, want)) and (out[0, :, 20000:] == 0).all()
    flat = d.view(width * 128, heads, 2)
    assert torch.equal(flat[:20000, :, 0].T.long(), want) and torch.equal(flat[:20000, :, 1].T.long(), want)
    assert torch.equal(flat[20000:].cpu(), k.view(width * 128, heads, 2)[20000:])


def test_evict_long_sequences(gpu):
    """Several segments of the move, over all the rows one workgroup's selection holds in registers."""
    w, bt, lens, k, _ = _evict_case(42, [20000, 17001], 157, 1, 64, 0, BF16)
    _check_evict(gpu, w, bt, lens, k, None, 9001, 4, 1000)
    w[:, :, ::2] = 1.0
    _check_evict(gpu, w, bt, lens, k, None, 12345, 0, 0, in_place=True)


def test_evict_rows_of_any_bytes(gpu):
    """Q8_0 rows of the latent cache: 612 bytes, 4-byte aligned; rows with room between them stay as they are there."""
    gen = torch.Generator().manual_seed(43)
    w, bt, lens, _, _ = _evict_case(43, [300, 200], 3, 1, 64, 0, BF16)
    k = torch.randint(0, 256, (8, 128, 1, 612), generator=gen, dtype=torch.uint8)
    _check_evict(gpu, w, bt, lens, k, None, 150, 2, 10)
    wide = torch.randint(0, 256, (8, 128, 2, 40), generator=gen, dtype=torch.uint8)
    import jittorinfer_amd as J
    w2 = torch.rand((2, 2, 384), generator=gen)
    want = R.evict(w2, bt, [300, 200], wide[..., 4:28].clone(), None, 150, 2, 10)
    d = wide.to(gpu)
    J.gqa_evict(w2.to(gpu), bt.to(gpu), lens.to(gpu), d[..., 4:28], n_keep=150, n_sink=2, n_recent=10)
    d = d.cpu()
    assert torch.equal(d[..., 4:28], want[3]) and torch.equal(d[..., :4], wide[..., :4]) and torch.equal(d[..., 28:], wide[..., 28:])


def test_evict_strided_weights_and_bad_pages(gpu):
    w, bt, lens, k, v = _evict_case(44, [300, 384], 3, 2, 64, 64, F16)
    bt[0, 1] = -1
    bt[1, 2] = 100000
    _check_evict(gpu, w, bt, lens, k, v, 140, 2, 10)
    wide = torch.rand((2, 4, 400))
    import jittorinfer_amd as J
    want = R.evict(wide[:, 1:3, 5:389].clone(), bt, lens.tolist(), k, v, 140, 2, 10)
    dw = wide.to(gpu)
    kept, new, out = J.gqa_evict(dw[:, 1:3, 5:389], bt.to(gpu), lens.to(gpu), k.to(gpu), v.to(gpu), n_keep=140, n_sink=2, n_recent=10, weights_out=dw[:, 1:3, 5:389])
    assert torch.equal(kept.cpu(), want[0]) and torch.equal(dw[:, 1:3, 5:389].cpu(), want[2])
    wide[:, 1:3, 5:389] = want[2]
    assert torch.equal(dw.cpu(), wide)


def test_evict_in_a_graph(gpu):
    import jittorinfer_amd as J
    w, bt, lens, k, v = _evict_case(45, [300, 384, 90], 3, 2, 64, 64, BF16)
    d = [t.to(gpu) for t in (w, bt, lens, k, v)]
    outs = dict(weights_out=torch.empty_like(d[0]), kept=torch.empty((3, 2, 100), dtype=torch.int32, device=gpu), new_lens=torch.empty(3, dtype=torch.int32, device=gpu))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        J.gqa_evict(*d, n_keep=100, n_sink=2, n_recent=10, **outs)
    for step in range(3):
        gen = torch.Generator().manual_seed(step)
        w = torch.rand(w.shape, generator=gen)
        lens = torch.randint(0, 385, (3,), generator=gen, dtype=torch.int32)
        for t, x in zip(d, (w, bt, lens, k, v)):
            t.copy_(x)
        g.replay()
        torch.cuda.synchronize()
        want = R.evict(w, bt, lens.tolist(), k, v, 100, 2, 10)
        assert torch.equal(outs["kept"].cpu(), want[0]) and torch.equal(outs["new_lens"].cpu(), want[1]) and torch.equal(outs["weights_out"].cpu(), want[2])
        assert torch.equal(d[3].cpu(), want[3]) and torch.equal(d[4].cpu(), want[4])


def test_latent_weights_and_a_long_eviction_in_a_graph(gpu):
    """Heads joined ahead of the sums, selection by several workgroups and the move, captured together: every replay leaves what eager calls leave."""
    import jittorinfer_amd as J
    gen = torch.Generator().manual_seed(47)
    width, n_keep = 260, 9000
    q = torch.randn((2, 64, 576), generator=gen).to(BF16).to(gpu)
    k0 = torch.randn((2 * width + 1, 128, 1, 576), generator=gen).to(BF16).to(gpu)
    bt = R.make_table(gen, [width * 128] * 2, width, 2 * width + 1).to(gpu)
    def step(k, w, lens, kept, new):
        J.gqa_attn(q, k, None, bt, lens, scale=0.05, weights=w)
        J.gqa_evict(w, bt, lens, k, n_keep=n_keep, n_sink=4, n_recent=500, weights_out=w, kept=kept, new_lens=new)
    fresh = lambda: (k0.clone(), torch.zeros((2, 1, width * 128), device=gpu), torch.zeros(2, dtype=torch.int32, device=gpu),
                     torch.empty((2, 1, n_keep), dtype=torch.int32, device=gpu), torch.empty(2, dtype=torch.int32, device=gpu))
    held = fresh()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step(*held)
    for lens in ([33000, 20000], [100, 33280], [9001, 0], [33280, 33280]):
        for t, x in zip(held, fresh()):
            t.copy_(x)
        held[2].copy_(torch.tensor(lens, dtype=torch.int32))
        eager = [t.clone() for t in held]
        g.replay()
        torch.cuda.synchronize()
        step(*eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager)), lens
        assert eager[4].tolist() == [min(n, n_keep) for n in lens]


# ---------------------------------------------------------------- refusals

def _refused(call, args, wrong, errors=(AssertionError,)):
    for name, value in wrong.items():
        with pytest.raises(errors):
            call(**{**args, **({name: value} if not isinstance(value, dict) else value)})


def test_calls_that_are_refused(gpu):
    """Tensors of another shape, type or device are errors before anything is launched."""
    import jittorinfer_amd as J
    z = lambda *s, dtype=BF16: torch.zeros(s, dtype=dtype, device=gpu)
    i = lambda *s: z(*s, dtype=torch.int32)
    q, k, bt, lens, w = z(2, 4, 64), z(3, 128, 2, 64), i(2, 1), i(2), z(2, 2, 128, dtype=F32)
    _refused(J.gqa_attn, dict(q=q, k_cache=k, v_cache=k.clone(), block_table=bt, seq_lens=lens, scale=1.0), dict(
        q=q[0], k_cache=k.float(), v_cache=k[:2], block_table=bt[:1], seq_lens=lens[:1], mask=w[:, 0], window=-1, out=q[:1],
        a=dict(q=q[..., :32]), b=dict(q=q.transpose(1, 2)), c=dict(block_table=bt.long()), d=dict(seq_lens=lens.cpu()), e=dict(mask=w[:1, 0].half()), f=dict(weights=w[..., :100]), g=dict(weights=w.half()),
        h=dict(weights=w[:1].expand(2, 2, 128)), j=dict(v_cache=None), l=dict(k_cache=k[:, :64]), m=dict(k_cache=k[:1].expand(3, 128, 2, 64)), n=dict(v_cache=k.half()), o=dict(out=q[:, :1].expand(2, 4, 64)),
        p=dict(v_cache=None, weights=w, out=q), r=dict(window=1 << 31), s=dict(seq_lens=lens[:, None])))
    _refused(J.gqa_attn, dict(q=q, k_cache=k, v_cache=k.clone(), block_table=bt, seq_lens=lens, scale=1.0), dict(
        a=dict(q=q.half()), b=dict(out=q.half()), c=dict(logit_softcap=-1.0), d=dict(q=z(2, 3, 64)), e=dict(mask=z(2, 0, dtype=F16)), n_workgroups=-1), (RuntimeError, ValueError))
    _refused(J.gqa_attn, dict(q=q, k_cache=k, v_cache=k.clone(), block_table=bt, seq_lens=lens, scale=1.0), dict(q=q.cpu(), scale="x", block_table=None), (RuntimeError, TypeError))
    x, pos = z(5, 2, 64), i(5)
    _refused(J.gqa_norm_rope, dict(q=x, k=x, v=x, pos=pos, n_dims=64, k_cache=k, v_cache=k.clone(), block_table=bt, seq_ids=pos), dict(
        a=dict(k=x[:4]), b=dict(k=x.half()), c=dict(pos=pos[:3]), d=dict(k_cache=None), e=dict(v_cache=None), f=dict(k=None, v=None), g=dict(q_weight=w[0, 0, :32]), h=dict(q_weight=w[0, 0, :64], k_weight=x[0, 0]),
        j=dict(seq_ids=pos[:1]), l=dict(slots=pos.long()), m=dict(k=x[:, :1], v=x[:, :1]), n=dict(v=x[..., :32]), o=dict(q_out=x[:3]), p=dict(freq_factors=w[0, 0, :8]), r=dict(q_out=x[:1].expand(5, 2, 64)),
        s=dict(pos=pos.cpu()), t=dict(k=None, v=None, k_cache=None, v_cache=None, k_weight=x[0, 0])))
    _refused(J.gqa_norm_rope, dict(q=x, k=x, v=x, pos=pos, n_dims=64, k_cache=k, v_cache=k.clone(), block_table=bt, seq_ids=pos), dict(
        n_dims=72, mode=1, freq_base=0.5, a=dict(ext_factor=1.0)), (RuntimeError,))
    _refused(J.gqa_evict, dict(weights=w, block_table=bt, seq_lens=lens, k_cache=k, v_cache=k.clone(), n_keep=10), dict(
        a=dict(weights=w[..., :100]), b=dict(weights=w[:, :1]), c=dict(seq_lens=lens[:1]), d=dict(v_cache=k[:, :, :1]), n_keep=-1, kept=i(2, 2, 11), new_lens=i(3), weights_out=w[..., :127],
        e=dict(weights_out=w[:1].expand(2, 2, 128)), f=dict(k_cache=k[:, :64]), g=dict(seq_lens=lens.cpu())))
    _refused(J.gqa_evict, dict(weights=w, block_table=bt, seq_lens=lens, k_cache=k, v_cache=k.clone(), n_keep=10), dict(
        a=dict(n_keep=0), n_sink=11, n_recent=-1, b=dict(n_sink=5, n_recent=6), new_lens=lens), (RuntimeError,))


def test_empty_batches_with_everything(gpu):
    """No sequence, no token: nothing to do, whatever else is handed in."""
    import jittorinfer_amd as J
    z = lambda *s, dtype=BF16: torch.zeros(s, dtype=dtype, device=gpu)
    k, bt, lens, w = z(3, 128, 2, 64), z(0, 2, dtype=torch.int32), z(0, dtype=torch.int32), z(0, 2, 256, dtype=F32)
    assert J.gqa_attn(z(0, 4, 64), k, k.clone(), bt, lens, scale=1.0, mask=z(0, 256, dtype=F16), weights=w, window=5).shape == (0, 4, 64)
    assert J.gqa_attn(z(0, 4, 576), z(3, 128, 1, 576), None, bt, lens, scale=1.0, weights=z(0, 1, 256, dtype=F32)).shape == (0, 1, 256)
    kept, new, out = J.gqa_evict(w, bt, lens, k, k.clone(), n_keep=10)
    assert kept.shape == (0, 2, 10) and new.shape == (0,) and out.shape == w.shape
    assert J.gqa_norm_rope(z(0, 4, 64), z(0, 2, 64), z(0, 2, 64), lens, n_dims=64, k_cache=k, v_cache=k.clone(), block_table=bt, seq_ids=lens).shape == (0, 4, 64)
    assert not k.any()


def test_integers_past_32_bits_are_refused(gpu):
    import jittorinfer_amd as J
    z = lambda *s, dtype=BF16: torch.zeros(s, dtype=dtype, device=gpu)
    k, bt, lens, w = z(3, 128, 2, 64), z(2, 1, dtype=torch.int32), z(2, dtype=torch.int32), z(2, 2, 128, dtype=F32)
    far = (1 << 32) + 8
    for name in ("n_keep", "n_sink", "n_recent"):
        with pytest.raises(OverflowError):
            J.gqa_evict(w, bt, lens, k, k.clone(), **{"n_keep": 20, name: far})
    with pytest.raises(OverflowError):
        J.gqa_attn(z(2, 4, 64), k, k.clone(), bt, lens, scale=1.0, n_workgroups=far)
    for name in ("n_dims", "mode", "n_ctx_orig"):
        with pytest.raises(OverflowError):
            J.gqa_norm_rope(z(2, 4, 64), None, None, lens, **{"n_dims": 8, name: far})


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_serving_loop(gpu, dtype):
    """Prompts, decode steps that add up their weights, an eviction that frees pages, and decode steps behind it: positions go on, rows are reused.
    The cache as it is on the device is what the plain form reads, so that its rounding does not add up over the steps."""
    import numpy as np
    import jittorinfer_amd as J
    H, G, D, KEEP = 8, 2, 64, 140
    gen = torch.Generator().manual_seed(50)
    pt = J.PageTable(12, 3, 4)
    kc, vc = (torch.zeros((12, 128, G, D), dtype=dtype, device=gpu) for _ in range(2))
    sums = torch.zeros((3, G, 512), device=gpu)
    wq, wk = torch.rand(D, generator=gen) + 0.5, torch.rand(D, generator=gen) + 0.5
    rope = dict(n_dims=D, mode=2, freq_base=10000.0)
    pos = [0, 0, 0]

    def feed(counts):
        """New tokens of every sequence; returns their queries."""
        ids = [b for b, n in enumerate(counts) for _ in range(n)]
        slots = [pt.seq_len(b) + i for b, n in enumerate(counts) for i in range(n)]
        p = [pos[b] + i for b, n in enumerate(counts) for i in range(n)]
        assert pt.find_slot(ids, slots) is not None
        for b, n in enumerate(counts):
            pos[b] += n
        qkv = torch.randn((len(ids), (H + 2 * G) * D), generator=gen).to(dtype)
        d = qkv.to(gpu)
        cut = lambda t: (t[:, :H * D].view(-1, H, D), t[:, H * D:(H + G) * D].view(-1, G, D), t[:, (H + G) * D:].view(-1, G, D))
        bt, _ = pt.fill_inputs([0, 1, 2])
        i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=gpu)
        q = J.gqa_norm_rope(*cut(d), i32(p), q_weight=wq.to(gpu), k_weight=wk.to(gpu), k_cache=kc, v_cache=vc, block_table=i32(bt), seq_ids=i32(ids), slots=i32(slots), **rope)
        want, off = R.heads(cut(qkv)[1], wk, 1e-6, torch.tensor(p), **rope)
        at = torch.tensor(slots)
        page = torch.from_numpy(bt).long()[torch.tensor(ids), at // 128]
        _near(kc.cpu()[page, at % 128], want, off, dtype, "keys")
        return q

    def step():
        q = feed([1, 1, 1])
        bt, lens = pt.fill_inputs([0, 1, 2])
        tb, tl = torch.from_numpy(bt).to(gpu), torch.from_numpy(lens).to(gpu)
        before = sums.cpu().double()
        out = J.gqa_attn(q, kc, vc, tb, tl, scale=0.125, weights=sums)
        torch.cuda.synchronize()
        want, off, w, w_off = R.attn(q.cpu(), kc.cpu(), vc.cpu(), torch.from_numpy(bt), lens.tolist(), 0.125)
        _near(out, want, off, dtype, "out")
        _near(sums, before + w, w_off, F32, "weights")

    feed([300, 40, 200])
    for _ in range(3):
        step()
    bt, lens = pt.fill_inputs([0, 1, 2])
    free = pt.free_pages
    assert all(pt.seq_evict(b, KEEP) for b in range(3))
    assert pt.free_pages == free + 1                # 303 rows on 3 pages, 203 on 2: 140 take two each
    want = R.evict(sums.cpu(), torch.from_numpy(bt), lens.tolist(), kc.cpu(), vc.cpu(), KEEP, 4, 30)
    kept, new, _ = J.gqa_evict(sums, torch.from_numpy(bt).to(gpu), torch.from_numpy(lens).to(gpu), kc, vc, n_keep=KEEP, n_sink=4, n_recent=30, weights_out=sums)
    torch.cuda.synchronize()
    assert torch.equal(kept.cpu(), want[0]) and torch.equal(sums.cpu(), want[2]) and torch.equal(kc.cpu(), want[3]) and torch.equal(vc.cpu(), want[4])
    assert new.tolist() == [140, 43, 140] == [pt.seq_len(b) for b in range(3)]
    for _ in range(3):
        step()
    assert pos == [306, 46, 206] and [pt.seq_len(b) for b in range(3)] == [143, 46, 143]
