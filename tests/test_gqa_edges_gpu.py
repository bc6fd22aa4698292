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
