"""The paged cache of ordinary heads on the GPU, at its edges: weights bit by bit, caps of any size, streams of the caller, and shapes that only one rule reaches."""
import math

import pytest
import torch

from tests import gqa_util as R
from tests.test_gqa_gpu import BF16, F16, F32, WIDTHS, _attn_case, _check_attn, _check_evict, _check_rows, _near

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -24


def _exact_scores_case(n, width, heads, kv_heads, dk, dv, dtype, seed=0):
    """One sequence whose scores are known exactly (a query of one 1, keys of one number t = -j / 64, scale 1), whose row i has its weight to itself in column i of
    128 or fewer: V is one-hot, so a result is the sum of few weights and nothing else."""
    gen = torch.Generator().manual_seed(seed)
    q, k, v, bt, lens = _attn_case(seed, [n], width, heads, kv_heads, dk, dv, dtype)
    at = torch.arange(n)
    page, row = bt[0].long()[at // 128], at % 128
    t = -(torch.randint(0, 61, (n,), generator=gen).double() / 64)
    q.zero_()
    q[..., 0] = 1
    k[page, row] = 0
    k[page, row, :, 0] = t.to(dtype)[:, None]
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
