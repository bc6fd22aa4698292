"""Attention of many query rows over the same keys on the GPU: ways that a call goes by its sizes, and masks of large numbers."""
import math

import pytest
import torch

from tests import gqa_util as R
from tests.test_gqa_batch_gpu import _shared, _wide
from tests.test_gqa_gpu import BF16, F16

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dk,dtype", [(64, F16), (128, BF16), (256, BF16)])
@pytest.mark.parametrize("n_seq", [1, 5])
def test_prefixes_that_nobody_can_share_are_gqa_attn(gpu, n_seq, dk, dtype):
    """A group each, with rows or without, under a table with much room: the same bits as gqa_attn's."""
    import jittorinfer_amd as J
    q, k, v, bt, lens, starts, plens = (t.to(gpu) for t in _shared(n_seq, [(1, 300)] * n_seq, [5, 0, 130, 1, 700][:n_seq], 8, 2, dk, dk, dtype))
    bt = _wide(bt, k, v)
    want = J.gqa_attn(q, k, v, bt, lens, scale=0.1)
    for shared in (plens, plens * 0):
        assert torch.equal(J.gqa_prefix_attn(q, k, v, bt, lens, starts, shared, scale=0.1), want)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (192, 128), (256, 256)])
@pytest.mark.parametrize("number", [100.0, 300.0, 700.0, -300.0, -700.0])
def test_prompt_mask_of_one_number_on_every_row(gpu, number, dk, dv, dtype):
    """Pairs of keys with the same score, in 16 columns after 16 columns' worth of seven sixteenths of a step of the sum that begins with the mask, or all at once: what is lost of the first
    ones one after the other is kept of the second.  Their values are 1 and -1, so every result is 0."""
    import jittorinfer_amd as J
    n, scale = 2048, 2.0 ** -4
    step = torch.tensor(abs(number) / scale)
    step = float(torch.nextafter(step, step * 2) - step)
    gen = torch.Generator().manual_seed(dk)
    k, v = torch.zeros((n // 128, 128, 1, dk), dtype=dtype), torch.ones((n // 128, 128, 1, dv), dtype=dtype)
    base = (torch.randint(-64, 65, (n // 2,), generator=gen) / 4).repeat_interleave(2).view(-1, 128)
    k[:, :, 0, 1] = base.to(dtype)
    k[:, 0::2, 0, 0::16] = 64 * 7 / 16 * step
    k[:, 1::2, 0, 0] = 64 * 7 / 16 * step * (dk // 16)
    v[:, 1::2] = -1
    mask = torch.full((1, n), number, dtype=F16).to(gpu)
    # a score that is added to as it comes is off by half a step, 2^-24 of it, for every 16 columns, while it is no larger than `most` in log2 units; a larger one is off by half a step of a
    # number below 1024 where the mask is added last.  A softmax of two halves turns a difference of d into d / 2.  The weights are off by up to half a step each, either way: six
    # times what n of those come to.
    most = 2.0 ** 15 / dk if dtype == F16 else 1024.0
    off = max(2.0 ** -24 * most * dk / 16, 2 * 2.0 ** -15) * math.log(2) / 2
    p = torch.softmax(base.flatten().double() * scale, 0)
    off += 6 * R.half_step(dtype) / math.sqrt(3) * float(p.norm())
    bt, lens = torch.arange(n // 128, dtype=torch.int32)[None].to(gpu), torch.tensor([n], dtype=torch.int32, device=gpu)
    for new in (8, 100, 300):
        q = torch.zeros((new, 1, dk), dtype=dtype)
        q[:, 0, 0::16] = 2.0 ** -6
        q[:, 0, 1] = 1.0
        out = J.gqa_prompt_attn(q.to(gpu), k.to(gpu), v.to(gpu), bt, lens, scale=scale, causal=False, mask=mask)
        assert out.abs().max() <= off, (new, float(out.abs().max()) / off)
