"""Attention of many query rows over the same keys on the GPU: ways that a call goes by its sizes, and masks of large numbers."""
import pytest
import torch

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
