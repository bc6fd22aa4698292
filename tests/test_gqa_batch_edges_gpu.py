"""Attention of many query rows over the same keys on the GPU: ways that a call goes by its sizes, and masks of large numbers."""
import math

import pytest
import torch

from tests import gqa_util as R
from tests.test_gqa_batch import CALLS
from tests.test_gqa_batch_edges import REFUSED
from tests.test_gqa_batch_gpu import _case, _check, _prefix, _shared, _wide
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


@pytest.mark.parametrize("dk,dtype,heads", [(64, F16, 1600), (128, BF16, 1600), (256, BF16, 1600)])
@pytest.mark.parametrize("new,rows", [(300, 300), (257, 400)])
def test_prompt_of_one_sequence_with_blocks_for_all(gpu, dk, dtype, heads, new, rows):
    """Four blocks and more for every workgroup that the card holds: one sequence's blocks are taken whole whatever its length, and no join is launched."""
    assert new // 128 * heads >= 4 * 256 * 3                                 # (blocks of 128 rows of all KV heads; three workgroups a CU at most)
    case = _case(new + dk, [new], [rows], -(-rows // 128), heads, heads, dk, dk, dtype)
    _check(gpu, *case)


def _many(gen, n_seq, long_at, long_rows, chunk):
    """One new token of most sequences, none of some, behind a few rows; one sequence far back in the batch is longer than all others together."""
    new = [1 if int(x) else 0 for x in torch.randint(0, 4, (n_seq,), generator=gen)]
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 90, (n_seq,), generator=gen))]
    new[long_at], lens[long_at] = chunk, long_rows
    return new, lens


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n_workgroups", [0, 1, 7, 64, 1000])
@pytest.mark.parametrize("n_seq,long_at,long_rows,chunk", [(300, 299, 90, 1), (300, 130, 6000, 1), (129, 128, 5000, 40), (65, 64, 9000, 3), (200, 70, 4000, 300)])
def test_prompt_runs_of_more_sequences_than_lanes(gpu, n_seq, long_at, long_rows, chunk, n_workgroups, causal):
    """Equal runs that begin and end in any set of 64 sequences: of a given number of workgroups, or because one sequence is far longer than a share."""
    gen = torch.Generator().manual_seed(n_seq)
    new, lens = _many(gen, n_seq, long_at, long_rows, chunk)
    _check(gpu, *_case(n_seq, new, lens, -(-max(lens) // 128), 4, 2, 64, 64, BF16), n_workgroups=n_workgroups, causal=causal)


@pytest.mark.parametrize("n_workgroups", [0, 1, 7, 64, 1000])
@pytest.mark.parametrize("dk,dtype", [(64, BF16), (128, F16)])
def test_prefixes_of_more_groups_than_lanes(gpu, dk, dtype, n_workgroups):
    """150 groups of one to four sequences, some without a shared row, one far back whose prefix is longer than all others together."""
    gen = torch.Generator().manual_seed(dk)
    groups = [(1 + int(m), [0, 77, 128, 200][int(p)]) for m, p in zip(torch.randint(0, 4, (150,), generator=gen), torch.randint(0, 4, (150,), generator=gen))]
    groups[100] = (3, 5000)
    own = [int(x) for x in torch.randint(0, 60, (2 + sum(m for m, _ in groups),), generator=gen)]
    _prefix(gpu, *_shared(dk, groups, own, 4, 2, dk, dk, dtype, before=2), n_workgroups=n_workgroups)


def test_python_entry_points_refuse_what_is_wrong(gpu):
    """The calls of the same table on tensors that there are: the accepted ones run, a wrong result tensor is refused like any other, before a launch."""
    source = CALLS.split("J.capi.native()\n")[0].replace("with FakeTensorMode():", "if True:").replace("torch.empty(", "torch.zeros(")
    scope = {}
    exec(source, scope)
    assert set(scope["calls"]) == set(REFUSED)
    for name, call in scope["calls"].items():
        if name.endswith("_alloc"):
            assert torch.isfinite(call()).all()
            continue
        with pytest.raises((AssertionError, TypeError, RuntimeError)) as e:
            call()
        kind, text = REFUSED[name] or ("AssertionError", "result.take(a, q, outp)")
        assert type(e.value).__name__ == kind and text in str(e.value), (name, e.value)
    torch.cuda.synchronize()
