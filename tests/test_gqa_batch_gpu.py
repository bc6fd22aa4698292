"""Attention of many query rows over the same keys on the GPU against plain forms in 64 bits (tests/gqa_batch_util.py)."""
import math

import pytest
import torch

from tests import gqa_batch_util as B
from tests import gqa_util as R
from tests.test_gqa_gpu import _near

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
WIDTHS = [(64, 64), (128, 128), (192, 128), (256, 256)]
NAN = float("nan")


def _starts(n):
    return torch.tensor([0] + n, dtype=torch.int32).cumsum(0).to(torch.int32)


def _case(seed, new, lens, width, heads, kv_heads, dk, dv, dtype, layout="cells", spare=2):
    """New tokens and rows of every sequence; pages hold what the lengths need and NaN everywhere else."""
    gen = torch.Generator().manual_seed(seed)
    pages = sum((min(max(n, 0), width * 128) + 127) // 128 for n in lens) + spare
    bt = R.make_table(gen, [min(n, width * 128) for n in lens], width, pages)
    k, v = (R.make_cache(gen, pages, kv_heads, d, dtype, layout, fill=NAN) for d in (dk, dv))
    for b, n in enumerate(lens):
        at = torch.arange(min(max(n, 0), width * 128))
        page = bt[b].long()[at // 128]
        k[page, at % 128] = torch.randn((len(at), kv_heads, dk), generator=gen).to(dtype)
        v[page, at % 128] = torch.randn((len(at), kv_heads, dv), generator=gen).to(dtype)
    q = torch.randn((sum(new), heads, dk), generator=gen).to(dtype)
    return q, k, v, bt, torch.tensor(lens, dtype=torch.int32), _starts(new)


def _check(gpu, q, k, v, bt, lens, starts, what="", given=True, **kw):
    import jittorinfer_amd as J
    scale = kw.pop("scale", 1 / math.sqrt(q.shape[2]))
    want, off = B.prompt(q, k, v, bt, lens, starts, scale, kw.get("logit_softcap", 0.0), kw.get("window", 0), kw.get("causal", True), kw.get("mask"))
    d = {n: (t.to(gpu) if isinstance(t, torch.Tensor) else t) for n, t in kw.items()}
    out = torch.full(want.shape, NAN, dtype=q.dtype, device=gpu)
    got = J.gqa_prompt_attn(q.to(gpu), k.to(gpu), v.to(gpu), bt.to(gpu), lens.to(gpu), starts.to(gpu) if given else None, scale=scale, out=out, **d)
    torch.cuda.synchronize()
    mine = ~torch.isnan(want[:, 0, 0])
    assert torch.isnan(got.cpu()[~mine]).all()
    _near(got[mine.to(gpu)], want[mine], off[mine], q.dtype, what)
    return got


NEW = [1, 0, 40, 129, 3, 64, 200]
LENS = [1, 70, 300, 129, 513, 64, 333]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dk,dv", WIDTHS)
@pytest.mark.parametrize("layout", ["cells", "heads"])
def test_prompt_widths_types_layouts(gpu, dk, dv, dtype, layout):
    _check(gpu, *_case(dk, NEW, LENS, 5, 8, 2, dk, dv, dtype, layout), "%s %s" % ((dk, dv), dtype))


@pytest.mark.parametrize("dk,dv", WIDTHS)
@pytest.mark.parametrize("new", [[1, 1, 1], [2, 9, 1], [16, 12, 14], [30, 40, 25]])
def test_prompt_few_tokens(gpu, dk, dv, new):
    """Blocks of 32, 64 and 128 rows: waves that share the keys of a tile."""
    _check(gpu, *_case(dk, new, [400, 130, 257], 4, 4, 2, dk, dv, BF16))
    _check(gpu, *_case(dk, new, [40, 130, 64], 4, 2, 2, dk, dv, F16), n_workgroups=7)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 7), (3, 1), (28, 4), (40, 1), (66, 1), (160, 1)])
def test_prompt_groups(gpu, heads, kv_heads):
    """Groups that no block holds a whole number of, and a token's heads in two blocks."""
    _check(gpu, *_case(heads, [5, 33, 0, 70], [5, 200, 3, 129], 2, heads, kv_heads, 64, 64, BF16))


@pytest.mark.parametrize("n_workgroups", [1, 2, 3, 5, 8, 13, 64, 1000])
@pytest.mark.parametrize("dk,dv", [(64, 64), (192, 128)])
def test_prompt_any_number_of_workgroups(gpu, dk, dv, n_workgroups):
    """Runs that hold several blocks, end inside one, or are empty."""
    _check(gpu, *_case(3, [100, 1, 0, 60, 128, 7], [700, 1, 0, 200, 128, 513], 6, 4, 2, dk, dv, F16), n_workgroups=n_workgroups)
    _check(gpu, *_case(4, [2, 1, 0, 3], [700, 1, 0, 200], 6, 4, 2, dk, dv, F16), n_workgroups=n_workgroups)


def test_prompt_more_sequences_than_lanes(gpu):
    gen = torch.Generator().manual_seed(5)
    new = [int(x) for x in torch.randint(0, 4, (300,), generator=gen)]
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 90, (300,), generator=gen))]
    new[:100] = lens[:100] = [0] * 100
    _check(gpu, *_case(5, new, lens, 1, 2, 1, 64, 64, BF16))


@pytest.mark.parametrize("window", [1, 5, 64, 100, 129, 1000])
def test_prompt_window(gpu, window):
    case = _case(6, [70, 1, 200, 33], [300, 128, 200, 411], 4, 4, 2, 128, 128, BF16)
    _check(gpu, *case, window=window)
    _check(gpu, *case, window=window, causal=False)
    _check(gpu, *case, window=window, n_workgroups=3)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("cap", [5.0, 50.0, 1e30])
def test_prompt_softcap(gpu, cap, dtype):
    _check(gpu, *_case(7, [1, 130, 20], [1, 200, 300], 3, 4, 1, 128, 128, dtype), logit_softcap=cap)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
@pytest.mark.parametrize("cap", [0.0, 9.0])
def test_prompt_scales(gpu, scale, cap):
    """A negative scale, none, and one that leaves a row to its largest score."""
    _check(gpu, *_case(8, [1, 130, 20], [1, 200, 300], 3, 4, 2, 64, 64, BF16), scale=scale, logit_softcap=cap)


def test_prompt_not_causal_and_equal_tokens(gpu):
    case = _case(9, [40, 40, 40], [40, 200, 300], 3, 4, 2, 64, 64, F16)
    _check(gpu, *case, causal=False)
    _check(gpu, *case, given=False)
    _check(gpu, *_case(9, [1, 1, 1], [40, 200, 300], 3, 4, 2, 64, 64, F16), given=False)


def test_prompt_lengths_outside_the_table_and_short_of_the_tokens(gpu):
    """A negative length is none, one past the table's room is that room, one below the number of new tokens leaves the first of them nothing."""
    case = _case(10, [4, 70, 20, 30], [0, 256, 200, 10], 2, 4, 2, 128, 128, BF16)
    case[4][0], case[4][1] = -7, 100000
    got = _check(gpu, *case)
    assert (got[:4] == 0).all() and (got[94:94 + 20] == 0).all() and (got[94 + 20:] != 0).any()


def _mask(gen, n_seq, n, dtype=F16):
    m = torch.zeros((n_seq, n), dtype=dtype)
    m[torch.rand((n_seq, n), generator=gen) < 0.3] = float("-inf")
    return m


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dk,dv", WIDTHS)
def test_prompt_mask(gpu, dk, dv, dtype):
    """Rows struck out, a sequence without any left, values that are not 0 (the lowest among them), keys and values of struck-out rows that are NaN or infinite."""
    q, k, v, bt, lens, starts = _case(11, [60, 129, 5, 40, 3], [300, 129, 64, 40, 200], 3, 6, 2, dk, dv, dtype)
    gen = torch.Generator().manual_seed(9)
    mask = _mask(gen, 5, 384)
    mask[2] = float("-inf")
    mask[3] = torch.randn(384, generator=gen).to(F16)
    mask[3, 5:9] = torch.finfo(F16).min
    for b, n in enumerate(lens.tolist()):
        for i in torch.nonzero(mask[b, :n] == float("-inf"))[:, 0].tolist():
            k[bt[b, i // 128], i % 128] = float("nan") if i % 2 else float("inf")
            v[bt[b, i // 128], i % 128] = float("inf") if i % 3 else float("nan")
    got = _check(gpu, q, k, v, bt, lens, starts, mask=mask)
    assert (got[189:194] == 0).all()
    for cut in (1, 64, 130, 299):
        _check(gpu, q, k, v, bt, lens, starts, mask=mask[:, :cut])
    wide = torch.full((5, 385), NAN, dtype=F16)[:, 1:]
    wide[:, :] = mask
    _check(gpu, q, k, v, bt, lens, starts, mask=wide, window=90, logit_softcap=20.0)
    if dk <= 128:
        _check(gpu, q[:64], k, v, bt, lens, _starts([10, 20, 5, 5, 3]), mask=mask)


@pytest.mark.parametrize("new", [[60, 129, 40], [2, 9, 1]])
@pytest.mark.parametrize("dk,dv", WIDTHS)
def test_prompt_mask_of_the_lowest_value_alone(gpu, dk, dv, new):
    """A number added to every row of a sequence changes nothing but the scores' rounding; rows of the lowest value beside others have no weight."""
    import jittorinfer_amd as J
    q, k, v, bt, lens, starts = _case(13, new, [300, 129, 260], 3, 6, 2, dk, dv, F16)
    low = torch.finfo(F16).min
    mask = torch.full((3, 384), low, dtype=F16)
    mask[1, ::2] = -30000.0                     # (a page of rows and one: every token sees one of these)
    hard = torch.zeros((3, 384), dtype=F16)
    hard[1, 1::2] = float("-inf")
    scale = dk ** -0.5
    want, off = B.prompt(q, k, v, bt, lens, starts, scale, mask=hard)
    # a score and the number are added in log2 units, below 2^17 in size: the sum is off by half a step, 2^-8, which is 2^-8 ln 2 of a weight, and a
    # softmax turns that into twice as much of a result; the score itself as without a mask
    gathered = torch.zeros_like(off)
    for b in range(3):
        n = int(lens[b])
        at = torch.arange(n)
        vv = v[bt[b].long()[at // 128], at % 128].double().abs().amax(0).repeat_interleave(3, 0)
        gathered[starts[b]:starts[b + 1]] = vv
    off = off + 2 * 2.0 ** -8 * math.log(2) * gathered
    out = J.gqa_prompt_attn(q.to(gpu), k.to(gpu), v.to(gpu), bt.to(gpu), lens.to(gpu), starts.to(gpu), scale=scale, mask=mask.to(gpu))
    _near(out, want, off, F16)
    # and as a whole: those errors are of either sign and independent, sqrt(3) below the bound each, and a result is off by its weights' errors as it is made of its weights
    err = (out.cpu().double() - want).norm() / want.norm()
    assert err < 2.0 ** -8 * math.log(2), err


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dk,dv,new", [(64, 64, 300), (128, 128, 300), (192, 128, 300), (256, 256, 300), (64, 64, 7), (128, 128, 14), (256, 256, 14)])
def test_prompt_infinities_of_rows_not_seen(gpu, dk, dv, new, dtype):
    """A key and a value that are NaN or infinite reach the tokens that see them, and no others."""
    q, k, v, bt, lens, starts = _case(12, [new, new], [300, 310], 3, 4, 2, dk, dv, dtype)
    clean, _ = B.prompt(q, k, v, bt, lens, starts, 0.1, window=150)
    at = 297
    page = bt[0, at // 128].long()
    kinds = [float("inf"), float("-inf"), NAN]
    for c in range(dv):
        if c % 5 < 3:
            v[page, at % 128, 0, c] = kinds[c % 5]
    import jittorinfer_amd as J
    for n in (0, 5):
        got = J.gqa_prompt_attn(q.to(gpu), k.to(gpu), v.to(gpu), bt.to(gpu), lens.to(gpu), starts.to(gpu), scale=0.1, window=150, n_workgroups=n).cpu().double()
        first = at - (300 - new)                             # the token whose row it is
        unseen = got[:first]
        assert torch.isfinite(unseen).all() and torch.isfinite(got[new:]).all() and torch.isfinite(got[:new, 2:]).all()
        assert (got[:, :, 3::5] - clean[:, :, 3::5]).abs().max() < 0.05
        for c in range(dv):
            seen = got[first:new, :2, c]
            if c % 5 == 0:
                assert (seen == float("inf")).all()
            elif c % 5 == 1:
                assert (seen == float("-inf")).all()
            elif c % 5 == 2:
                assert torch.isnan(seen).all()
    k[page, at % 128, 0] = NAN
    got = J.gqa_prompt_attn(q.to(gpu), k.to(gpu), v.to(gpu), bt.to(gpu), lens.to(gpu), starts.to(gpu), scale=0.1, window=150).cpu()
    assert torch.isfinite(got[:first]).all() and torch.isnan(got[first:new, :2]).all() and torch.isfinite(got[new:]).all()


def test_prompt_bad_pages_and_tokens_of_no_sequence(gpu):
    """Rows of a page id outside the pool count as masked; tokens before the first sequence's and behind the last one's keep what out held."""
    q, k, v, bt, lens, starts = _case(13, [60, 70, 30], [300, 256, 129], 3, 4, 2, 64, 64, BF16)
    bt[0, 1], bt[1, 0], bt[2] = -1, 10 ** 9, k.shape[0]
    _check(gpu, q, k, v, bt, lens, starts)
    q = torch.cat((q, q, q))
    got = _check(gpu, q, k, v, bt, lens, starts + 17)
    assert torch.isnan(got[:17]).all() and torch.isnan(got[17 + 160:]).all() and torch.isfinite(got[17:177]).all()


def test_prompt_strides(gpu):
    """q a view of a projection's output, out a view with other strides, caches that share their rows' memory side by side, an empty batch."""
    import jittorinfer_amd as J
    q, k, v, bt, lens, starts = _case(14, [60, 70], [300, 256], 3, 4, 2, 64, 64, BF16)
    want, off = B.prompt(q, k, v, bt, lens, starts, 0.125)
    wide = torch.full((130, 4, 200), NAN, dtype=BF16)
    wide[..., 8:72] = q
    both = torch.full((k.shape[0], 128, 2, 136), NAN, dtype=BF16)
    both[..., :64], both[..., 72:] = k, v
    both = both.to(gpu)
    out = torch.full((4, 130, 100), NAN, dtype=BF16, device=gpu)
    view = out.transpose(0, 1)[..., 4:68]
    got = J.gqa_prompt_attn(wide.to(gpu)[..., 8:72], both[..., :64], both[..., 72:], bt.to(gpu), lens.to(gpu), starts.to(gpu), scale=0.125, out=view)
    assert got.data_ptr() == view.data_ptr()
    _near(view, want, off, BF16)
    assert torch.isnan(out[..., :4]).all() and torch.isnan(out[..., 68:]).all()
    none = J.gqa_prompt_attn(q[:0].to(gpu), k.to(gpu), v.to(gpu), bt.to(gpu), lens.to(gpu), (starts * 0).to(gpu), scale=0.125)
    assert none.shape == (0, 4, 64)
    none = J.gqa_prompt_attn(q[:0].to(gpu), k.to(gpu), v.to(gpu), bt[:0].to(gpu), lens[:0].to(gpu), scale=0.125)
    assert none.shape == (0, 4, 64)


@pytest.mark.parametrize("dtype,dk,dv", [(BF16, 128, 128), (F16, 64, 64)])
def test_prompt_long(gpu, dtype, dk, dv):
    """A chunk behind a long context, and many tokens: against the same formula in f32 on the GPU, whose own error is below what is allowed."""
    import jittorinfer_amd as J
    q, k, v, bt, lens, starts = _case(15, [37, 1500], [20001, 1500], 160, 4, 2, dk, dv, dtype)
    want, off = B.prompt(q, k, v, bt, lens, starts, 0.1)
    got = J.gqa_prompt_attn(q.to(gpu), k.to(gpu), v.to(gpu), bt.to(gpu), lens.to(gpu), starts.to(gpu), scale=0.1)
    _near(got, want, off, dtype)
    again = J.gqa_prompt_attn(q.to(gpu), k.to(gpu), v.to(gpu), bt.to(gpu), lens.to(gpu), starts.to(gpu), scale=0.1)
    assert torch.equal(got, again)


def test_prompt_of_one_token_is_gqa_attn(gpu):
    """One new token a sequence: what gqa_attn answers, but for the rounding of the weights."""
    import jittorinfer_amd as J
    q, k, v, bt, lens, starts = (t.to(gpu) for t in _case(16, [1] * 5, [1, 70, 300, 129, 511], 4, 8, 2, 128, 128, F16))
    a = J.gqa_attn(q, k, v, bt, lens, scale=0.1).double()
    b = J.gqa_prompt_attn(q, k, v, bt, lens, scale=0.1).double()
    assert (a - b).abs().max() < 2.0 ** -10 * v[torch.isfinite(v)].abs().max().double()


# ---------------------------------------------------------------- an encoder's states

def _states(seed, new, n, heads, kv_heads, dk, dv, dtype, most=None):
    gen = torch.Generator().manual_seed(seed)
    most = most or max(n + [1])
    k, v = (torch.full((len(n), most, kv_heads, d), NAN, dtype=dtype) for d in (dk, dv))
    for b, x in enumerate(n):
        k[b, :x] = torch.randn((x, kv_heads, dk), generator=gen).to(dtype)
        v[b, :x] = torch.randn((x, kv_heads, dv), generator=gen).to(dtype)
    return torch.randn((sum(new), heads, dk), generator=gen).to(dtype), k, v, _starts(new), torch.tensor(n, dtype=torch.int32)


def _cross(gpu, q, k, v, starts, lens, given=True, packed=False, **kw):
    import jittorinfer_amd as J
    scale = 1 / math.sqrt(q.shape[2])
    want, off = B.cross(q, k, v, starts, lens, scale, kw.get("logit_softcap", 0.0), kw.get("mask"))
    if packed:
        at = {"kv_starts": _starts(lens.tolist())}
        k, v = (torch.cat([x[b, :n] for b, n in enumerate(lens.tolist())]) for x in (k, v))
    else:
        at = {"kv_lens": lens}
    d = {n: (t.to(gpu) if isinstance(t, torch.Tensor) else t) for n, t in {**kw, **at}.items()}
    got = J.gqa_cross_attn(q.to(gpu), k.to(gpu), v.to(gpu), q_starts=starts.to(gpu) if given else None, scale=scale, **d)
    torch.cuda.synchronize()
    _near(got, want, off, q.dtype)
    return got


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dk,dv", WIDTHS)
@pytest.mark.parametrize("packed", [False, True])
def test_cross_widths_types(gpu, dk, dv, dtype, packed):
    _cross(gpu, *_states(dk, [40, 1, 129, 0, 7], [300, 1, 77, 5, 0], 4, 2, dk, dv, dtype), packed=packed)
    _cross(gpu, *_states(dk, [3, 1, 2, 1, 7], [300, 1, 77, 5, 0], 4, 4, dk, dv, dtype), packed=packed)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dk,dv", WIDTHS)
@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (8, 2), (40, 1), (24, 8)])
@pytest.mark.parametrize("packed", [False, True])
def test_cross_of_one_token(gpu, dk, dv, dtype, heads, kv_heads, packed):
    """A decode step: one token a sequence, over states of odd numbers, none among them."""
    case = _states(dk + heads, [1] * 7, [300, 1, 129, 0, 640, 31, 128], heads, kv_heads, dk, dv, dtype)
    got = _cross(gpu, *case, given=False, packed=packed)
    assert (got[3] == 0).all()
    _cross(gpu, *case, given=True, packed=packed, n_workgroups=5)


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("new", [1, 30])
def test_cross_mask_and_cap(gpu, new, given):
    """Padding masked, a sequence without any state left, NaN and infinities behind the mask and behind the lengths."""
    q, k, v, starts, lens = _states(20, [new] * 4, [300, 77, 129, 5], 4, 2, 64, 64, BF16, most=310)
    gen = torch.Generator().manual_seed(3)
    mask = _mask(gen, 4, 310)
    mask[1] = float("-inf")
    for b in range(4):
        k[b, mask[b] == float("-inf")] = NAN
        v[b, mask[b] == float("-inf")] = float("inf")
    got = _cross(gpu, q, k, v, starts, lens, given=given, mask=mask)
    assert (got[new:2 * new] == 0).all()
    _cross(gpu, q, k, v, starts, lens, given=given, mask=mask[:, :50], logit_softcap=10.0)


def test_cross_lengths_and_starts_out_of_range(gpu):
    """No lengths: all states; lengths below 0 and past the states; starts outside the buffer, sequences whose states overlap."""
    import jittorinfer_amd as J
    q, k, v, starts, lens = _states(21, [9, 4, 2], [200, 200, 200], 4, 2, 64, 64, F16)
    d = [t.to(gpu) for t in (q, k, v)]
    want, off = B.cross(q, k, v, starts, lens, 0.125)
    _near(J.gqa_cross_attn(*d, q_starts=starts.to(gpu), scale=0.125), want, off, F16)
    odd = torch.tensor([-3, 1000, 5], dtype=torch.int32)
    want, off = B.cross(q, k, v, starts, odd, 0.125)
    _near(J.gqa_cross_attn(*d, q_starts=starts.to(gpu), kv_lens=odd.to(gpu), scale=0.125), want, off, F16)
    flat = [t.reshape(600, 2, 64) for t in (k, v)]
    at, n = torch.tensor([-1, 550, 100], dtype=torch.int32), torch.tensor([50, 500, 300], dtype=torch.int32)
    want, off = B.cross(q, *flat, starts, n, 0.125, kv_starts=at)
    got = J.gqa_cross_attn(d[0], *[t.to(gpu) for t in flat], q_starts=starts.to(gpu), kv_starts=at.to(gpu), kv_lens=n.to(gpu), scale=0.125)
    _near(got, want, off, F16)
    assert (got[:9] == 0).all()
    at[1] = 601
    got = J.gqa_cross_attn(d[0], *[t.to(gpu) for t in flat], q_starts=starts.to(gpu), kv_starts=at.to(gpu), kv_lens=n.to(gpu), scale=0.125)
    assert (got[:13] == 0).all() and (got[13:] != 0).any()


def test_cross_without_states(gpu):
    """No row at all, padded and packed: zeros."""
    import jittorinfer_amd as J
    for new in (1, 50):
        q = torch.randn((2 * new, 4, 64), device=gpu).to(F16)
        none = torch.empty((2, 0, 2, 64), dtype=F16, device=gpu)
        zero = torch.zeros(3, dtype=torch.int32, device=gpu)
        for kw in (dict(), dict(kv_lens=zero[:2]), dict(logit_softcap=9.0)):
            out = torch.full_like(q, NAN)
            assert (J.gqa_cross_attn(q, none, none, scale=0.1, out=out, **kw) == 0).all()
        out = torch.full_like(q, NAN)
        assert (J.gqa_cross_attn(q, none[0], none[0], kv_starts=zero, scale=0.1, out=out) == 0).all()


@pytest.mark.parametrize("new", [1, 20])
def test_cross_strides(gpu, new):
    """States with heads outermost, expanded over the heads or over the sequences, out given."""
    import jittorinfer_amd as J
    q, k, v, starts, lens = _states(22, [new] * 3, [150, 150, 150], 4, 2, 64, 64, BF16)
    want, off = B.cross(q, k, v, starts, lens, 0.125)
    k2, v2 = (t.transpose(1, 2).contiguous().transpose(1, 2).to(gpu) for t in (k, v))
    out = torch.full((3 * new, 4, 64), NAN, dtype=BF16, device=gpu)
    got = J.gqa_cross_attn(q.to(gpu), k2, v2, scale=0.125, out=out)
    assert got.data_ptr() == out.data_ptr()
    _near(got, want, off, BF16)
    one = [t[:1, :, :1].expand(3, 150, 2, 64) for t in (k, v)]
    want, off = B.cross(q, *one, starts, lens, 0.125)
    _near(J.gqa_cross_attn(q.to(gpu), *[t[:1, :, :1].to(gpu).expand(3, 150, 2, 64) for t in (k, v)], scale=0.125), want, off, BF16)


# ---------------------------------------------------------------- shared prefixes

def _shared(seed, groups, own, heads, kv_heads, dk, dv, dtype, layout="cells", before=0, spare=2, width=None):
    """groups: (sequences, shared rows); own: rows of its own of every sequence; the first `before` sequences and those past the groups share nothing.  Whole
    pages of a prefix are the same pages, the one it ends in is each sequence's own copy."""
    gen = torch.Generator().manual_seed(seed)
    n_seq = len(own)
    shared = [0] * before + [p for m, p in groups for _ in range(m)]
    shared += [0] * (n_seq - len(shared))
    starts = torch.tensor([before] + [m for m, _ in groups], dtype=torch.int32).cumsum(0).to(torch.int32)
    lens = [s + o for s, o in zip(shared, own)]
    width = width or max(1, max((n + 127) // 128 for n in lens))
    n_pages = sum(p // 128 for _, p in groups) + sum((n + 127) // 128 for n in lens) + spare
    ids = torch.randperm(n_pages, generator=gen).tolist()
    k, v = (R.make_cache(gen, n_pages, kv_heads, d, dtype, layout, fill=NAN) for d in (dk, dv))
    bt = torch.zeros((n_seq, width), dtype=torch.int32)
    fill = lambda page, rows: [c.__setitem__((page, slice(0, rows)), torch.randn((rows, kv_heads, c.shape[3]), generator=gen).to(dtype)) for c in (k, v)]
    for g, (m, p) in enumerate(groups):
        pages = [ids.pop() for _ in range(p // 128)]
        for page in pages:
            fill(page, 128)
        for b in range(int(starts[g]), int(starts[g + 1])):
            bt[b, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
    for b in range(n_seq):
        for j in range(shared[b] // 128, (lens[b] + 127) // 128):
            bt[b, j] = ids.pop()
            fill(int(bt[b, j]), min(128, lens[b] - j * 128))
    for g, (m, p) in enumerate(groups):
        for b in range(int(starts[g]) + 1, int(starts[g + 1])):
            if p % 128:
                for c in (k, v):
                    c[bt[b, p // 128].long(), :p % 128] = c[bt[int(starts[g]), p // 128].long(), :p % 128]
    q = torch.randn((n_seq, heads, dk), generator=gen).to(dtype)
    return q, k, v, bt, torch.tensor(lens, dtype=torch.int32), starts, torch.tensor([p for _, p in groups], dtype=torch.int32)


def _wide(bt, k, v):
    """A block table with room for 2^28 bytes of rows, pages that are none behind those it has: the prefixes are worked on by themselves."""
    row = k.shape[2] * (k.shape[3] + v.shape[3]) * 2
    width = -(-2 ** 28 // (bt.shape[0] * 128 * row))
    return torch.cat([bt, torch.full((bt.shape[0], max(0, width - bt.shape[1])), -1, dtype=torch.int32, device=bt.device)], 1)


def _prefix(gpu, q, k, v, bt, lens, starts, plens, nan=(), **kw):
    """Twice, with a block table that has little room and one that has much.  nan: sequences that see a NaN."""
    import jittorinfer_amd as J
    scale = 1 / math.sqrt(q.shape[2])
    each = torch.arange(len(lens) + 1)
    want, off = B.prompt(q, k, v, bt, lens, each, scale, kw.get("logit_softcap", 0.0), 0, True, kw.get("mask"))
    d = {n: (t.to(gpu) if isinstance(t, torch.Tensor) else t) for n, t in kw.items()}
    fine = [b for b in range(len(lens)) if b not in nan]
    for table in (bt, _wide(bt, k, v)):
        got = J.gqa_prefix_attn(*[t.to(gpu) for t in (q, k, v, table, lens, starts, plens)], scale=scale, **d)
        torch.cuda.synchronize()
        assert torch.isnan(got[list(nan)]).all() and torch.isnan(want[list(nan)]).all()
        _near(got[fine], want[fine], off[fine], q.dtype)
    return got


GROUPS = [(3, 300), (1, 128), (2, 77), (4, 640)]
OWN = [5, 0, 130, 1, 300, 64, 10, 0, 1, 200, 129, 7]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dk,dv", WIDTHS)
@pytest.mark.parametrize("layout", ["cells", "heads"])
def test_prefix_widths_types_layouts(gpu, dk, dv, dtype, layout):
    _prefix(gpu, *_shared(dk, GROUPS, OWN, 8, 2, dk, dv, dtype, layout, before=1))


@pytest.mark.parametrize("dk,dv", WIDTHS)
@pytest.mark.parametrize("members,heads,kv_heads", [(2, 4, 4), (20, 8, 4), (40, 4, 2), (9, 7, 1), (70, 8, 2), (5, 40, 1)])
def test_prefix_blocks_of_all_sizes(gpu, dk, dv, members, heads, kv_heads):
    """32, 64 and 128 rows a block, groups that fill several, heads of one sequence in two blocks."""
    gen = torch.Generator().manual_seed(members)
    own = [int(x) for x in torch.randint(0, 40, (members,), generator=gen)]
    _prefix(gpu, *_shared(members, [(members, 500)], own, heads, kv_heads, dk, dv, BF16))
    _prefix(gpu, *_shared(members, [(members, 500)], own, heads, kv_heads, dk, dv, F16), n_workgroups=5)


@pytest.mark.parametrize("n_workgroups", [1, 2, 3, 7, 16, 100])
def test_prefix_any_number_of_workgroups(gpu, n_workgroups):
    _prefix(gpu, *_shared(3, GROUPS, OWN, 4, 2, 64, 64, BF16), n_workgroups=n_workgroups)


def test_prefix_four_heads_a_workgroup_behind_it(gpu):
    """A block table with room for many pages: the rows behind the prefixes are read by waves of a KV head each."""
    _prefix(gpu, *_shared(4, GROUPS, OWN, 16, 8, 128, 128, BF16, width=40))
    _prefix(gpu, *_shared(4, GROUPS, OWN, 16, 8, 128, 128, F16, width=40), n_workgroups=3)
    _prefix(gpu, *_shared(5, [(3, 300), (9, 200)], OWN, 40, 1, 128, 128, BF16, width=300))


def test_prefix_groups_of_none_and_lengths_out_of_range(gpu):
    """Groups without a sequence, prefixes of no row, below 0 and past the table's room, sequences shorter than their prefix, sequences without a row, no group at all."""
    import jittorinfer_amd as J
    q, k, v, bt, lens, starts, plens = _shared(6, [(5, 512)], [0, 1, 30, 0, 9, 77], 4, 2, 64, 64, BF16)
    lens[:4] = torch.tensor([0, 100, 512, 300])
    got = _prefix(gpu, q, k, v, bt, lens, starts, plens)
    assert (got[0] == 0).all()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)
    for s, n in ((i32(0, 0, 5, 5, 5), i32(100, 512, 3, 0)), (i32(0, 5), i32(0)), (i32(0, 5), i32(-9)), (i32(2, 5), i32(256)), (i32(0, 3, 5), i32(512, 128)), (i32(0), i32())):
        _prefix(gpu, q, k, v, bt, lens, s, n)
    q, k, v, bt, lens, starts, plens = _shared(7, [(3, 512)], [0, 0, 0], 4, 2, 64, 64, F16)
    _prefix(gpu, q, k, v, bt, lens, starts, i32(100000))
    lens[1] = 100000
    _prefix(gpu, q, k, v, bt, lens, starts, plens)
    none = J.gqa_prefix_attn(q[:0].to(gpu), k.to(gpu), v.to(gpu), bt[:0].to(gpu), lens[:0].to(gpu), (starts * 0).to(gpu), plens.to(gpu), scale=1.0)
    assert none.shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dk,dv", [(64, 64), (192, 128), (256, 256)])
def test_prefix_mask_and_cap(gpu, dk, dv, dtype):
    """Every sequence its own mask over the shared rows, one that leaves nothing; keys and values that all of them but one take out are NaN or infinite."""
    q, k, v, bt, lens, starts, plens = _shared(8, GROUPS, OWN, 6, 2, dk, dv, dtype, before=1)
    mask = _mask(torch.Generator().manual_seed(5), 12, bt.shape[1] * 128)
    mask[:, 10:14] = float("-inf")
    mask[:, 130] = float("-inf")
    mask[8] = float("-inf")
    mask[9] = torch.randn(mask.shape[1], generator=torch.Generator().manual_seed(6)).to(F16)
    mask[9, 130] = float("-inf")
    for b in range(12):
        for i in (10, 11, 12, 13, 130):
            if i < lens[b]:
                k[bt[b, i // 128].long(), i % 128] = NAN
                v[bt[b, i // 128].long(), i % 128] = float("inf") if i % 2 else NAN
    got = _prefix(gpu, q, k, v, bt, lens, starts, plens, nan=[9], mask=mask)
    assert (got[8] == 0).all()
    _prefix(gpu, q, k, v, bt, lens, starts, plens, nan=[9], mask=mask[:, :200], logit_softcap=15.0, n_workgroups=4)
    _prefix(gpu, q, k, v, bt, lens, starts, plens, nan=[9], mask=mask[:, :90])
    mask[9, 10:14] = float("-inf")
    _prefix(gpu, q, k, v, bt, lens, starts, plens, mask=mask)
    # a shared row that half of a group of 4 masks: the others' results are not finite, theirs are
    import jittorinfer_amd as J
    b0 = int(starts[3])
    at = 200
    mask[b0:b0 + 4, at] = 0.0
    mask[b0, at] = mask[b0 + 2, at] = float("-inf")
    v[bt[b0, at // 128].long(), at % 128] = float("inf")
    got = J.gqa_prefix_attn(*[t.to(gpu) for t in (q, k, v, _wide(bt, k, v), lens, starts, plens)], scale=0.1, mask=mask.to(gpu)).cpu()
    assert (got[b0 + 1] == float("inf")).all() and (got[b0 + 3] == float("inf")).all()
    for b in set(range(12)) - {b0 + 1, b0 + 3}:
        assert torch.isfinite(got[b]).all(), b


def test_prefix_bad_pages(gpu):
    q, k, v, bt, lens, starts, plens = _shared(9, [(3, 512), (2, 300)], [100, 3, 50, 9, 200, 10], 4, 2, 64, 64, BF16)
    bt[:3, 1], bt[4, 2], bt[5] = -1, k.shape[0], 10 ** 9
    import jittorinfer_amd as J
    got = J.gqa_prefix_attn(*[t.to(gpu) for t in (q, k, v, _wide(bt, k, v), lens, starts, plens)], scale=0.125)
    # the shared rows of the page that sequence 4 lacks are read through sequence 3's table; its own ones of that page, 300 .. 383, count as masked
    own, mask = bt.clone(), torch.zeros((6, bt.shape[1] * 128), dtype=F16)
    own[4, 2] = bt[3, 2]
    mask[4, 300:384] = float("-inf")
    want, off = B.prompt(q, k, v, own, lens, torch.arange(7), 0.125, mask=mask)
    _near(got, want, off, BF16)


def test_prefix_many_sequences(gpu):
    gen = torch.Generator().manual_seed(5)
    own = [int(x) for x in torch.randint(0, 200, (310,), generator=gen)]
    _prefix(gpu, *_shared(10, [(100, 200), (1, 128), (150, 300), (40, 256)], own, 2, 1, 64, 64, BF16, before=9))


def test_prefix_is_gqa_attn(gpu):
    """The same call without groups is gqa_attn; with them it differs by the rounding of the weights over the prefix."""
    import jittorinfer_amd as J
    q, k, v, bt, lens, starts, plens = (t.to(gpu) for t in _shared(11, GROUPS, OWN, 8, 2, 128, 128, BF16, before=1))
    a = J.gqa_attn(q, k, v, bt, lens, scale=0.1)
    assert torch.equal(a, J.gqa_prefix_attn(q, k, v, bt, lens, starts[:1], plens[:0], scale=0.1))
    assert torch.equal(a, J.gqa_prefix_attn(q, k, v, bt, lens, starts, plens, scale=0.1))       # (a table with little room)
    bt = _wide(bt, k, v)
    b = J.gqa_prefix_attn(q, k, v, bt, lens, starts, plens, scale=0.1)
    assert (a.double() - b.double()).abs().max() < 2.0 ** -6 * v[torch.isfinite(v)].abs().max().double()
    assert torch.equal(b, J.gqa_prefix_attn(q, k, v, bt, lens, starts, plens, scale=0.1))


@pytest.mark.parametrize("new,lens", [([900, 0, 700, 130], [1000, 70, 700, 1300]), ([2, 1600, 3], [12000, 1600, 3]), ([3200], [3200]), ([1600, 1600], [100, 1700])])
def test_prompt_of_many_blocks(gpu, new, lens):
    """Blocks enough for a workgroup each, by what the device finds (a few that are much longer than the others among them) or in any case."""
    case = _case(17, new, lens, 96, 64, 64, 64, 64, BF16)
    _check(gpu, *case, window=300)
    if sum(lens) < 3000:
        _check(gpu, *case)
