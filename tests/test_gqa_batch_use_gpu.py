"""Attention of many query rows over the same keys as a serving loop uses it: in graphs, on streams of the caller, from threads, and all of it in a row."""
import threading

import pytest
import torch

from tests import gqa_batch_util as B
from tests import gqa_util as R
from tests.test_gqa_batch_gpu import GROUPS, NAN, OWN, _case, _shared, _starts, _states, _wide
from tests.test_gqa_gpu import BF16, F16, _near

pytestmark = pytest.mark.gpu


def _calls(gpu, seed=0, dtype=BF16):
    """One call of each operator and form: (call(out=, stream=), what it gives)."""
    import jittorinfer_amd as J
    p = [t.to(gpu) for t in _case(30 + seed, [70, 1, 200, 33], [300, 128, 500, 900], 8, 8, 2, 128, 128, dtype)]
    x = [t.to(gpu) for t in _states(31 + seed, [40, 1, 129], [700, 30, 900], 8, 2, 64, 64, dtype)]
    one = [t.to(gpu) for t in _states(32 + seed, [1] * 6, [700, 30, 900, 0, 128, 500], 8, 8, 64, 64, dtype)]
    s = [t.to(gpu) for t in _shared(33 + seed, GROUPS, OWN, 8, 2, 128, 128, dtype, before=1)]
    far = _wide(s[3], s[1], s[2])
    calls = [lambda **kw: J.gqa_prompt_attn(*p, scale=0.1, **kw), lambda **kw: J.gqa_cross_attn(*x[:3], q_starts=x[3], kv_lens=x[4], scale=0.1, **kw),
             lambda **kw: J.gqa_cross_attn(*one[:3], kv_lens=one[4], scale=0.1, **kw), lambda **kw: J.gqa_prefix_attn(*s, scale=0.1, **kw),
             lambda **kw: J.gqa_prefix_attn(*s[:3], far, *s[4:], scale=0.1, **kw)]
    return [(c, c()) for c in calls]


def test_on_another_stream(gpu):
    calls = _calls(gpu)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for call, want in calls:
        with pytest.raises(ValueError):
            call(stream=side.cuda_stream)
        out = torch.empty_like(want)
        call(out=out, stream=side.cuda_stream)
        with torch.cuda.stream(side):
            again = call()
        side.synchronize()
        assert torch.equal(out, want) and torch.equal(again, want)


def test_forked_branches_of_one_capture(gpu):
    """On the current stream and, through stream=, on a side stream of the same capture, side by side at every replay: neither uses the other's scratch."""
    calls = _calls(gpu) + _calls(gpu, 100)
    outs = [torch.empty_like(w) for _, w in calls]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fork = torch.cuda.Event()
        fork.record()
        side.wait_event(fork)
        for i, ((call, _), out) in enumerate(zip(calls, outs)):
            call(out=out, stream=side.cuda_stream if i % 2 else None)
        torch.cuda.current_stream().wait_stream(side)
    for step in range(4):
        for o in outs:
            o.fill_(NAN)
        calls[0][0]()                                                  # eager work between the replays
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, (_, w) in zip(outs, calls)), step


def test_two_graphs_side_by_side(gpu):
    """Captured on one stream, replayed on two at once, with eager calls on a third."""
    sets = [_calls(gpu, s) for s in (0, 50)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for calls in sets:
        o = [torch.empty_like(w) for _, w in calls]
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            for (call, _), out in zip(calls, o):
                call(out=out)
        graphs.append(g)
        outs.append(o)
    streams = [torch.cuda.Stream() for _ in graphs]
    for step in range(4):
        for o in outs:
            for t in o:
                t.fill_(NAN)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        eager = [call() for call, _ in sets[0]]
        torch.cuda.synchronize()
        for calls, o in zip(sets, outs):
            assert all(torch.equal(a, w) for a, (_, w) in zip(o, calls)), step
        assert all(torch.equal(a, w) for a, (_, w) in zip(eager, sets[0]))


def test_lengths_change_under_a_graph(gpu):
    """The work is dealt from what the device finds: whole blocks at one replay, runs with pieces to be joined at the next, nothing at all at a third."""
    import jittorinfer_amd as J
    heads, kv_heads, d = 16, 16, 64
    q, k, v, bt, lens, starts = _case(40, [300, 300, 300, 300], [1300, 400, 400, 8000], 64, heads, kv_heads, d, d, BF16)
    cases = [(lens.tolist(), starts.tolist()), ([300, 300, 300, 300], [0, 300, 600, 900, 1200]), ([1200, 0, 0, 0], [0, 1200, 1200, 1200, 1200]), ([1300, 400, 400, 8000], [0, 1, 2, 3, 1200]), ([0, 0, 0, 0], [0] * 5),
             ([5, 400, 7, 8000], [0, 5, 100, 107, 110]), (lens.tolist(), starts.tolist())]
    d_ = [t.to(gpu) for t in (q, k, v, bt, lens, starts)]
    out = torch.empty((1200, heads, d), dtype=BF16, device=gpu)
    # pages past a sequence's rows hold NaN; rows of the cache that a longer length would show are the sequence's own, so lengths only fall
    J.gqa_prompt_attn(*d_, scale=0.125, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        J.gqa_prompt_attn(*d_, scale=0.125, out=out)
    for n, st in cases:
        d_[4].copy_(torch.tensor(n, dtype=torch.int32))
        d_[5].copy_(torch.tensor(st, dtype=torch.int32))
        out.fill_(7.0)
        g.replay()
        eager = J.gqa_prompt_attn(*d_, scale=0.125, out=torch.full_like(out, 7.0))
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        want, off = B.prompt(q, k, v, bt, n, st, 0.125)
        mine = ~torch.isnan(want[:, 0, 0])
        _near(out[mine.to(gpu)], want[mine], off[mine], BF16, str(n))
        assert (out.cpu()[~mine] == 7.0).all()


def test_groups_change_under_a_graph(gpu):
    import jittorinfer_amd as J
    case = _shared(41, [(4, 512), (4, 300)], [5, 9, 0, 30, 200, 1, 77, 3, 50], 8, 2, 64, 64, F16)
    d = [t.to(gpu) for t in case]
    d[3] = _wide(d[3], d[1], d[2])
    out = torch.empty((9, 8, 64), dtype=F16, device=gpu)
    J.gqa_prefix_attn(*d, scale=0.125, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        J.gqa_prefix_attn(*d, scale=0.125, out=out)
    want, off = B.prompt(*case[:5], torch.arange(10), 0.125)
    for starts, lens in (([0, 4, 8], [512, 300]), ([0, 2, 8], [400, 0]), ([0, 0, 0], [512, 300]), ([1, 4, 4], [256, 9]), ([0, 4, 8], [512, 300])):
        d[5].copy_(torch.tensor(starts, dtype=torch.int32))
        d[6].copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(NAN)
        g.replay()
        torch.cuda.synchronize()
        _near(out, want, off, F16, "%s %s" % (starts, lens))


def test_two_threads_on_one_stream(gpu):
    """Calls of two threads share their stream's scratch: the kernels of a call stay together."""
    sets = [_calls(gpu, s) for s in (0, 50)]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        outs = [call() for _ in range(30) for call, _ in sets[i]]
        torch.cuda.synchronize()
        bad.extend(1 for j, o in enumerate(outs) if not torch.equal(o, sets[i][j % len(sets[i])][1]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_scratch_that_other_calls_have_filled(gpu):
    """Nothing of a call's scratch is taken to hold anything: areas full of ones, of NaN, and of what calls of other sizes left there."""
    from jittorinfer_amd import capi
    calls = _calls(gpu) + _calls(gpu, 50)
    area = capi._workspace(gpu, 1 << 20)
    for fill in (0xff, 0x7f, 1, 0):
        for call, want in calls:
            area.fill_(fill)
            assert torch.equal(call(), want)
    for (a, wa), (b, wb) in zip(calls, calls[::-1]):
        assert torch.equal(a(), wa) and torch.equal(b(), wb)


def test_results_on_operands_are_refused(gpu):
    import jittorinfer_amd as J
    q, k, v, bt, lens, starts = (t.to(gpu) for t in _case(42, [4, 4], [200, 30], 2, 2, 2, 64, 64, BF16))
    i = torch.tensor([0, 8], dtype=torch.int32, device=gpu)
    long = torch.empty(3 * q.numel(), dtype=BF16, device=gpu)
    shifted = long[64:64 + q.numel()].view_as(q)
    whole = long[:q.numel()].view_as(q).copy_(q)
    for out in (q, k.view(-1)[:q.numel()].view_as(q), v.view(-1)[64:64 + q.numel()].view_as(q)):
        with pytest.raises(RuntimeError, match="share memory"):
            J.gqa_prompt_attn(q, k, v, bt, lens, starts, scale=1.0, out=out)
    with pytest.raises(RuntimeError, match="share memory"):
        J.gqa_prompt_attn(whole, k, v, bt, lens, starts, scale=1.0, out=shifted)
    with pytest.raises(RuntimeError, match="share memory"):
        J.gqa_cross_attn(whole, k[:2], v[:2], scale=1.0, out=shifted)
    with pytest.raises(RuntimeError, match="share memory"):
        J.gqa_prefix_attn(whole[:2], k, v, bt, lens, i[:2] * 0, lens[:1], scale=1.0, out=whole[1:3])
    # views of one buffer that share no byte are apart
    both = torch.empty((8, 2, 128), dtype=BF16, device=gpu)
    both[..., :64] = q
    J.gqa_prompt_attn(both[..., :64], k, v, bt, lens, starts, scale=0.125, out=both[..., 64:])
    assert torch.equal(both[..., 64:], J.gqa_prompt_attn(q, k, v, bt, lens, starts, scale=0.125)) and torch.equal(both[..., :64], q)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_serving_loop_with_a_shared_prompt(gpu, dtype):
    """A system prompt filled in two chunks, sequences that share its pages, their own prompts behind it, decode steps that read it once, draft tokens verified and
    partly taken back, and a decoder's layer over an encoder's states in between.  The cache as it is on the device is what the plain forms read."""
    import numpy as np
    import jittorinfer_amd as J
    H, G, D, SCALE = 8, 2, 64, 0.125
    gen = torch.Generator().manual_seed(50)
    pt = J.PageTable(32, 5, 6)
    kc, vc = (torch.zeros((32, 128, G, D), dtype=dtype, device=gpu) for _ in range(2))
    states = [torch.randn((5, 90, G, D), generator=gen).to(dtype) for _ in range(2)]
    n_states = torch.tensor([90, 1, 33, 0, 64], dtype=torch.int32)
    rope = dict(n_dims=D, mode=2, freq_base=10000.0)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=gpu)

    def feed(seqs, counts):
        """New tokens of some sequences: their queries, block table and lengths."""
        ids = [b for b, n in zip(seqs, counts) for _ in range(n)]
        pos = [pt.seq_len(b) + i for b, n in zip(seqs, counts) for i in range(n)]
        assert pt.find_slot(ids, pos) is not None
        bt, lens = pt.fill_inputs(seqs)
        row = [seqs.index(b) for b in ids]
        qkv = torch.randn((len(ids), H + 2 * G, D), generator=gen).to(dtype).to(gpu)
        q = J.gqa_norm_rope(qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:], i32(pos), k_cache=kc, v_cache=vc, block_table=i32(bt), seq_ids=i32(row), **rope)
        return q, bt, lens

    def prompt(seqs, counts):
        q, bt, lens = feed(seqs, counts)
        starts = _starts(list(counts))
        got = J.gqa_prompt_attn(q, kc, vc, i32(bt), i32(lens), starts.to(gpu), scale=SCALE)
        want, off = B.prompt(q.cpu(), kc.cpu(), vc.cpu(), torch.from_numpy(bt), lens.tolist(), starts, SCALE)
        _near(got, want, off, dtype, "prompt")
        if len(seqs) == 5:                                # a layer over the encoder's states
            got = J.gqa_cross_attn(q, *[t.to(gpu) for t in states], q_starts=starts.to(gpu), kv_lens=n_states.to(gpu), scale=SCALE)
            want, off = B.cross(q.cpu(), *states, starts, n_states, SCALE)
            _near(got, want, off, dtype, "cross")

    def step(seqs):
        q, bt, lens = feed(seqs, [1] * len(seqs))
        starts, plens = pt.shared_prefixes(seqs)
        assert max(plens) >= 384
        want, off = B.prompt(q.cpu(), kc.cpu(), vc.cpu(), torch.from_numpy(bt), lens.tolist(), torch.arange(len(seqs) + 1), SCALE)
        for table in (i32(bt), _wide(i32(bt), kc, vc)):
            _near(J.gqa_prefix_attn(q, kc, vc, table, i32(lens), i32(starts), i32(plens), scale=SCALE), want, off, dtype, "step")
        return starts.tolist(), plens.tolist()

    prompt([0], [300])
    prompt([0], [110])
    free = pt.free_pages
    for b in (1, 2, 3):                                   # 410 rows: three pages shared, 26 rows copied
        src, dst, n = pt.seq_cp(0, b)
        assert n == 26
        for c in (kc, vc):
            flat = c.view(-1, G, D)
            flat[dst:dst + n] = flat[src:src + n]
    assert pt.free_pages == free - 3
    prompt([0, 1, 2, 3, 4], [3, 40, 1, 150, 70])          # the fifth shares nothing
    for _ in range(3):
        assert step([0, 1, 2, 3, 4]) == ([0, 4, 5], [384, 0])
    prompt([0, 1, 2, 3, 4], [4, 4, 4, 4, 4])              # drafts: three of them are taken back
    for b in (0, 2, 4):
        assert pt.seq_rm(b, pt.seq_len(b) - 3)
    assert step([4, 3, 2, 1, 0]) == ([0, 1, 5], [0, 384])
    assert step([1, 4, 0, 2]) == ([0, 1, 2, 4], [0, 0, 384])


def test_offsets_past_32_bits(gpu):
    """Pages, packed states and queries that lie more than 4 GB into their tensors."""
    import jittorinfer_amd as J
    q, k, v, bt, lens, starts = _case(60, [70, 5], [300, 129], 3, 8, 8, 128, 128, BF16, spare=0)
    n = k.shape[0]
    far = 20000                                          # pages of 256 KB: 5 GB
    big = [torch.empty((far + n, 128, 8, 128), dtype=BF16, device=gpu) for _ in range(2)]
    for b, small in zip(big, (k, v)):
        b[far:] = small.to(gpu)
    want, off = B.prompt(q, k, v, bt, lens, starts, 0.1)
    table = torch.where(torch.arange(3)[None] * 128 < lens[:, None], bt + far, 0).to(torch.int32).to(gpu)
    _near(J.gqa_prompt_attn(q.to(gpu), *big, table, lens.to(gpu), starts.to(gpu), scale=0.1), want, off, BF16)
    each = torch.arange(3, dtype=torch.int32)
    want, off = B.prompt(q[:2], k, v, bt, lens, each, 0.1)
    for group, shared in (([0, 1, 2], [300, 0]), ([0, 1], [256])):
        got = J.gqa_prefix_attn(q[:2].to(gpu), *big, _wide(table, k, v), lens.to(gpu), torch.tensor(group, dtype=torch.int32, device=gpu), torch.tensor(shared, dtype=torch.int32, device=gpu), scale=0.1)
        _near(got, want, off, BF16)
    # the same memory as packed states, rows of 2 KB
    flat = [b.view(-1, 8, 128) for b in big]
    first = [int(bt[0, 0]), int(bt[1, 0])]
    at = torch.tensor([(far + p) * 128 for p in first], dtype=torch.int32)
    for new in (1, 40):
        x = torch.randn((2 * new, 8, 128), generator=torch.Generator().manual_seed(new)).to(BF16)
        rows = torch.tensor([100, 128], dtype=torch.int32)
        want, off = B.cross(x, torch.stack([k[p] for p in first]), torch.stack([v[p] for p in first]), [0, new, 2 * new], rows, 0.1)
        _near(J.gqa_cross_attn(x.to(gpu), *flat, kv_starts=at.to(gpu), kv_lens=rows.to(gpu), scale=0.1), want, off, BF16)
    # queries and results with a stride of their own
    wide = torch.empty((75, 8, 1 << 22), dtype=BF16, device=gpu)
    wide[:, :, :128] = q.to(gpu)
    want, off = B.prompt(q, k, v, bt, lens, starts, 0.1)
    out = wide[:, :, 4096:4096 + 128]
    J.gqa_prompt_attn(wide[:, :, :128], *big, table, lens.to(gpu), starts.to(gpu), scale=0.1, out=out)
    _near(out, want, off, BF16)
