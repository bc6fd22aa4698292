"""Attention of many query rows over the same keys without a GPU: which way a call goes by its sizes, and what each refusal of the Python entry points says."""
import ctypes as C
import json
import subprocess
import sys

import pytest
import torch

import jittorinfer_amd as J
from tests.test_gqa_batch import CALLS, ROOT, _prefix


def test_prefixes_that_nobody_can_share_are_gqa_attn():
    """As many groups as sequences (what shared_prefixes gives a batch that shares nothing), one sequence alone: no row is there to be read once for two, whatever the
    table has room for.  One group fewer, and two sequences may share."""
    lib = J.library()
    size = lambda **kw: lib.gqa_prefix_attn_workspace_size(C.byref(_prefix(**kw)))
    for widths in (dict(), dict(dk=64, dv=64), dict(dk=256, dv=256)):
        for n_seq in (1, 2, 30):
            for stride in (4, 20000):
                call = dict(n_seq=n_seq, bt_stride=stride, **widths)
                alone = size(n_prefix=0, **call)
                for n_prefix in (n_seq, n_seq + 1, 3 * n_seq):
                    assert size(n_prefix=n_prefix, **call) == alone > 0
                if n_seq > 1 and stride == 20000:
                    assert size(n_prefix=n_seq - 1, **call) > alone
                assert size(n_prefix=n_seq, n_workgroups=16, **call) > size(n_prefix=0, n_workgroups=16, **call)


# What each call of test_gqa_batch.CALLS is refused for: its exception and a part of its text.  None: the result tensor is looked at behind the stream, which needs a device (the accepted calls
# get that far too); tests/test_gqa_batch_edges_gpu.py has those.
REFUSED = dict(
    prompt_cpu=("RuntimeError", "GPU only"), prompt_lens_cpu=("AssertionError", "device()"), prompt_f32=("AssertionError", "queries(a, q, starts, n_seq)"), prompt_types=("AssertionError", "cache_ok(*kc"),
    prompt_cache_f32=("AssertionError", "cache_ok(*kc"), prompt_dims=("AssertionError", "queries(a, q, starts, n_seq)"), prompt_width=("AssertionError", "kc->size(3) == a.dk"),
    prompt_v_heads=("AssertionError", "vc->size(2) == kc->size(2)"), prompt_v_pages=("AssertionError", "vc->size(0) == kc->size(0)"), prompt_table=("AssertionError", "ints(*lens, table->size(0))"),
    prompt_lens=("AssertionError", "ints(*lens, table->size(0))"), prompt_starts=("AssertionError", "queries(a, q, starts, n_seq)"), prompt_starts_type=("AssertionError", "queries(a, q, starts, n_seq)"),
    prompt_uneven=("AssertionError", "queries(a, q, starts, n_seq)"), prompt_mask_type=("AssertionError", "row_mask(a, mask, n_seq)"), prompt_mask_rows=("AssertionError", "row_mask(a, mask, n_seq)"),
    prompt_window=("AssertionError", "window >= 0"), prompt_window_big=("AssertionError", "window < INTS"), prompt_out=None, prompt_out_type=None, prompt_out_expanded=None,
    prompt_none=("TypeError", "torch tensor"), prompt_scale=("TypeError", "real number"), prompt_page=("AssertionError", "cache_ok(*kc"), prompt_column=("AssertionError", "queries(a, q, starts, n_seq)"),
    prompt_alloc=None,
    cross_cpu=("RuntimeError", "GPU only"), cross_lens_cpu=("AssertionError", "device()"), cross_types=("AssertionError", "mla_type(*t) == mla_type(q)"), cross_f32=("AssertionError", "queries(a, q, starts, n_seq)"),
    cross_dims=("AssertionError", "rows_ok(*t, d, false)"), cross_packed_dims=("AssertionError", "rows_ok(*t, d, false)"), cross_seqs=("AssertionError", "queries(a, q, starts, n_seq)"),
    cross_v_rows=("AssertionError", "v->size(d - 3) == k->size(d - 3)"), cross_v_heads=("AssertionError", "v->size(d - 2) == k->size(d - 2)"), cross_lens=("AssertionError", "ints(*kv_lens, n_seq)"),
    cross_starts=("AssertionError", "queries(a, q, starts, n_seq)"), cross_starts_short=("AssertionError", "kv_starts->numel() >= n_seq"), cross_uneven=("AssertionError", "queries(a, q, starts, n_seq)"),
    cross_mask=("AssertionError", "row_mask(a, mask, n_seq)"), cross_out=None, cross_alloc=None,
    prefix_cpu=("RuntimeError", "GPU only"), prefix_lens_cpu=("AssertionError", "device()"), prefix_f32=("AssertionError", "mla_type(q) > 0"), prefix_cache=("AssertionError", "cache_ok(*kc"),
    prefix_seqs=("AssertionError", "table->size(0) == n_seq"), prefix_table=("AssertionError", "table->size(0) == n_seq"), prefix_starts=("AssertionError", "ints(*starts, plens->numel() + 1)"),
    prefix_starts_type=("AssertionError", "ints(*starts, plens->numel() + 1)"), prefix_none=("TypeError", "torch tensor"), prefix_out=None, prefix_mask=("AssertionError", "row_mask(a, mask, n_seq)"), prefix_alloc=None,
)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the accepted calls would run")
def test_python_entry_points_refuse_what_is_wrong():
    """Every wrong tensor is refused for what is wrong with it, and not because there is no device."""
    calls, behind = CALLS.split("J.capi.native()\n")
    source = calls + "J.capi.native()\n" + behind.replace('seen[name] = "raised" if', 'seen[name] = [type(e).__name__, str(e)] if')
    r = subprocess.run([sys.executable, "-c", source], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:]
    seen = json.loads([l for l in r.stdout.splitlines() if l.startswith("SEEN ")][0][5:])
    assert set(seen) == set(REFUSED)
    for name, want in REFUSED.items():
        kind, text = seen[name]
        if want is None:
            assert kind == seen["prompt_alloc"][0] and kind not in ("AssertionError", "TypeError"), (name, kind, text)
        else:
            assert kind == want[0] and want[1] in text, (name, kind, text)
