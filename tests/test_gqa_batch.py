"""Attention of many query rows over the same keys without a GPU: what the entry points of include/gqa_batch.h refuse, the ctypes mirrors of their argument
blocks, what the Python entry points raise, and the plain forms the GPU tests compare with."""
import ctypes as C
import json
import math
import os
import re
import subprocess
import sys

import pytest
import torch

import jittorinfer_amd as J
from tests import gqa_batch_util as B
from tests import gqa_util as R
from tests.test_gqa import ALIGN, NULL, SHAPE, TYPE, UNSUPPORTED, WORKSPACE, _name, _pool

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _set(a, kw):
    for name, v in kw.items():
        o = a
        *path, last = name.split("__")
        for part in path:
            o = getattr(o, part)
        setattr(o, last, v)
    return a


def _common(a):
    if hasattr(a, "n_tok"):
        a.n_tok, a.n_seq = 30, 3
    a.n_head, a.n_head_kv, a.dk, a.dv = 8, 2, 128, 128
    a.type, a.scale = J.MLA_TYPE_BF16, 0.1
    a.q, a.q_nb1, a.q_nb2 = 4096, 256, 2048
    a.k, a.v = _pool(128), _pool(128, base=1 << 24)
    a.dst, a.d_nb1, a.d_nb2 = 32768, 256, 2048
    return a


def _prompt(**kw):
    """A call that is accepted, on made-up addresses (never dereferenced), with some fields replaced."""
    a = _common(J.GqaPromptAttnArgs())
    a.causal, a.n_pages, a.block_table, a.bt_stride, a.seq_lens, a.q_starts = 1, 16, 8192, 4, 16384, 16640
    return _set(a, kw)


def _cross(**kw):
    a = _common(J.GqaCrossAttnArgs())
    a.n_kv = 500
    return _set(a, kw)


def _prefix(**kw):
    a = _common(J.GqaPrefixAttnArgs())
    a.n_seq, a.n_prefix, a.n_pages, a.block_table, a.bt_stride, a.seq_lens, a.prefix_starts, a.prefix_lens = 30, 2, 16, 8192, 4, 16384, 16640, 17408
    return _set(a, kw)


COMMON_REFUSED = [
    (dict(type=J.MLA_TYPE_F32), TYPE), (dict(type=J.MLA_TYPE_Q8_0), TYPE),
    (dict(n_tok=-1), SHAPE), (dict(n_seq=-1), SHAPE), (dict(n_head=0), SHAPE), (dict(n_head_kv=0), SHAPE), (dict(n_head_kv=3), SHAPE), (dict(n_workgroups=-1), SHAPE), (dict(n_workgroups=65537), SHAPE),
    (dict(q_starts=None, n_tok=31), SHAPE), (dict(n_tok=1 << 28), SHAPE), (dict(n_head=65536 * 8, n_head_kv=65536), SHAPE),
    (dict(dk=96), UNSUPPORTED), (dict(dv=64), UNSUPPORTED), (dict(dk=192, dv=192), UNSUPPORTED), (dict(dk=576, dv=512), UNSUPPORTED), (dict(dk=0, dv=0), UNSUPPORTED),
    (dict(logit_softcap=-1.0), UNSUPPORTED), (dict(logit_softcap=float("nan")), UNSUPPORTED), (dict(logit_softcap=float("inf")), UNSUPPORTED),
    (dict(q=None), NULL), (dict(dst=None), NULL), (dict(k__data=None), NULL), (dict(v__data=None), NULL),
    (dict(q=4100), ALIGN), (dict(q_nb1=248), ALIGN), (dict(q_nb2=2056), ALIGN), (dict(k__nb_row=520), ALIGN), (dict(v__nb_head=264), ALIGN), (dict(k__data=(1 << 20) + 8), ALIGN), (dict(dst=32772), ALIGN),
    (dict(d_nb1=260), ALIGN), (dict(mask=65537, mask_ne0=512, mask_nb1=1024), ALIGN), (dict(mask=65536, mask_ne0=512, mask_nb1=1023), ALIGN), (dict(mask=65536, mask_ne0=-1), SHAPE),
    (dict(k__nb_page=-65536), SHAPE), (dict(v__nb_row=(1 << 23) + 16), SHAPE), (dict(k__nb_head=-256), SHAPE),
    (dict(dst=4096), UNSUPPORTED), (dict(dst=1 << 20), UNSUPPORTED), (dict(dst=1 << 24), UNSUPPORTED), (dict(mask=32768, mask_ne0=512, mask_nb1=1024), UNSUPPORTED), (dict(q_starts=32768), UNSUPPORTED),
]
PROMPT_REFUSED = COMMON_REFUSED + [
    (dict(window=-1), SHAPE), (dict(block_table=None), NULL), (dict(seq_lens=None), NULL), (dict(n_pages=0), SHAPE), (dict(bt_stride=0), SHAPE), (dict(bt_stride=1 << 23), SHAPE), (dict(bt_stride=1 << 62), SHAPE),
    (dict(dst=8192), UNSUPPORTED), (dict(dst=16384), UNSUPPORTED),
]
CROSS_REFUSED = COMMON_REFUSED + [
    (dict(n_kv=-1), SHAPE), (dict(n_kv=1 << 30), SHAPE), (dict(kv_starts=8192), SHAPE), (dict(kv_starts=32768, k__nb_page=0, v__nb_page=0), UNSUPPORTED), (dict(kv_lens=32768), UNSUPPORTED),
]


PREFIX_REFUSED = [(kw, code) for kw, code in COMMON_REFUSED if not {"n_tok", "q_starts"} & set(kw) and kw != dict(dk=576, dv=512)] + [
    (dict(n_prefix=-1), SHAPE), (dict(block_table=None), NULL), (dict(seq_lens=None), NULL), (dict(prefix_starts=None), NULL), (dict(prefix_lens=None), NULL), (dict(n_pages=0), SHAPE), (dict(bt_stride=0), SHAPE),
    (dict(bt_stride=1 << 23), SHAPE), (dict(k__nb_page=1 << 32), SHAPE), (dict(n_seq=32768), SHAPE), (dict(dk=576, dv=0, n_head_kv=1), UNSUPPORTED),
    (dict(dst=8192), UNSUPPORTED), (dict(dst=16384), UNSUPPORTED), (dict(dst=16640), UNSUPPORTED), (dict(dst=17408), UNSUPPORTED),
]


@pytest.mark.parametrize("kw,code", PREFIX_REFUSED, ids=_name)
def test_prefix_refuses(kw, code):
    lib, a = J.library(), _prefix(**kw)
    assert lib.gqa_prefix_attn_check(C.byref(a)) == code and lib.gqa_prefix_attn_launch(C.byref(a), None) == code and lib.gqa_prefix_attn_workspace_size(C.byref(a)) == 0


@pytest.mark.parametrize("kw,code", PROMPT_REFUSED, ids=_name)
def test_prompt_refuses(kw, code):
    lib, a = J.library(), _prompt(**kw)
    assert lib.gqa_prompt_attn_check(C.byref(a)) == code and lib.gqa_prompt_attn_launch(C.byref(a), None) == code and lib.gqa_prompt_attn_workspace_size(C.byref(a)) == 0


@pytest.mark.parametrize("kw,code", CROSS_REFUSED, ids=_name)
def test_cross_refuses(kw, code):
    lib, a = J.library(), _cross(**kw)
    assert lib.gqa_cross_attn_check(C.byref(a)) == code and lib.gqa_cross_attn_launch(C.byref(a), None) == code and lib.gqa_cross_attn_workspace_size(C.byref(a)) == 0


def _accepted(name, make, calls):
    lib = J.library()
    check, size, launch = (getattr(lib, name + x) for x in ("_check", "_workspace_size", "_launch"))
    assert check(None) == NULL and size(None) == 0
    for kw in calls:
        a = make(**kw)
        assert check(C.byref(a)) == 0, kw
        need = size(C.byref(a))
        assert (need > 0) == (getattr(a, "n_tok", 1) > 0 and a.n_seq > 0), kw
        if not need:
            assert launch(C.byref(a), None) == 0
            continue
        # without a device: one byte short, misaligned, none
        for ws, n in ((None, need), (1 << 30, need - 1), ((1 << 30) + 128, need)):
            a.workspace, a.workspace_size = ws, n
            assert launch(C.byref(a), None) == WORKSPACE


COMMON_ACCEPTED = [dict(), dict(n_tok=0, q=None), dict(n_seq=0, q=None), dict(q_starts=None), dict(mask=65536, mask_ne0=0, mask_nb1=0), dict(scale=-1.0), dict(n_workgroups=7),
                   dict(type=J.MLA_TYPE_F16, dk=192), dict(dk=64, dv=64), dict(dk=256, dv=256), dict(k__nb_row=0), dict(n_head=40, n_head_kv=1)]


def test_prompt_accepts():
    _accepted("gqa_prompt_attn", _prompt, COMMON_ACCEPTED + [dict(window=5, causal=0), dict(n_tok=0, block_table=None), dict(bt_stride=(1 << 23) - 1)])


def test_cross_accepts():
    _accepted("gqa_cross_attn", _cross, COMMON_ACCEPTED + [dict(n_kv=0), dict(n_kv=0, k__data=None, v__data=None), dict(kv_lens=8192), dict(kv_starts=8192, k__nb_page=0, v__nb_page=0), dict(k__nb_page=1 << 40)])


def test_prefix_accepts():
    _accepted("gqa_prefix_attn", _prefix, [kw for kw in COMMON_ACCEPTED if not {"n_tok", "q_starts"} & set(kw)] + [dict(n_prefix=0), dict(n_prefix=0, prefix_starts=None, prefix_lens=None), dict(n_prefix=100)])


def test_prefixes_are_worked_on_by_themselves_where_the_table_has_room_for_many_rows():
    """Scratch of the prefixes' pieces from 2^28 bytes of rows on, or where the workgroups are given; else of gqa_attn alone."""
    lib = J.library()
    size = lambda **kw: lib.gqa_prefix_attn_workspace_size(C.byref(_prefix(**kw)))
    a = _prefix()
    page = a.n_seq * 128 * a.n_head_kv * (a.dk + a.dv) * 2
    least = -(-2 ** 28 // page)
    for stride in (1, least - 1, least, least + 1):
        alone = size(bt_stride=stride, n_prefix=0)
        assert (size(bt_stride=stride) > alone) == (stride >= least)
        assert size(bt_stride=stride, n_workgroups=16) > size(bt_stride=stride, n_workgroups=16, n_prefix=0)


def test_launches_of_more_threads_than_there_are_refused():
    """Nothing starts of a call whose last kernel could not: 2^24 workgroups of 256 threads, one a block."""
    lib = J.library()
    a = _prompt(n_tok=(1 << 28) - 1, n_head=8, n_head_kv=1, dk=256, dv=256)
    assert lib.gqa_prompt_attn_check(C.byref(a)) == SHAPE
    a.n_tok = 1 << 24
    assert lib.gqa_prompt_attn_check(C.byref(a)) == 0


def test_exports_and_mirrors_match_the_header(tmp_path):
    """Every function the header declares is exported; every ctypes mirror has the C compiler's size and field offsets."""
    text = open(os.path.join(ROOT, "include", "gqa_batch.h")).read()
    bare = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    declared = set(re.findall(r"\b(gqa_\w+)\s*\(", bare))
    mirrors = {"gqa_prompt_attn_args": J.GqaPromptAttnArgs, "gqa_cross_attn_args": J.GqaCrossAttnArgs, "gqa_prefix_attn_args": J.GqaPrefixAttnArgs}
    assert declared == {n[:-5] + s for n in mirrors for s in ("_check", "_workspace_size", "_launch")}
    for name in declared:
        assert hasattr(J.library(), name)
    lines = []
    for name, cls in mirrors.items():
        lines.append('printf("%s . %%zu\\n", sizeof(%s));' % (name, name))
        lines += ['printf("%s %s %%zu\\n", offsetof(%s, %s));' % (name, f[0], name, f[0]) for f in cls._fields_]
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gqa_batch.h"\nint main(void){%s return 0;}\n' % "\n".join(lines))
    subprocess.run(["gcc", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "t")], check=True)
    for line in subprocess.run([str(tmp_path / "t")], check=True, stdout=subprocess.PIPE, text=True).stdout.splitlines():
        name, field, value = line.split()
        assert int(value) == (C.sizeof(mirrors[name]) if field == "." else getattr(mirrors[name], field).offset), (name, field)


CALLS = r"""
import json
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
import jittorinfer_amd as J
with FakeTensorMode():
    f = lambda *shape, dtype=torch.bfloat16: torch.empty(shape, dtype=dtype, device="cuda")
    i = lambda *shape: f(*shape, dtype=torch.int32)
    q, k, v, bt, lens, starts = f(10, 4, 64), f(3, 128, 2, 64), f(3, 128, 2, 64), i(2, 1), i(2), i(3)
    ek, ev, m = f(2, 50, 2, 64), f(2, 50, 2, 64), f(2, 128, dtype=torch.float16)
    wide = f(3, 128, 2, 64, dtype=torch.float32)
P = lambda **kw: J.gqa_prompt_attn(**{**dict(q=q, k_cache=k, v_cache=v, block_table=bt, seq_lens=lens, q_starts=starts, scale=1.0), **kw})
X = lambda **kw: J.gqa_cross_attn(**{**dict(q=q, k=ek, v=ev, q_starts=starts, scale=1.0), **kw})
S = lambda **kw: J.gqa_prefix_attn(**{**dict(q=q[:2], k_cache=k, v_cache=v, block_table=bt, seq_lens=lens, prefix_starts=lens, prefix_lens=lens[:1], scale=1.0), **kw})
cpu = torch.zeros(2, dtype=torch.int32)
calls = dict(
    prompt_cpu=lambda: P(q=torch.zeros(10, 4, 64)), prompt_lens_cpu=lambda: P(seq_lens=cpu), prompt_f32=lambda: P(q=q.float()), prompt_types=lambda: P(q=q.half()), prompt_cache_f32=lambda: P(k_cache=wide, v_cache=wide),
    prompt_dims=lambda: P(q=q[0]), prompt_width=lambda: P(q=q[..., :32]), prompt_v_heads=lambda: P(v_cache=v[:, :, :1]), prompt_v_pages=lambda: P(v_cache=v[:2]), prompt_table=lambda: P(block_table=bt[:1]),
    prompt_lens=lambda: P(seq_lens=lens[:1]), prompt_starts=lambda: P(q_starts=lens), prompt_starts_type=lambda: P(q_starts=starts.long()), prompt_uneven=lambda: P(q=q[:9], q_starts=None),
    prompt_mask_type=lambda: P(mask=m.float()), prompt_mask_rows=lambda: P(mask=m[:1]), prompt_window=lambda: P(window=-1), prompt_window_big=lambda: P(window=1 << 40), prompt_out=lambda: P(out=q[:9]),
    prompt_out_type=lambda: P(out=q.float()), prompt_out_expanded=lambda: P(out=q[:1].expand(10, 4, 64)), prompt_none=lambda: P(k_cache=None), prompt_scale=lambda: P(scale="x"),
    prompt_page=lambda: P(k_cache=k[:, :64], v_cache=v[:, :64]), prompt_column=lambda: P(q=q.transpose(1, 2)), prompt_alloc=lambda: P(),
    cross_cpu=lambda: X(q=torch.zeros(10, 4, 64)), cross_lens_cpu=lambda: X(kv_lens=cpu), cross_types=lambda: X(k=ek.half()), cross_f32=lambda: X(q=q.float(), k=ek.float(), v=ev.float()), cross_dims=lambda: X(k=ek[0], v=ev[0]),
    cross_packed_dims=lambda: X(kv_starts=starts), cross_seqs=lambda: X(k=ek[:1], v=ev[:1]), cross_v_rows=lambda: X(v=ev[:, :49]), cross_v_heads=lambda: X(v=ev[:, :, :1]), cross_lens=lambda: X(kv_lens=starts),
    cross_starts=lambda: X(k=ek[0], v=ev[0], kv_starts=lens), cross_starts_short=lambda: X(k=ek[0], v=ev[0], kv_starts=lens[:1], kv_lens=lens), cross_uneven=lambda: X(q=q[:9], q_starts=None), cross_mask=lambda: X(mask=m[:1]),
    cross_out=lambda: X(out=q[:9]), cross_alloc=lambda: X(),
    prefix_cpu=lambda: S(q=torch.zeros(2, 4, 64)), prefix_lens_cpu=lambda: S(prefix_lens=cpu[:1]), prefix_f32=lambda: S(q=q[:2].float()), prefix_cache=lambda: S(k_cache=wide, v_cache=wide), prefix_seqs=lambda: S(q=q),
    prefix_table=lambda: S(block_table=bt[:1]), prefix_starts=lambda: S(prefix_starts=starts), prefix_starts_type=lambda: S(prefix_starts=lens.long()), prefix_none=lambda: S(prefix_lens=None), prefix_out=lambda: S(out=q),
    prefix_mask=lambda: S(mask=m[:1]), prefix_alloc=lambda: S(),
)
J.capi.native()
seen = {}
for name, call in calls.items():
    try:
        call()
        seen[name] = "returned"
    except Exception as e:
        seen[name] = "raised" if isinstance(e, (RuntimeError, AssertionError, TypeError, ValueError)) else repr(e)
print("SEEN " + json.dumps(seen), flush=True)
"""


@pytest.mark.skipif(torch.cuda.is_available(), reason="the accepted calls would run")
def test_python_entry_points_raise():
    """Wrong tensors are Python errors, raised before a launch; so is an allocation that fails.  Tensors without storage, in a process of their own."""
    r = subprocess.run([sys.executable, "-c", CALLS], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:]
    seen = json.loads([l for l in r.stdout.splitlines() if l.startswith("SEEN ")][0][5:])
    assert len(seen) > 50 and set(seen.values()) == {"raised"}, {k: v for k, v in seen.items() if v != "raised"}


# ---------------------------------------------------------------- the plain forms themselves

def test_plain_prompt_by_hand():
    """Two new tokens behind three rows, one head: the softmax of what each sees."""
    gen = torch.Generator().manual_seed(0)
    k, v = (torch.randn((1, 128, 1, 4), generator=gen).bfloat16() for _ in range(2))
    q = torch.randn((2, 1, 4), generator=gen).bfloat16()
    for window in (0, 2):
        out, off = B.prompt(q, k, v, torch.zeros((1, 1), dtype=torch.int32), [5], [0, 2], 0.5, window=window)
        for t in range(2):
            rows = range(max(0, 4 + t - window) if window else 0, 4 + t)
            e = [math.exp(0.5 * float(q[t, 0].double() @ k[0, i, 0].double())) for i in rows]
            want = sum(x * v[0, i, 0].double() for x, i in zip(e, rows)) / sum(e)
            assert torch.allclose(out[t, 0], want, rtol=1e-12) and (off[t, 0] > 0).all()


def test_plain_prompt_of_one_token_is_plain_attention():
    gen = torch.Generator().manual_seed(1)
    k, v = (R.make_cache(gen, 3, 2, 8, torch.bfloat16) for _ in range(2))
    bt = torch.tensor([[2, 0], [1, 1]], dtype=torch.int32)
    q = torch.randn((2, 4, 8), generator=gen).bfloat16()
    a, _, _, _ = R.attn(q, k, v, bt, [200, 17], 0.3, 2.0, 50)
    b, _ = B.prompt(q, k, v, bt, [200, 17], [0, 1, 2], 0.3, 2.0, 50)
    assert torch.allclose(a, b, rtol=1e-12)


def test_plain_cross_is_prompt_without_order():
    gen = torch.Generator().manual_seed(2)
    k, v = (torch.randn((2, 128, 2, 8), generator=gen).bfloat16() for _ in range(2))
    q = torch.randn((5, 4, 8), generator=gen).bfloat16()
    a, _ = B.cross(q, k, v, [0, 2, 5], [100, 3], 0.3)
    b, _ = B.prompt(q, k, v, torch.tensor([[0], [1]], dtype=torch.int32), [100, 3], [0, 2, 5], 0.3, causal=False)
    c, _ = B.cross(q, torch.cat((k[0, :100], k[1, :3])), torch.cat((v[0, :100], v[1, :3])), [0, 2, 5], [100, 3], 0.3, kv_starts=[0, 100])
    assert torch.allclose(a, b, rtol=1e-12) and torch.allclose(a, c, rtol=1e-12)


def test_shared_prefixes_of_a_batch():
    """Groups are neighbours whose tables begin with the same pages, cut so that the most page reads are spared."""
    pt = J.PageTable(64, 8, 16)
    pt.find_slot([0] * 1000, list(range(1000)))          # 7 whole pages and 104 rows
    for s in (1, 2, 3):
        pt.seq_cp(0, s, -1, [0, 1000, 700, 300][s])      # 7, 5 and 2 pages shared
    pt.find_slot([4] * 200, list(range(200)))
    pt.seq_cp(4, 5)                                      # 1 page shared
    groups = lambda ids: tuple(x.tolist() for x in pt.shared_prefixes(ids))
    assert groups([0, 1]) == ([0, 2], [896])
    assert groups([0, 1, 2]) == ([0, 3], [640])          # 2 x 5 pages spared, 7 without the third
    assert groups([0, 1, 2, 3]) == ([0, 3, 4], [640, 0])  # 10, against 3 x 2 of all four
    assert groups([0, 1, 3, 2]) == ([0, 2, 4], [896, 256])
    assert groups([4, 0, 1, 5]) == ([0, 1, 3, 4], [0, 896, 0])
    assert groups([4, 5, 0, 1, 6]) == ([0, 2, 4, 5], [128, 896, 0])
    assert groups([7]) == ([0, 1], [0]) and groups([]) == ([0], []) and groups([6, 7]) == ([0, 1, 2], [0, 0])
    pt.seq_rm(0, 100)
    pt.seq_rm(1, 90)
    assert groups([0, 1]) == ([0, 2], [100])             # one page, of which the longer one has 100 rows
    with pytest.raises(ValueError):
        pt.shared_prefixes([0, 8])
    lib = J.library()
    assert lib.mla_page_table_shared_prefixes(None, 0, None, None, None) == -2
