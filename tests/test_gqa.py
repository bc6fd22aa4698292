"""The paged cache of ordinary heads without a GPU: what the entry points of include/gqa_attn.h refuse, the ctypes mirrors of their argument
blocks, the pages an eviction gives back, and the plain forms the GPU tests compare with."""
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
from jittorinfer_amd import capi
from tests import gqa_util as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SHAPE, TYPE, ALIGN, WORKSPACE, NULL, UNSUPPORTED = -1, -2, -3, -4, -5, -6


def _pool(width, heads=2, es=2, base=1 << 20):
    return J.GqaPool(base, 128 * heads * width * es, heads * width * es, width * es)


def _name(x):
    """A test's name: the same in every process, whatever addresses its objects have."""
    return " ".join("%s=%s" % (n, v) if isinstance(v, int) else n for n, v in x.items()) if isinstance(x, dict) else str(x)


def _attn(**kw):
    """A call that is accepted, on made-up addresses (never dereferenced), with some fields replaced."""
    a = J.GqaAttnArgs()
    a.n_seq, a.n_head, a.n_head_kv, a.dk, a.dv = 3, 8, 2, 128, 128
    a.q_type = a.kv_type = a.dst_type = J.MLA_TYPE_BF16
    a.scale = 0.1
    a.q, a.q_nb1, a.q_nb2 = 4096, 256, 2048
    a.k, a.v, a.n_pages = _pool(128), _pool(128, base=1 << 24), 16
    a.block_table, a.bt_stride, a.seq_lens = 8192, 4, 16384
    a.dst, a.d_nb1, a.d_nb2 = 32768, 256, 2048
    for name, v in kw.items():
        o = a
        *path, last = name.split("__")
        for part in path:
            o = getattr(o, part)
        setattr(o, last, v)
    return a


def _latent(**kw):
    base = dict(n_head=128, n_head_kv=1, dk=576, dv=0, k=_pool(576, 1), v=J.GqaPool(), dst=None, weights=65536, w_nb1=2048, w_nb2=2048, q_nb1=1152, q_nb2=147456)
    return _attn(**{**base, **kw})


ATTN_REFUSED = [
    (dict(kv_type=J.MLA_TYPE_Q8_0), TYPE), (dict(kv_type=J.MLA_TYPE_F32), TYPE), (dict(q_type=J.MLA_TYPE_F16), TYPE), (dict(dst_type=J.MLA_TYPE_F16), TYPE),
    (dict(n_seq=-1), SHAPE), (dict(n_head=0), SHAPE), (dict(n_head_kv=0), SHAPE), (dict(n_head=7), SHAPE), (dict(window=-1), SHAPE),
    (dict(n_workgroups=-1), SHAPE), (dict(n_workgroups=1 << 20), SHAPE),
    (dict(dk=96, dv=96), UNSUPPORTED), (dict(dk=128, dv=64), UNSUPPORTED), (dict(dk=192, dv=192), UNSUPPORTED), (dict(dk=576, dv=512), UNSUPPORTED), (dict(dv=0), UNSUPPORTED),
    (dict(logit_softcap=-1.0), UNSUPPORTED), (dict(logit_softcap=float("nan")), UNSUPPORTED),
    (dict(q=None), NULL), (dict(k__data=None), NULL), (dict(v__data=None), NULL), (dict(block_table=None), NULL), (dict(seq_lens=None), NULL), (dict(dst=None), NULL),
    (dict(q=4098), ALIGN), (dict(q_nb1=264), ALIGN), (dict(q_nb2=2056), ALIGN), (dict(dst=32772), ALIGN), (dict(d_nb1=260), ALIGN), (dict(dst_type=J.MLA_TYPE_F32, d_nb1=264), ALIGN),
    (dict(k__data=(1 << 20) + 8), ALIGN), (dict(v__nb_row=520), ALIGN), (dict(k__nb_page=65544), ALIGN), (dict(k__nb_head=260), ALIGN),
    (dict(k__nb_row=-512), SHAPE), (dict(k__nb_row=1 << 24), SHAPE), (dict(v__nb_page=-65536), SHAPE), (dict(v__nb_head=-256), SHAPE),
    (dict(n_pages=0), SHAPE), (dict(bt_stride=0), SHAPE), (dict(bt_stride=1 << 24), SHAPE), (dict(n_seq=65536), SHAPE), (dict(n_seq=20000, bt_stride=1 << 20), SHAPE),
    (dict(mask=8193, mask_nb1=1024, mask_ne0=512), ALIGN), (dict(mask=8192, mask_nb1=1023, mask_ne0=512), ALIGN), (dict(mask=8192, mask_nb1=1024, mask_ne0=-1), SHAPE),
    (dict(weights=65537, w_nb1=2048, w_nb2=4096), ALIGN), (dict(weights=65536, w_nb1=2047, w_nb2=4096), ALIGN), (dict(weights=65536, w_nb1=2048, w_nb2=4098), ALIGN),
]


@pytest.mark.parametrize("kw,code", ATTN_REFUSED, ids=lambda x: str(x)[:60])
def test_attn_refuses(kw, code):
    lib = J.library()
    a = _attn(**kw)
    assert lib.gqa_attn_check(C.byref(a)) == code
    assert lib.gqa_attn_launch(C.byref(a), None) == code            # before anything touches a device
    assert lib.gqa_attn_workspace_size(C.byref(a)) == 0


def test_attn_accepts_and_wants_scratch():
    lib = J.library()
    assert lib.gqa_attn_check(None) == NULL
    a = _attn()
    assert lib.gqa_attn_check(C.byref(a)) == 0
    need = lib.gqa_attn_workspace_size(C.byref(a))
    assert need > 0 and lib.gqa_attn_launch(C.byref(a), None) == WORKSPACE
    a.workspace, a.workspace_size = 1 << 30, need - 1
    assert lib.gqa_attn_launch(C.byref(a), None) == WORKSPACE
    a.workspace, a.workspace_size = (1 << 30) + 128, need
    assert lib.gqa_attn_launch(C.byref(a), None) == WORKSPACE
    w = _attn(weights=65536, w_nb1=2048, w_nb2=4096)
    assert lib.gqa_attn_workspace_size(C.byref(w)) >= need + 3 * 8 * 4 * 128 * 4       # every score, in f32
    empty = _attn(n_seq=0, q=None, block_table=None)
    assert lib.gqa_attn_check(C.byref(empty)) == 0 and lib.gqa_attn_launch(C.byref(empty), None) == 0
    for dk, dv in ((64, 64), (192, 128), (256, 256)):
        a = _attn(dk=dk, dv=dv, k=_pool(dk), v=_pool(dv))
        assert lib.gqa_attn_check(C.byref(a)) == 0


@pytest.mark.parametrize("kw,code", [(dict(weights=None), NULL), (dict(dst=32768), UNSUPPORTED), (dict(v=_pool(512, 1)), UNSUPPORTED)], ids=_name)
def test_latent_weights_refuse(kw, code):
    a = _latent()
    assert J.library().gqa_attn_check(C.byref(a)) == 0
    a = _latent(**kw)
    assert J.library().gqa_attn_check(C.byref(a)) == code


@pytest.mark.parametrize("n_head,n_head_kv", [(128, 2), (128, 128), (4, 2)])
def test_latent_weights_refuse_more_than_one_kv_head(n_head, n_head_kv):
    a = _latent(n_head=n_head, n_head_kv=n_head_kv, k=_pool(576, n_head_kv))
    assert J.library().gqa_attn_check(C.byref(a)) == UNSUPPORTED and J.library().gqa_attn_workspace_size(C.byref(a)) == 0
    assert J.library().gqa_attn_launch(C.byref(a), None) == UNSUPPORTED


def _rows(**kw):
    a = J.GqaNormRopeArgs()
    a.n_tok, a.n_head, a.n_head_kv, a.dk, a.dv, a.n_seq = 4, 8, 2, 128, 128, 3
    a.src_type = a.dst_type = a.kv_type = J.MLA_TYPE_BF16
    a.w_type = J.MLA_TYPE_F32
    a.q, a.q_nb1, a.q_nb2 = 4096, 256, 2048
    a.k, a.k_nb1, a.k_nb2 = 8192, 256, 512
    a.v, a.v_nb1, a.v_nb2 = 16384, 256, 512
    a.q_weight, a.k_weight, a.eps = 1 << 16, 1 << 17, 1e-6
    a.n_dims, a.mode, a.n_ctx_orig = 128, 2, 4096
    a.freq_base, a.freq_scale, a.ext_factor, a.attn_factor, a.beta_fast, a.beta_slow = 1e4, 1.0, 0.0, 1.0, 32.0, 1.0
    a.pos, a.q_dst, a.qd_nb1, a.qd_nb2 = 1 << 18, 1 << 19, 256, 2048
    a.k_cache, a.v_cache, a.n_pages = _pool(128), _pool(128, base=1 << 24), 16
    a.block_table, a.bt_stride, a.seq_ids = 1 << 21, 4, 1 << 22
    for name, v in kw.items():
        o = a
        *path, last = name.split("__")
        for part in path:
            o = getattr(o, part)
        setattr(o, last, v)
    return a


ROWS_REFUSED = [
    (dict(src_type=J.MLA_TYPE_Q8_0), TYPE), (dict(w_type=2), TYPE), (dict(dst_type=2), TYPE), (dict(kv_type=J.MLA_TYPE_F32), TYPE), (dict(kv_type=J.MLA_TYPE_Q8_0), TYPE),
    (dict(n_tok=-1), SHAPE), (dict(n_head=0), SHAPE), (dict(dk=0), SHAPE), (dict(dk=100), SHAPE), (dict(dk=264), SHAPE), (dict(dv=4), SHAPE), (dict(dv=512), SHAPE),
    (dict(n_head_kv=0), SHAPE), (dict(n_seq=-1), SHAPE), (dict(k=None), SHAPE),
    (dict(mode=1), UNSUPPORTED), (dict(n_dims=-8), SHAPE), (dict(n_dims=136), SHAPE), (dict(n_dims=24), SHAPE), (dict(n_dims=12, mode=0), SHAPE),
    (dict(freq_base=1.0), UNSUPPORTED), (dict(freq_base=float("nan")), UNSUPPORTED), (dict(ext_factor=1.0, freq_scale=0.0), UNSUPPORTED), (dict(ext_factor=1.0, n_ctx_orig=0), UNSUPPORTED),
    (dict(ext_factor=1.0, beta_fast=0.0), UNSUPPORTED),
    (dict(q=None), NULL), (dict(pos=None), NULL), (dict(q_dst=None), NULL), (dict(block_table=None), NULL), (dict(seq_ids=None), NULL), (dict(k_cache__data=None), NULL), (dict(v_cache__data=None), NULL),
    (dict(q=4100), ALIGN), (dict(q_nb1=248), ALIGN), (dict(k_nb2=520), ALIGN), (dict(v=16392), ALIGN), (dict(qd_nb2=2040), ALIGN), (dict(q_weight=65540), ALIGN), (dict(k_weight=65540), ALIGN),
    (dict(k_cache__nb_row=516), ALIGN), (dict(v_cache__nb_head=8), ALIGN), (dict(k_cache__nb_page=-65536), SHAPE), (dict(n_pages=0), SHAPE), (dict(bt_stride=0), SHAPE),
]


@pytest.mark.parametrize("kw,code", ROWS_REFUSED, ids=lambda x: str(x)[:60])
def test_norm_rope_refuses(kw, code):
    lib = J.library()
    a = _rows(**kw)
    assert lib.gqa_norm_rope_check(C.byref(a)) == code
    assert lib.gqa_norm_rope_launch(C.byref(a), None) == code


def test_norm_rope_accepts():
    lib = J.library()
    assert lib.gqa_norm_rope_check(None) == NULL
    for kw in (dict(), dict(k=None, v=None, k_cache=J.GqaPool(), block_table=None), dict(v=None, v_cache=J.GqaPool()), dict(n_dims=0), dict(q_weight=None, k_weight=None),
               dict(mode=0, n_dims=8), dict(slots=64), dict(n_tok=0, q=None, pos=None)):
        a = _rows(**kw)
        assert lib.gqa_norm_rope_check(C.byref(a)) == 0, kw
    a = _rows(n_tok=0)
    assert lib.gqa_norm_rope_launch(C.byref(a), None) == 0


def _cut(**kw):
    a = J.GqaEvictArgs()
    a.n_seq, a.n_head_kv, a.n_keep, a.n_sink, a.n_recent, a.k_row_bytes, a.v_row_bytes = 3, 2, 100, 4, 20, 256, 256
    a.k, a.v, a.n_pages = _pool(128), _pool(128, base=1 << 24), 16
    a.block_table, a.bt_stride, a.seq_lens = 8192, 4, 16384
    a.weights, a.w_nb1, a.w_nb2 = 32768, 2048, 4096
    a.weights_dst, a.wd_nb1, a.wd_nb2 = 65536, 2048, 4096
    a.kept, a.new_lens = 1 << 17, 1 << 18
    for name, v in kw.items():
        o = a
        *path, last = name.split("__")
        for part in path:
            o = getattr(o, part)
        setattr(o, last, v)
    return a


CUT_REFUSED = [
    (dict(n_seq=-1), SHAPE), (dict(n_head_kv=0), SHAPE), (dict(n_keep=0), SHAPE), (dict(n_sink=-1), SHAPE), (dict(n_recent=-1), SHAPE), (dict(n_sink=60, n_recent=41), SHAPE),
    (dict(n_sink=2 ** 31 - 1, n_recent=2 ** 31 - 1), SHAPE), (dict(n_pages=0), SHAPE), (dict(bt_stride=0), SHAPE), (dict(bt_stride=1 << 23), SHAPE), (dict(n_seq=40000), SHAPE),
    (dict(weights=None), NULL), (dict(weights_dst=None), NULL), (dict(kept=None), NULL), (dict(new_lens=None), NULL), (dict(block_table=None), NULL), (dict(seq_lens=None), NULL), (dict(k__data=None), NULL),
    (dict(k_row_bytes=255), ALIGN), (dict(k_row_bytes=0), SHAPE), (dict(k_row_bytes=4), SHAPE), (dict(v_row_bytes=16388), SHAPE), (dict(v__nb_row=511), ALIGN), (dict(v__data=(1 << 24) + 1), ALIGN), (dict(k__nb_head=-256), SHAPE),
    (dict(weights=32769), ALIGN), (dict(wd_nb2=4095), ALIGN), (dict(weights_dst=32768, wd_nb1=4096), SHAPE), (dict(new_lens=16384), UNSUPPORTED),
]


@pytest.mark.parametrize("kw,code", CUT_REFUSED, ids=lambda x: str(x)[:60])
def test_evict_refuses(kw, code):
    lib = J.library()
    a = _cut(**kw)
    assert lib.gqa_evict_check(C.byref(a)) == code
    assert lib.gqa_evict_launch(C.byref(a), None) == code


def test_evict_accepts():
    lib = J.library()
    assert lib.gqa_evict_check(None) == NULL
    for kw in (dict(), dict(v=J.GqaPool(), v_row_bytes=0), dict(k_row_bytes=612), dict(weights_dst=32768), dict(n_sink=0, n_recent=100), dict(n_seq=0, weights=None)):
        a = _cut(**kw)
        assert lib.gqa_evict_check(C.byref(a)) == 0, kw
    a = _cut()
    need = lib.gqa_evict_workspace_size(C.byref(a))
    assert need > 0 and lib.gqa_evict_launch(C.byref(a), None) == WORKSPACE
    a.workspace, a.workspace_size = 1 << 30, need - 1
    assert lib.gqa_evict_launch(C.byref(a), None) == WORKSPACE
    assert lib.gqa_evict_workspace_size(C.byref(_cut(n_keep=0))) == 0


def test_launches_of_more_threads_than_there_are_refused():
    """Nothing starts of a call whose last kernel could not: 65532 heads of rows of 612 bytes, 40 rows a workgroup."""
    lib = J.library()
    far = dict(n_seq=32766, k_row_bytes=612, v=J.GqaPool(), bt_stride=1024, w_nb1=1024 * 512, w_nb2=1024 * 1024, wd_nb1=1024 * 512, wd_nb2=1024 * 1024, weights_dst=1 << 40)
    assert lib.gqa_evict_check(C.byref(_cut(n_keep=100000, **far))) == SHAPE and lib.gqa_evict_workspace_size(C.byref(_cut(n_keep=100000, **far))) == 0
    assert lib.gqa_evict_check(C.byref(_cut(n_keep=5000, **far))) == 0
    assert lib.gqa_norm_rope_check(C.byref(_rows(n_tok=1 << 24))) == SHAPE and lib.gqa_norm_rope_check(C.byref(_rows(n_tok=(1 << 24) - 1))) == 0


@pytest.mark.parametrize("kw", [dict(weights_dst=32768 + 4), dict(weights_dst=32768 - 2044), dict(weights_dst=32768 + 2044), dict(v=_pool(128))], ids=_name)
def test_evict_refuses_what_overlaps(kw):
    a = _cut(**kw)
    assert J.library().gqa_evict_check(C.byref(a)) == UNSUPPORTED and J.library().gqa_evict_launch(C.byref(a), None) == UNSUPPORTED
    for dst in (32768, 32768 + 2048, 32768 - 2048):       # itself; rows between the rows (4 rows of 2048 bytes in 8192)
        a = _cut(w_nb1=4096, w_nb2=8192, wd_nb1=4096, wd_nb2=8192, weights_dst=dst)
        assert J.library().gqa_evict_check(C.byref(a)) == 0


@pytest.mark.parametrize("kw", [dict(q_dst=4096, qd_nb1=512, qd_nb2=4096), dict(q_dst=4096, dst_type=J.MLA_TYPE_F16), dict(q_dst=4096 + 16), dict(q_dst=4096 - 240), dict(q_dst=4096 - 256, dst_type=J.MLA_TYPE_F32),
                                dict(v_cache=_pool(128))], ids=_name)
def test_norm_rope_refuses_what_overlaps(kw):
    a = _rows(**kw)
    assert J.library().gqa_norm_rope_check(C.byref(a)) == UNSUPPORTED and J.library().gqa_norm_rope_launch(C.byref(a), None) == UNSUPPORTED
    for dst in (4096, 4096 + 256, 4096 - 256):
        a = _rows(q_nb1=512, q_nb2=4096, qd_nb1=512, qd_nb2=4096, q_dst=dst)
        assert J.library().gqa_norm_rope_check(C.byref(a)) == 0


def test_exports_and_mirrors_match_the_header(tmp_path):
    """Every function the header declares is exported; every ctypes mirror has the C compiler's size and field offsets."""
    text = open(os.path.join(ROOT, "include", "gqa_attn.h")).read()
    bare = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    declared = set(re.findall(r"\b(gqa_\w+)\s*\(", bare))
    assert declared == {p + s for p in ("gqa_norm_rope", "gqa_attn", "gqa_evict") for s in ("_check", "_launch")} | {"gqa_attn_workspace_size", "gqa_evict_workspace_size"}
    for name in declared:
        assert hasattr(J.library(), name)
    mirrors = {"gqa_pool": J.GqaPool, "gqa_norm_rope_args": J.GqaNormRopeArgs, "gqa_attn_args": J.GqaAttnArgs, "gqa_evict_args": J.GqaEvictArgs}
    lines = []
    for name, cls in mirrors.items():
        lines.append('printf("%s . %%zu\\n", sizeof(%s));' % (name, name))
        lines += ['printf("%s %s %%zu\\n", offsetof(%s, %s));' % (name, f[0], name, f[0]) for f in cls._fields_]
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "gqa_attn.h"\nint main(void){%s return 0;}\n' % "\n".join(lines))
    subprocess.run(["gcc", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "t")], check=True)
    for line in subprocess.run([str(tmp_path / "t")], check=True, stdout=subprocess.PIPE, text=True).stdout.splitlines():
        name, field, value = line.split()
        assert int(value) == (C.sizeof(mirrors[name]) if field == "." else getattr(mirrors[name], field).offset), (name, field)


def test_seq_evict_gives_pages_back():
    pt = J.PageTable(8, 3, 4)
    pt.find_slot([0] * 400, list(range(400)))
    assert pt.free_pages == 4
    assert pt.seq_evict(0, 400) and pt.seq_evict(0, 1000) and pt.seq_len(0) == 400 and pt.free_pages == 4       # nothing to cut
    assert pt.seq_evict(0, 130) and pt.seq_len(0) == 130 and pt.free_pages == 6
    assert pt.find_slot([0], [130]) is not None and pt.seq_len(0) == 131                                          # the next row follows the ones kept
    for args in ((0, 0), (0, -1), (3, 10), (-1, 10)):
        with pytest.raises(ValueError):
            pt.seq_evict(*args)
    assert pt.seq_len(0) == 131


def test_seq_evict_refuses_shared_pages():
    pt = J.PageTable(8, 3, 4)
    pt.find_slot([0] * 300, list(range(300)))
    pt.seq_cp(0, 1)
    assert not pt.seq_evict(0, 100) and not pt.seq_evict(1, 100)
    assert pt.seq_len(0) == pt.seq_len(1) == 300
    pt.seq_rm(1)
    assert pt.seq_evict(0, 100) and pt.free_pages == 7


CALLS = r"""
import json
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
import jittorinfer_amd as J
with FakeTensorMode():
    f = lambda *shape, dtype=torch.bfloat16: torch.empty(shape, dtype=dtype, device="cuda")
    i = lambda *shape: f(*shape, dtype=torch.int32)
    q, k, v, bt, lens = f(2, 4, 64), f(3, 128, 2, 64), f(3, 128, 2, 64), i(2, 1), i(2)
    x, pos, w = f(5, 2, 64), i(5), f(2, 2, 128, dtype=torch.float32)
    wide = f(3, 128, 2, 64, dtype=torch.float32)
A = lambda **kw: J.gqa_attn(**{**dict(q=q, k_cache=k, v_cache=v, block_table=bt, seq_lens=lens, scale=1.0), **kw})
N = lambda **kw: J.gqa_norm_rope(**{**dict(q=x, k=x, v=x, pos=pos, n_dims=64, k_cache=k, v_cache=v, block_table=bt, seq_ids=pos), **kw})
E = lambda **kw: J.gqa_evict(**{**dict(weights=w, block_table=bt, seq_lens=lens, k_cache=k, v_cache=v, n_keep=10), **kw})
cpu = torch.zeros(2, dtype=torch.int32)
calls = dict(
    attn_cpu=lambda: A(q=torch.zeros(2, 4, 64)), attn_table_on_cpu=lambda: A(seq_lens=cpu), attn_q_dims=lambda: A(q=x[0]), attn_cache_type=lambda: A(k_cache=wide), attn_cache_width=lambda: A(q=q[..., :32]),
    attn_v_pages=lambda: A(v_cache=v[:2]), attn_table_rows=lambda: A(block_table=bt[:1]), attn_table_type=lambda: A(block_table=w[:, 0, :1]), attn_lens=lambda: A(seq_lens=lens[:1]),
    attn_mask_type=lambda: A(mask=w[:, 0]), attn_mask_rows=lambda: A(mask=w[:1, 0].half()), attn_weights_short=lambda: A(weights=w[..., :100]), attn_weights_type=lambda: A(weights=w.half()),
    attn_weights_expanded=lambda: A(weights=w[:1].expand(2, 2, 128)), attn_window=lambda: A(window=-1), attn_window_big=lambda: A(window=1 << 40), attn_no_values=lambda: A(v_cache=None), attn_page=lambda: A(k_cache=k[:, :64], v_cache=v[:, :64]),
    attn_none=lambda: A(q=None), attn_list=lambda: A(seq_lens=[1, 2]), attn_scale=lambda: A(scale="x"), attn_column=lambda: A(q=q.transpose(1, 2)), attn_cache_expanded=lambda: A(k_cache=k[:1].expand(3, 128, 2, 64)),
    attn_alloc=lambda: A(), attn_alloc_weights=lambda: A(weights=w),
    rows_cpu=lambda: N(q=torch.zeros(5, 2, 64)), rows_tokens=lambda: N(k=x[:4]), rows_types=lambda: N(k=x.half()), rows_pos=lambda: N(pos=pos[:3]), rows_no_cache=lambda: N(k_cache=None), rows_v_no_cache=lambda: N(v_cache=None),
    rows_cache_no_k=lambda: N(k=None, v=None), rows_weight=lambda: N(q_weight=w[0, 0, :32]), rows_weight_types=lambda: N(q_weight=w[0, 0, :64], k_weight=x[0, 0]), rows_ids=lambda: N(seq_ids=pos[:1]), rows_slots=lambda: N(slots=w[0, 0, :5]),
    rows_heads=lambda: N(k=x[:, :1], v=x[:, :1]), rows_v_width=lambda: N(v=x[..., :32]), rows_out=lambda: N(q_out=x[:3]), rows_factors=lambda: N(freq_factors=w[0, 0, :8]), rows_out_expanded=lambda: N(q_out=x[:1].expand(5, 2, 64)),
    rows_alloc=lambda: N(),
    cut_cpu=lambda: E(weights=torch.zeros(2, 2, 128)), cut_weights=lambda: E(weights=w[..., :100]), cut_heads=lambda: E(weights=w[:, :1]), cut_lens=lambda: E(seq_lens=lens[:1]), cut_v=lambda: E(v_cache=v[:, :, :1]), cut_keep=lambda: E(n_keep=-1),
    cut_kept=lambda: E(kept=i(2, 2, 11)), cut_new=lambda: E(new_lens=i(3)), cut_out=lambda: E(weights_out=w[..., :127]), cut_out_expanded=lambda: E(weights_out=w[:1].expand(2, 2, 128)), cut_alloc=lambda: E(),
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
    assert len(seen) == 53 and set(seen.values()) == {"raised"}, {k: v for k, v in seen.items() if v != "raised"}


# ---------------------------------------------------------------- the plain forms themselves

def test_plain_attention_is_softmax():
    gen = torch.Generator().manual_seed(0)
    bt = torch.tensor([[1, 0]], dtype=torch.int32)
    k, v = (R.make_cache(gen, 2, 1, 4, torch.float32) for _ in range(2))
    q = torch.randn((1, 2, 4), generator=gen)
    out, _, w, _ = R.attn(q, k, v, bt, [200], 0.5)
    rows = torch.cat((k[1], k[0]))[:200, 0].double()
    vals = torch.cat((v[1], v[0]))[:200, 0].double()
    for h in range(2):
        e = [math.exp(0.5 * float(q[0, h].double() @ r)) for r in rows]
        want = sum(x * y for x, y in zip(e, vals)) / sum(e)
        assert torch.allclose(out[0, h], want, rtol=1e-12)
    assert abs(float(w.sum()) - 2) < 1e-12 and (w[0, 0, 200:] == 0).all()


def test_plain_eviction_by_hand():
    bt = torch.tensor([[0]], dtype=torch.int32)
    k = torch.arange(128.0).view(1, 128, 1, 1)
    w = torch.zeros((1, 1, 128))
    w[0, 0, :8] = torch.tensor([0.0, 5.0, 1.0, 3.0, 3.0, 3.0, 9.0, 0.0])
    kept, new, out, k2, _ = R.evict(w, bt, [8], k, None, 5, 1, 1)
    assert kept[0, 0].tolist() == [0, 1, 3, 6, 7] and new.tolist() == [5]          # 5, 9 and the first of the three 3s, beside the ends
    assert out[0, 0, :6].tolist() == [0, 5, 3, 9, 0, 0] and k2[0, :8, 0, 0].tolist() == [0, 1, 3, 6, 7, 5, 6, 7]


def test_plain_rotation_is_a_rotation():
    x = torch.randn((3, 2, 16), generator=torch.Generator().manual_seed(1))
    y, _ = R.heads(x, None, 0, torch.tensor([0, 1, 1000]), 16, 0)
    assert torch.allclose(y[0], x[0].double()) and torch.allclose(y.norm(dim=-1), x.double().norm(dim=-1))
    a, b = float(x[1, 0, 0]), float(x[1, 0, 1])
    assert abs(float(y[1, 0, 0]) - (a * math.cos(1) - b * math.sin(1))) < 1e-6


def test_constants_of_the_module():
    assert capi.PAGE_TOKENS == R.PAGE
