"""The paged cache of ordinary heads without a GPU, at its edges: what the entry points of include/gqa_attn.h refuse and accept beside tests/test_gqa.py."""
import ctypes as C
import os
import subprocess

import pytest

import jittorinfer_amd as J
from tests.test_gqa import ROOT, SHAPE, UNSUPPORTED, _attn, _cut, _latent, _pool, _rows


@pytest.mark.parametrize("cap,code", [(float("inf"), UNSUPPORTED), (float("nan"), UNSUPPORTED), (3.4e38, 0), (1e-45, 0)])
def test_softcaps_are_finite(cap, code):
    """c tanh(s / c) has no value at an infinite c."""
    for a in (_attn(logit_softcap=cap), _latent(logit_softcap=cap)):
        assert J.library().gqa_attn_check(C.byref(a)) == code


def test_scratch_is_allocated_as_its_own_streams(monkeypatch):
    """An area for a stream that is not the current one is allocated with that stream as the current one (a stand-in for torch's allocator, on the CPU)."""
    import contextlib
    import sys
    import types
    import jittorinfer_amd.capi as capi

    now, made = [7], []

    @contextlib.contextmanager
    def stream(s):
        now.append(s)
        yield
        now.pop()
    cuda = types.SimpleNamespace(current_stream=lambda d: types.SimpleNamespace(cuda_stream=now[-1]), stream=stream, ExternalStream=lambda h, device=None: h,
                                 default_stream=lambda d: 0, is_current_stream_capturing=lambda: now[-1] == 11)
    fake = types.SimpleNamespace(uint8=None, cuda=cuda, empty=lambda n, dtype=None, device=None: made.append(now[-1]) or types.SimpleNamespace(numel=lambda: n))
    monkeypatch.setitem(sys.modules, "torch", fake)
    monkeypatch.setattr(capi, "_workspaces", {})
    monkeypatch.setattr(capi, "_retired", [])
    for s in (7, 9, 0):
        ws = capi._workspace("dev", 1 << 21, stream=s)
        assert capi._workspace("dev", 1 << 20, stream=s) is ws and now == [7]
    assert capi._scratch_elsewhere("dev", 1 << 21, 9) is capi._workspaces["dev", 9]
    assert made == [7, 9, 0]
    own = capi._scratch_elsewhere("dev", 100, 11)                    # under capture: the graph's own, kept in no table
    assert made == [7, 9, 0, 11] and own.numel() == 100 and ("dev", 11) not in capi._workspaces and now == [7]


def test_scratch_areas_have_locks_of_their_own(tmp_path):
    """Areas as the allocator places them (2 MB apart and further, or 512 bytes) do not wait for each other; the same area does, and no area holds nothing."""
    src = tmp_path / "t.cpp"
    src.write_text(r"""
#include "scratch_lock.hpp"
#include <set>
#include <thread>
int main() {
    for (uint64_t base : { 0x7f0000000000ull, 0x7e1c40000000ull }) for (uint64_t step : { 512ull, 1ull << 21, 1ull << 23, 1ull << 26, 1ull << 30 }) {
        std::set<unsigned> seen;
        for (uint64_t i = 0; i < 16; i++) seen.insert(mla::scratch_lock_index((const void *) (base + i * step)));
        if (seen.size() < 14) return 1;
        for (unsigned i : seen) if (i >= 256) return 2;
    }
    { const mla::ScratchLock a(nullptr), b(nullptr); const mla::ScratchLock c((const void *) 0x7f0000200000ull); }
    int inside = 0, most = 0, done = 0;
    auto work = [&] { for (int i = 0; i < 20000; i++) { const mla::ScratchLock l((const void *) 0x7f0000200000ull); most = ++inside > most ? inside : most; --inside; done++; } };
    std::thread t(work); work(); t.join();
    return most == 1 && done == 40000 ? 0 : 3;
}
""")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I", os.path.join(ROOT, "jittorinfer_amd", "csrc"), str(src), "-o", str(tmp_path / "t"), "-pthread"], check=True)
    assert subprocess.run([str(tmp_path / "t")], timeout=60).returncode == 0


def test_evict_of_many_segments_a_head():
    """Rows that fill a segment of the move alone: as many may stay as a launch has workgroups for, whatever a head's share of them."""
    lib = J.library()
    one = dict(n_seq=1, n_head_kv=1, k_row_bytes=16384, v=J.GqaPool(), bt_stride=1 << 17, w_nb1=1 << 26, w_nb2=1 << 26, wd_nb1=1 << 26, wd_nb2=1 << 26, weights_dst=1 << 40)
    odd = J.GqaPool(1 << 20, 128 * 16388, 16388, 16388)
    for n_keep, code in ((32256, 0), (32257, 0), ((1 << 23) - 1, 0), (1 << 23, SHAPE)):
        a = _cut(k=odd, n_keep=n_keep, **one)
        assert lib.gqa_evict_check(C.byref(a)) == code, n_keep
        assert (lib.gqa_evict_workspace_size(C.byref(a)) > 4 * n_keep) == (code == 0)


@pytest.mark.parametrize("kw", [dict(dst=4096), dict(dst=1 << 20), dict(dst=1 << 24), dict(dst=16384), dict(weights=1 << 20), dict(weights=8192), dict(weights=32768), dict(weights=4096)], ids=str)
def test_attn_refuses_results_on_its_operands(kw):
    a = _attn(w_nb1=2048, w_nb2=4096, **kw)
    assert J.library().gqa_attn_check(C.byref(a)) == UNSUPPORTED and J.library().gqa_attn_launch(C.byref(a), None) == UNSUPPORTED


def test_overlap_of_strided_tensors(tmp_path):
    """What says whether two tensors share bytes, against their sets of bytes: views of one buffer with the same strides, and any two."""
    src = tmp_path / "t.cpp"
    src.write_text(r"""
#include "tensor_overlap.hpp"
#include <random>
#include <set>
#include <vector>
struct T { int64_t at, el; std::vector<int64_t> n, s; };
static std::set<int64_t> bytes(const T & t) {
    std::set<int64_t> r;
    std::vector<int64_t> i(t.n.size(), 0);
    for (auto x : t.n) if (!x) return r;
    for (;;) {
        int64_t a = t.at;
        for (size_t d = 0; d < i.size(); d++) a += i[d] * t.s[d] * t.el;
        for (int64_t e = 0; e < t.el; e++) r.insert(a + e);
        size_t d = 0;
        for (; d < i.size(); d++) { if (++i[d] < t.n[d]) break; i[d] = 0; }
        if (d == i.size()) return r;
    }
}
static mla::Extent extent(const T & t) { return mla::Extent((const void *) t.at, t.el, (int) t.n.size(), t.n.data(), t.s.data()); }
int main() {
    std::mt19937 g(1);
    auto rnd = [&](int lo, int hi) { return (int64_t) (lo + g() % (hi - lo + 1)); };
    long met = 0;
    for (int it = 0; it < 20000; it++) {
        T a, b;
        const bool alike = it % 2;
        a.el = 1 << rnd(0, 2); b.el = alike ? a.el : 1 << rnd(0, 2);
        a.at = 10000; b.at = 10000 + (alike ? a.el * rnd(-60, 60) : rnd(-120, 120));
        int64_t st = 1;
        for (int i = 0, d = rnd(1, 3); i < d; i++) {
            const int64_t na = rnd(1, 4), nb = rnd(1, 4);
            a.n.push_back(na); a.s.push_back(st);
            if (alike) { b.n.push_back(nb); b.s.push_back(st); }
            st = st * (na > nb ? na : nb) + rnd(0, 3);
        }
        if (!alike) {
            for (int i = 0, d = rnd(0, 3); i < d; i++) { b.n.push_back(rnd(0, 4)); b.s.push_back(rnd(0, 20)); }
            if (rnd(0, 1)) for (auto & x : a.s) x = rnd(0, 20);
        }
        const auto p = bytes(a), q = bytes(b);
        bool over = false;
        for (auto x : p) over = over || q.count(x);
        met += over;
        const mla::Shares want = over ? mla::Shares::YES : mla::Shares::NO;
        if (mla::shares(extent(a), extent(b)) != want || mla::shares(extent(b), extent(a)) != want) return 1;
    }
    if (met < 1000 || met > 19000) return 2;
    // large ones: two caches side by side in every page; a tensor in the gaps of another, which takes more looks than there are
    const int64_t big = (int64_t) 1 << 40;
    T k{ big, 2, { 20000, 128, 8, 128 }, { 2 * 131072, 1024, 128, 1 } }, v = k, w{ big + 4096, 4, { 1 << 20 }, { 997 } };
    v.at += 2 * 131072;
    if (mla::shares(extent(k), extent(v)) != mla::Shares::NO) return 3;
    v.at -= 2;
    if (mla::shares(extent(k), extent(v)) != mla::Shares::YES) return 4;
    if (mla::shares(extent(k), extent(w)) == mla::Shares::NO) return 5;
    return 0;
}
""")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I", os.path.join(ROOT, "jittorinfer_amd", "csrc"), str(src), "-o", str(tmp_path / "t")], check=True)
    assert subprocess.run([str(tmp_path / "t")], timeout=60).returncode == 0


def test_attn_refuses_groups_whose_last_launch_could_not_start():
    """A workgroup a head of a group and 2048 for the weights: fewer than 2^24."""
    lib = J.library()
    far = dict(n_seq=1, n_head_kv=1, bt_stride=1, q_nb1=256, q_nb2=1 << 33, weights=1 << 40, w_nb1=512, w_nb2=512, d_nb1=256, d_nb2=1 << 33)
    assert lib.gqa_attn_check(C.byref(_attn(n_head=(1 << 24) - 2048, **far))) == SHAPE
    assert lib.gqa_attn_check(C.byref(_attn(n_head=(1 << 24) - 2049, **far))) == 0
