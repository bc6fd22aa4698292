// The Python entry points' way from torch tensors to the C ABI (include/mla_attn.h, mla_kv_write.h, mla_front.h, gqa_attn.h, gqa_batch.h): one call that checks the
// tensors, fills the argument block and launches.  Filling a ctypes structure field by field took 6 us of a 13 us attention call and
// most of the 70 us a layer of a decode step spent on the host, more than its kernels run for small batches; here it takes
// under 1 us a call.  Every function takes its arguments by position; capi.py gives them names and defaults.
// What torch throws (out of memory, a tensor without strides or storage) ends at entry<>, as the Python exception torch itself would
// raise; every reference and buffer taken on the way has an owner that gives it back.
#include <Python.h>

#include <string.h>

#include <algorithm>
#include <vector>

#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include "../../include/gqa_attn.h"
#include "../../include/gqa_batch.h"
#include "../../include/mla_attn.h"
#include "../../include/mla_front.h"
#include "../../include/mla_kv_write.h"
#include "scratch_lock.hpp"
#include "tensor_overlap.hpp"

namespace {

constexpr int PAGE = MLA_PAGE_TOKENS;

// A launch may wait for room in the device's queue: other Python threads run meanwhile.
struct Unlocked {
    PyThreadState * t = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(t); }
};
template <typename F> int unlocked(F f) {
    const Unlocked u;
    return f();
}
// The same for a launch of several kernels that hand each other scratch: two threads on one stream share it, and the kernels of one call must
// not be queued between those of another.
template <typename F> int unlocked(const void * scratch, F f) {
    const Unlocked u;
    const mla::ScratchLock l(scratch);
    return f();
}

// The library's entry points, the Python layer's workspace table and what grows it, torch's raw current stream: handed over by bind().
struct Bound {
    decltype(&mla_attn_workspace_size) workspace_size;
    decltype(&mla_attn_launch)         attn;
    decltype(&mla_kv_write_launch)     kv_write;
    decltype(&mla_kv_write_rope_launch) kv_write_rope;
    decltype(&mla_rope_launch)         rope;
    decltype(&mla_mul_mat_launch)      mul_mat;
    decltype(&mla_copy_f32_launch)     copy;
    decltype(&mla_front_batch_launch)  front_batch;
    decltype(&gqa_norm_rope_launch)    norm_rope;
    decltype(&gqa_attn_workspace_size) gqa_workspace_size;
    decltype(&gqa_attn_launch)         gqa_attn;
    decltype(&gqa_evict_workspace_size) evict_workspace_size;
    decltype(&gqa_evict_launch)        evict;
    decltype(&gqa_prompt_attn_workspace_size) prompt_workspace_size;
    decltype(&gqa_prompt_attn_launch)  prompt_attn;
    decltype(&gqa_cross_attn_workspace_size) cross_workspace_size;
    decltype(&gqa_cross_attn_launch)   cross_attn;
    decltype(&gqa_prefix_attn_workspace_size) prefix_workspace_size;
    decltype(&gqa_prefix_attn_launch)  prefix_attn;
    PyObject * workspace, * workspaces, * raw_stream, * capturing, * elsewhere;
} lib;

#define REQUIRE(cond)                                        \
    do {                                                     \
        if (!(cond)) {                                       \
            PyErr_SetString(PyExc_AssertionError, #cond);    \
            return nullptr;                                  \
        }                                                    \
    } while (0)

const at::Tensor * tensor(PyObject * o) {
    if (THPVariable_Check(o)) return &THPVariable_Unpack(o);
    PyErr_SetString(PyExc_TypeError, "expected a torch tensor");
    return nullptr;
}
// a tensor or None
bool optional_tensor(PyObject * o, const at::Tensor *& t) {
    t = nullptr;
    if (o == Py_None) return true;
    t = tensor(o);
    return t != nullptr;
}
bool on_gpu(const at::Tensor & t) {
    if (t.is_cuda()) return true;
    PyErr_SetString(PyExc_RuntimeError, "jittorinfer_amd runs on a gfx950 GPU only (there is no CPU path)");
    return false;
}
bool arg_count(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
    return false;
}
PyObject * failed(const char * what, int rc) {
    PyErr_Format(PyExc_RuntimeError, "%s failed with code %d", what, rc);
    return nullptr;
}
// the stream to launch on: a raw handle, or None for the tensor's device's current one
bool stream_of(PyObject * o, const at::Tensor & t, void *& st) {
    if (o != Py_None) {
        st = PyLong_AsVoidPtr(o);
        return !PyErr_Occurred();
    }
    THPObjectPtr idx(PyLong_FromLong(t.device().index()));
    THPObjectPtr raw(idx ? PyObject_CallOneArg(lib.raw_stream, idx.get()) : nullptr);
    if (!raw) return false;
    st = PyLong_AsVoidPtr(raw.get());
    return !PyErr_Occurred();
}
// ggml-order sizes and byte strides of a tensor of up to 4 dimensions (last torch dimension = ggml dimension 0)
void nb4(const at::Tensor & t, int64_t ne[4], int64_t nb[4]) {
    const int d = (int) t.dim();
    const int64_t es = (int64_t) t.element_size();
    for (int i = 0; i < 4; i++) ne[i] = i < d ? t.size(d - 1 - i) : 1;
    for (int i = 0; i < 4; i++) nb[i] = i < d ? t.stride(d - 1 - i) * es : nb[i - 1] * ne[i - 1];
}
int64_t row_bytes(long kv_type) { return kv_type == MLA_TYPE_F16 || kv_type == MLA_TYPE_BF16 ? 1152 : kv_type == MLA_TYPE_Q8_0 ? 612 : -1; }

// The scratch area of (device, stream): a look-up in the Python layer's table; too small or missing, the Python layer makes one.  The
// caller keeps what is returned until its launch is queued: another thread may give areas back meanwhile.
template <typename Args> THPObjectPtr workspace(PyObject * q, void * st, size_t need, Args & a) {
    THPObjectPtr dev(PyObject_GetAttrString(q, "device")), handle(dev ? PyLong_FromVoidPtr(st) : nullptr);
    THPObjectPtr key(handle ? PyTuple_Pack(2, dev.get(), handle.get()) : nullptr);
    if (!key) return THPObjectPtr();
    PyObject * const found = PyDict_GetItemWithError(lib.workspaces, key.get());
    if (!found && PyErr_Occurred()) return THPObjectPtr();
    THPObjectPtr ws(Py_XNewRef(found));
    if (!ws || (size_t) THPVariable_Unpack(ws.get()).numel() < need) {
        THPObjectPtr n(PyLong_FromSize_t(need));
        ws = n ? PyObject_CallFunctionObjArgs(lib.workspace, dev.get(), n.get(), handle.get(), nullptr) : nullptr;
        if (!ws) return ws;
    }
    const at::Tensor * t = tensor(ws.get());
    if (!t) return THPObjectPtr();
    a.workspace = t->data_ptr(); a.workspace_size = (size_t) t->numel();
    return ws;
}

// attn(q, k, kv_type, dv, mask, scale, max_bias, logit_softcap, block_table, seq_lens, out, n_splits, flags, rows_per_wg, stream) -> out
PyObject * attn(PyObject *, PyObject * const * v, Py_ssize_t n) {
    if (!arg_count(n, 15)) return nullptr;
    const at::Tensor * qp = tensor(v[0]), * kp = qp ? tensor(v[1]) : nullptr, * mask, * table, * lens, * outp;
    if (!kp || !optional_tensor(v[4], mask) || !optional_tensor(v[8], table) || !optional_tensor(v[9], lens) || !optional_tensor(v[10], outp)) return nullptr;
    const at::Tensor & q = *qp, & k = *kp;
    if (!on_gpu(q)) return nullptr;
    mla_attn_args a;
    memset(&a, 0, sizeof a);
    a.kv_type = (int32_t) PyLong_AsLong(v[2]); a.dv = (int32_t) PyLong_AsLong(v[3]);
    a.scale = (float) PyFloat_AsDouble(v[5]); a.max_bias = (float) PyFloat_AsDouble(v[6]); a.logit_softcap = (float) PyFloat_AsDouble(v[7]);
    a.n_splits = (int32_t) PyLong_AsLong(v[11]); a.flags = (uint32_t) PyLong_AsUnsignedLongMask(v[12]); a.rows_per_wg = (int32_t) PyLong_AsLong(v[13]);
    if (PyErr_Occurred()) return nullptr;
    REQUIRE(q.scalar_type() == at::kFloat && q.dim() == 4 && q.size(3) == 576 && q.stride(3) == 1);
    const int64_t row = row_bytes(a.kv_type), es = (int64_t) k.element_size();
    if (row < 0) { PyErr_SetObject(PyExc_KeyError, v[2]); return nullptr; }
    const int64_t n_seq = q.size(0), n_head = q.size(1), n_tok = q.size(2);
    a.n_seq = (int32_t) n_seq; a.n_head = (int32_t) n_head; a.n_tok = (int32_t) n_tok; a.dk = 576; a.q_type = MLA_TYPE_F32;
    a.q = q.data_ptr(); a.q_nb1 = q.stride(2) * 4; a.q_nb2 = q.stride(1) * 4; a.q_nb3 = q.stride(0) * 4;
    REQUIRE(k.dim() >= 1 && k.stride(-1) == 1 && k.size(-1) * es == row);
    a.kv = k.data_ptr();
    if (table) {
        REQUIRE(k.dim() == 2 && k.size(0) % PAGE == 0);
        a.kv_nb1 = k.stride(0) * es; a.n_kv = k.size(0);
        REQUIRE(table->scalar_type() == at::kInt && table->dim() == 2 && table->size(0) == n_seq && table->is_contiguous());
        REQUIRE(lens && lens->scalar_type() == at::kInt && lens->numel() == n_seq && lens->is_contiguous());
        a.block_table = (const int32_t *) table->data_ptr(); a.bt_stride = table->size(1); a.seq_lens = (const int32_t *) lens->data_ptr();
    } else {
        REQUIRE(k.dim() == 3 && (k.size(0) == 1 || k.size(0) == n_seq));
        a.kv_nb1 = k.stride(1) * es; a.kv_nb3 = k.size(0) > 1 ? k.stride(0) * es : 0; a.n_kv = k.size(1);
    }
    if (mask) {
        REQUIRE(mask->scalar_type() == at::kHalf && mask->dim() == 2 && mask->stride(1) == 1 && mask->size(0) >= n_tok);
        a.mask = mask->data_ptr(); a.mask_nb1 = mask->stride(0) * 2; a.mask_ne0 = mask->size(1);
    }
    at::Tensor made;
    if (!outp) {
        made = at::empty({ n_seq, n_tok, n_head, 576 }, q.options());
        outp = &made;
    }
    const at::Tensor & out = *outp;
    REQUIRE(out.scalar_type() == at::kFloat && out.dim() == 4 && out.is_contiguous() && out.size(0) == n_seq && out.size(1) == n_tok && out.size(2) == n_head && out.size(3) >= a.dv);
    a.dst = (float *) out.data_ptr(); a.dst_nb1 = out.size(3) * 4;
    void * st;
    if (!stream_of(v[14], q, st)) return nullptr;
    THPObjectPtr ws = workspace(v[0], st, lib.workspace_size(&a), a);
    if (!ws) return nullptr;
    const int rc = unlocked(a.workspace, [&] { return lib.attn(&a, st); });
    if (rc) return failed("mla_attn_launch", rc);
    if (made.defined()) return THPVariable_Wrap(made);
    Py_INCREF(v[10]);
    return v[10];
}

// The argument block of an op of a batch: kept as bytes by the batch until it is launched.
PyObject * add_to_batch(PyObject * batch, int kind, const void * args, size_t size, PyObject * result) {
    THPObjectPtr k(PyLong_FromLong(kind)), b(PyBytes_FromStringAndSize((const char *) args, (Py_ssize_t) size)), name(PyUnicode_InternFromString("add"));
    if (!k || !b || !name) return nullptr;
    THPObjectPtr r(PyObject_CallMethodObjArgs(batch, name.get(), k.get(), b.get(), nullptr));
    return r ? Py_NewRef(result) : nullptr;
}

// values: pos, n_dims, mode, n_ctx_orig, freq_base, freq_scale, ext_factor, attn_factor, beta_fast, beta_slow, freq_factors
constexpr int N_ROPE = 11;
PyObject * fill_rope(mla_rope_args & a, const at::Tensor & x, const at::Tensor & out, PyObject * const * v, int64_t n_pos) {
    const at::Tensor * pos = tensor(v[0]), * ff;
    if (!pos || !optional_tensor(v[10], ff)) return nullptr;
    a.n_dims = (int32_t) PyLong_AsLong(v[1]); a.mode = (int32_t) PyLong_AsLong(v[2]); a.n_ctx_orig = (int32_t) PyLong_AsLong(v[3]);
    a.freq_base = (float) PyFloat_AsDouble(v[4]); a.freq_scale = (float) PyFloat_AsDouble(v[5]); a.ext_factor = (float) PyFloat_AsDouble(v[6]);
    a.attn_factor = (float) PyFloat_AsDouble(v[7]); a.beta_fast = (float) PyFloat_AsDouble(v[8]); a.beta_slow = (float) PyFloat_AsDouble(v[9]);
    if (PyErr_Occurred()) return nullptr;
    REQUIRE(pos->scalar_type() == at::kInt && pos->is_contiguous() && pos->numel() == n_pos);
    int64_t ne_out[4];
    nb4(x, a.ne, a.src_nb);
    nb4(out, ne_out, a.dst_nb);
    a.src = x.data_ptr(); a.dst = out.data_ptr(); a.pos = (const int32_t *) pos->data_ptr();
    if (ff) {
        REQUIRE(ff->scalar_type() == at::kFloat && ff->is_contiguous() && ff->numel() >= a.n_dims / 2);
        a.freq_factors = (const float *) ff->data_ptr();
    }
    return Py_None;   // (borrowed: anything but nullptr)
}

// rope(x, out, stream, batch, *values) -> out
PyObject * rope(PyObject *, PyObject * const * v, Py_ssize_t n) {
    if (!arg_count(n, 4 + N_ROPE)) return nullptr;
    const at::Tensor * xp = tensor(v[0]), * outp;
    if (!xp || !optional_tensor(v[1], outp)) return nullptr;
    const at::Tensor & x = *xp;
    if (!on_gpu(x)) return nullptr;
    REQUIRE(x.scalar_type() == at::kFloat && x.dim() == 3 && x.stride(2) == 1);
    at::Tensor made;
    if (!outp) { made = at::empty(x.sizes(), x.options()); outp = &made; }
    const at::Tensor & out = *outp;
    REQUIRE(out.sizes() == x.sizes() && out.scalar_type() == at::kFloat && out.stride(2) == 1);
    mla_rope_args a;
    memset(&a, 0, sizeof a);
    if (!fill_rope(a, x, out, v + 4, x.size(0))) return nullptr;
    THPObjectPtr result(made.defined() ? THPVariable_Wrap(made) : Py_NewRef(v[1]));
    if (!result) return nullptr;
    if (v[3] != Py_None) return add_to_batch(v[3], MLA_FRONT_ROPE, &a, sizeof a, result.get());
    void * st;
    if (!stream_of(v[2], x, st)) return nullptr;
    const int rc = unlocked([&] { return lib.rope(&a, st); });
    if (rc) return failed("mla_rope_launch", rc);
    return result.release();
}

// mul_mat(w, w_type, x, out, stream, batch) -> out
PyObject * mul_mat(PyObject *, PyObject * const * v, Py_ssize_t n) {
    if (!arg_count(n, 6)) return nullptr;
    const at::Tensor * wp = tensor(v[0]), * xp = wp ? tensor(v[2]) : nullptr, * outp;
    if (!xp || !optional_tensor(v[3], outp)) return nullptr;
    const at::Tensor & w = *wp, & x = *xp;
    if (!on_gpu(x)) return nullptr;
    REQUIRE(w.dim() == 3 && x.dim() == 3 && w.element_size() == 2 && x.scalar_type() == at::kFloat);
    REQUIRE(w.stride(2) == 1 && x.stride(2) == 1 && w.size(2) == x.size(2));
    at::Tensor made;
    if (!outp) { made = at::empty({ x.size(0), x.size(1), w.size(1) }, x.options()); outp = &made; }
    const at::Tensor & out = *outp;
    REQUIRE(out.dim() == 3 && out.size(0) == x.size(0) && out.size(1) == x.size(1) && out.size(2) == w.size(1) && out.scalar_type() == at::kFloat && out.stride(2) == 1);
    mla_mul_mat_args a;
    memset(&a, 0, sizeof a);
    a.w_type = (int32_t) PyLong_AsLong(v[1]);
    if (PyErr_Occurred()) return nullptr;
    a.w = w.data_ptr(); a.x = x.data_ptr(); a.dst = out.data_ptr();
    a.K = w.size(2); a.N = w.size(1); a.w_ne2 = w.size(0); a.w_ne3 = 1;
    a.M = x.size(1); a.ne2 = x.size(0); a.ne3 = 1;
    a.w_nb1 = w.stride(1) * 2; a.w_nb2 = w.stride(0) * 2; a.w_nb3 = a.w_nb2 * a.w_ne2;
    a.x_nb1 = x.stride(1) * 4; a.x_nb2 = x.stride(0) * 4; a.x_nb3 = a.x_nb2 * a.ne2;
    a.d_nb1 = out.stride(1) * 4; a.d_nb2 = out.stride(0) * 4; a.d_nb3 = a.d_nb2 * a.ne2;
    THPObjectPtr result(made.defined() ? THPVariable_Wrap(made) : Py_NewRef(v[3]));
    if (!result) return nullptr;
    if (v[5] != Py_None) return add_to_batch(v[5], MLA_FRONT_MUL_MAT, &a, sizeof a, result.get());
    void * st;
    if (!stream_of(v[4], x, st)) return nullptr;
    const int rc = unlocked([&] { return lib.mul_mat(&a, st); });
    if (rc) return failed("mla_mul_mat_launch", rc);
    return result.release();
}

// copy(src, dst, stream, batch) -> dst
PyObject * copy(PyObject *, PyObject * const * v, Py_ssize_t n) {
    if (!arg_count(n, 4)) return nullptr;
    const at::Tensor * sp = tensor(v[0]), * dp = sp ? tensor(v[1]) : nullptr;
    if (!dp) return nullptr;
    const at::Tensor & src = *sp, & dst = *dp;
    if (!on_gpu(src)) return nullptr;
    REQUIRE(src.scalar_type() == at::kFloat && dst.scalar_type() == at::kFloat && src.sizes() == dst.sizes() && src.dim() >= 1 && src.dim() <= 4);
    REQUIRE(src.stride(-1) == 1 && dst.stride(-1) == 1);
    mla_copy_args a;
    memset(&a, 0, sizeof a);
    int64_t ne_dst[4];
    nb4(src, a.ne, a.src_nb);
    nb4(dst, ne_dst, a.dst_nb);
    a.src = src.data_ptr(); a.dst = dst.data_ptr();
    if (v[3] != Py_None) return add_to_batch(v[3], MLA_FRONT_COPY, &a, sizeof a, v[1]);
    void * st;
    if (!stream_of(v[2], src, st)) return nullptr;
    const int rc = unlocked([&] { return lib.copy(&a, st); });
    if (rc) return failed("mla_copy_f32_launch", rc);
    return Py_NewRef(v[1]);
}

// kv_write(src, cache, kv_type, row0, rows, block_table, seq_ids, positions, stream, batch, k_pe[, *rope values]) -> cache
PyObject * kv_write(PyObject *, PyObject * const * v, Py_ssize_t n) {
    if (n != 11 && !arg_count(n, 11 + N_ROPE)) return nullptr;
    const at::Tensor * sp = tensor(v[0]), * cp = sp ? tensor(v[1]) : nullptr, * rows, * table, * ids, * positions, * k_pe;
    if (!cp || !optional_tensor(v[4], rows) || !optional_tensor(v[5], table) || !optional_tensor(v[6], ids) || !optional_tensor(v[7], positions) || !optional_tensor(v[10], k_pe)) return nullptr;
    const at::Tensor & src = *sp, & cache = *cp;
    if (!on_gpu(src)) return nullptr;
    const bool with_rope = k_pe != nullptr;
    REQUIRE(with_rope == (n > 11));
    mla_kv_write_rope_args ra;
    memset(&ra, 0, sizeof ra);
    mla_kv_write_args & a = ra.w;
    REQUIRE(src.dim() == 2 && src.stride(1) == 1 && cache.dim() == 2 && cache.stride(1) == 1);
    if (with_rope) {
        REQUIRE(k_pe->scalar_type() == at::kFloat && k_pe->dim() == 2 && k_pe->size(0) == src.size(0) && k_pe->size(1) == 64 && k_pe->stride(1) == 1);
        if (!fill_rope(ra.rope, *k_pe, *k_pe, v + 11, src.size(0))) return nullptr;
        // [tokens, 64] is [tokens, 1 head, 64]
        ra.rope.ne[2] = ra.rope.ne[1]; ra.rope.ne[1] = 1;
        ra.rope.src_nb[2] = ra.rope.dst_nb[2] = ra.rope.src_nb[1];
        ra.rope.src_nb[3] = ra.rope.dst_nb[3] = ra.rope.src_nb[2] * ra.rope.ne[2];
    }
    a.n_tok = (int32_t) src.size(0);
    a.kv_type = (int32_t) PyLong_AsLong(v[2]);
    if (PyErr_Occurred()) return nullptr;
    const int64_t row = row_bytes(a.kv_type);
    if (row < 0) { PyErr_SetObject(PyExc_KeyError, v[2]); return nullptr; }
    const bool f32 = src.scalar_type() == at::kFloat;
    a.src_type = f32 ? MLA_TYPE_F32 : a.kv_type;
    REQUIRE(cache.size(1) * (int64_t) cache.element_size() == row);
    if (f32) REQUIRE(src.size(1) == 576 || (with_rope && src.size(1) >= 512));
    else     REQUIRE(src.size(1) * (int64_t) src.element_size() == row);
    a.src = src.data_ptr(); a.src_nb1 = src.stride(0) * (int64_t) src.element_size();
    a.kv = cache.data_ptr(); a.kv_nb1 = cache.stride(0) * (int64_t) cache.element_size(); a.n_kv_rows = cache.size(0);
    REQUIRE((v[3] != Py_None) + (rows != nullptr) + (table != nullptr) == 1);
    if (v[3] != Py_None) {
        a.row0 = PyLong_AsLongLong(v[3]);
        if (PyErr_Occurred()) return nullptr;
    } else if (rows) {
        REQUIRE((rows->scalar_type() == at::kInt || rows->scalar_type() == at::kLong) && rows->is_contiguous() && rows->numel() == a.n_tok);
        a.rows = rows->data_ptr(); a.rows_type = rows->scalar_type() == at::kLong ? 1 : 0;
    } else {
        REQUIRE(ids && positions);
        for (const at::Tensor * t : { table, ids, positions }) REQUIRE(t->scalar_type() == at::kInt && t->is_contiguous());
        REQUIRE(table->dim() == 2 && ids->numel() == a.n_tok && positions->numel() == a.n_tok);
        a.block_table = (const int32_t *) table->data_ptr(); a.bt_stride = table->size(1);
        a.seq_ids = (const int32_t *) ids->data_ptr(); a.positions = (const int32_t *) positions->data_ptr();
    }
    if (v[9] != Py_None) return with_rope ? add_to_batch(v[9], MLA_FRONT_KV_WRITE_ROPE, &ra, sizeof ra, v[1]) : add_to_batch(v[9], MLA_FRONT_KV_WRITE, &a, sizeof a, v[1]);
    void * st;
    if (!stream_of(v[8], src, st)) return nullptr;
    const int rc = unlocked([&] { return with_rope ? lib.kv_write_rope(&ra, st) : lib.kv_write(&a, st); });
    if (rc) return failed(with_rope ? "mla_kv_write_rope_launch" : "mla_kv_write_launch", rc);
    return Py_NewRef(v[1]);
}

struct Buffers {
    std::vector<Py_buffer> held;
    ~Buffers() { for (Py_buffer & b : held) PyBuffer_Release(&b); }
};

// front_batch(ops, stream): ops = [(kind, argument block: bytes or anything with a buffer), ...]
PyObject * front_batch(PyObject *, PyObject * const * v, Py_ssize_t n) {
    if (!arg_count(n, 2)) return nullptr;
    REQUIRE(PyList_Check(v[0]));
    const Py_ssize_t count = PyList_GET_SIZE(v[0]);
    std::vector<mla_front_op> ops((size_t) std::max<Py_ssize_t>(count, 1));
    Buffers b;
    b.held.reserve((size_t) count);
    for (Py_ssize_t i = 0; i < count; i++) {
        PyObject * op = PyList_GET_ITEM(v[0], i);
        Py_buffer  buf;
        if (!PyTuple_Check(op) || PyTuple_GET_SIZE(op) != 2) {
            PyErr_SetString(PyExc_TypeError, "front_batch: ops are (kind, argument block) pairs");
            return nullptr;
        }
        if (PyObject_GetBuffer(PyTuple_GET_ITEM(op, 1), &buf, PyBUF_SIMPLE) != 0) return nullptr;
        b.held.push_back(buf);
        ops[(size_t) i] = mla_front_op{ (int32_t) PyLong_AsLong(PyTuple_GET_ITEM(op, 0)), 0, buf.buf };
        if (PyErr_Occurred()) return nullptr;
    }
    void * st = PyLong_AsVoidPtr(v[1]);
    if (PyErr_Occurred()) return nullptr;
    const int rc = unlocked([&] { return lib.front_batch(ops.data(), (int32_t) count, st); });
    if (rc) return failed("mla_front_batch_launch", rc);
    Py_RETURN_NONE;
}

// ---- the cache of ordinary heads (include/gqa_attn.h)

bool int_of(PyObject * o, int32_t & v) {                      // (a number past 32 bits is an error, not its low half)
    const long x = PyLong_AsLong(o);
    v = (int32_t) x;
    if (!PyErr_Occurred() && x != v) PyErr_SetString(PyExc_OverflowError, "an integer argument does not fit 32 bits");
    return !PyErr_Occurred();
}
constexpr int64_t INTS = (int64_t) 1 << 31;                   // sizes below
int mla_type(const at::Tensor & t) {
    switch (t.scalar_type()) {
        case at::kFloat:    return MLA_TYPE_F32;
        case at::kHalf:     return MLA_TYPE_F16;
        case at::kBFloat16: return MLA_TYPE_BF16;
        default:            return -1;
    }
}
at::ScalarType torch_type(int type) { return type == MLA_TYPE_F32 ? at::kFloat : type == MLA_TYPE_F16 ? at::kHalf : at::kBFloat16; }
bool ints(const at::Tensor & t, int64_t n) { return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous(); }
bool table_ok(const at::Tensor & t) { return t.scalar_type() == at::kInt && t.dim() == 2 && t.is_contiguous() && t.size(1) >= 1; }
// `dim` dimensions, the last one contiguous; the elements of a tensor that is written must not lie on each other: from the smallest
// stride up, each steps past all that the ones before it reach.
bool rows_ok(const at::Tensor & t, int64_t dim, bool written) {
    if (t.dim() != dim || (t.size(-1) > 1 && t.stride(-1) != 1)) return false;
    if (!written || t.numel() == 0) return true;
    std::pair<int64_t, int64_t> steps[4];                     // (dim <= 4)
    int n = 0;
    for (int64_t d = 0; d < dim; d++) if (t.size(d) > 1) steps[n++] = { t.stride(d), t.size(d) };
    std::sort(steps, steps + n);
    int64_t reach = 0;
    for (int i = 0; i < n; i++) {
        if (steps[i].first <= reach) return false;
        reach += steps[i].first * (steps[i].second - 1);
    }
    return true;
}
bool cache_ok(const at::Tensor & c, int type) { return mla_type(c) == type && rows_ok(c, 4, true) && c.size(0) >= 1 && c.size(1) == PAGE; }
// Bytes from one to the next along a dimension; where there is no next one a stride may be anything, and is none.
int64_t step(const at::Tensor & t, int64_t d) { return t.size(d) > 1 ? t.stride(d) * (int64_t) t.element_size() : 0; }
gqa_pool pool_of(const at::Tensor & c) { return gqa_pool{ c.data_ptr(), step(c, 0), step(c, 1), step(c, 2) }; }
// The stream to launch on.  The result tensors a call makes for itself belong to the device's current stream, so a call on another one
// brings its own (`makes` = false).
struct GqaStream {
    void * st;
    bool   current;
    bool take(PyObject * o, const at::Tensor & t, bool makes) {
        if (!stream_of(Py_None, t, st)) return false;
        current = true;
        if (o == Py_None) return true;
        void * const now = st;
        if (!stream_of(o, t, st)) return false;
        current = st == now;
        if (!makes || current) return true;
        PyErr_SetString(PyExc_ValueError, "a launch on another stream than the current one takes its result tensors from the caller");
        return false;
    }
};
// Scratch of a launch, the launch's stream's own.  Under graph capture it is the graph's: two graphs captured on one stream may be replayed side by side.
struct GqaScratch {
    THPObjectPtr ws;
    at::Tensor   own;
    template <typename Args> bool take(PyObject * o, const at::Tensor & t, const GqaStream & s, size_t need, Args & a) {
        if (!need) return true;
        if (!s.current) {
            THPObjectPtr dev(PyObject_GetAttrString(o, "device")), n(PyLong_FromSize_t(need)), handle(PyLong_FromVoidPtr(s.st));
            if (!dev || !n || !handle) return false;
            ws = THPObjectPtr(PyObject_CallFunctionObjArgs(lib.elsewhere, dev.get(), n.get(), handle.get(), nullptr));
            if (!ws) return false;
            if (!THPVariable_Check(ws.get())) { PyErr_SetString(PyExc_TypeError, "expected a torch tensor"); return false; }
            const at::Tensor & w = THPVariable_Unpack(ws.get());
            a.workspace = w.data_ptr(); a.workspace_size = (size_t) w.numel();
            return true;
        }
        THPObjectPtr capturing(PyObject_CallNoArgs(lib.capturing));
        if (!capturing) return false;
        if (capturing.get() == Py_True) {
            own = at::empty({ (int64_t) need }, t.options().dtype(at::kByte));
            a.workspace = own.data_ptr(); a.workspace_size = need;
            return true;
        }
        ws = workspace(o, s.st, need, a);
        return (bool) ws;
    }
};
// What a call writes has to lie apart from what it reads and from what else it writes, but for the one tensor it may work on in place; views of one buffer that
// share no byte are apart.  Layouts too tangled to tell are let through.  (Most tensors lie in memory of their own: their ranges are taken once and compared first.)
class Apart {
    struct Item { const char * name; const at::Tensor * t; uintptr_t lo, hi; };
    Item items[16];
    int  n = 0;

  public:
    // a tensor or nullptr; those that are written come first
    void add(const char * name, const at::Tensor * t) {
        if (!t) return;
        const auto sizes = t->sizes(), strides = t->strides();
        int64_t span = 1;
        for (size_t d = 0; d < sizes.size(); d++) {
            if (sizes[d] == 0) return;
            span += (sizes[d] - 1) * strides[d];
        }
        const uintptr_t lo = (uintptr_t) t->data_ptr();
        items[n++] = Item{ name, t, lo, lo + (uintptr_t) (span * (int64_t) t->element_size()) };
    }
    int count() const { return n; }
    // items 0 .. written - 1 against all that follow them
    bool check(const char * call, int written, const at::Tensor * in_place_on = nullptr) const {
        for (int i = 0; i < written; i++)
            for (int k = i + 1; k < n; k++) {
                const Item & a = items[i], & b = items[k];
                if (a.lo >= b.hi || b.lo >= a.hi) continue;
                if (i == 0 && b.t == in_place_on && a.lo == b.lo) continue;            // (its strides and type are the launch's to check)
                auto extent = [](const Item & x) { return mla::Extent((const void *) x.lo, (int64_t) x.t->element_size(), (int) x.t->dim(), x.t->sizes().data(), x.t->strides().data()); };
                if (mla::shares(extent(a), extent(b)) != mla::Shares::YES) continue;
                PyErr_Format(PyExc_RuntimeError, "%s: %s and %s share memory", call, a.name, b.name);
                return false;
            }
        return true;
    }
};
#define SAME_DEVICE(t) REQUIRE(!(t) || (t)->device() == q.device())

// gqa_norm_rope(q, k, v, pos, q_weight, k_weight, eps, n_dims, mode, n_ctx_orig, freq_base, freq_scale, ext_factor, attn_factor, beta_fast,
//               beta_slow, freq_factors, q_out, k_cache, v_cache, block_table, seq_ids, slots, stream) -> q_out
PyObject * gqa_norm_rope(PyObject *, PyObject * const * o, Py_ssize_t n) {
    if (!arg_count(n, 24)) return nullptr;
    const at::Tensor * qp = tensor(o[0]), * pos = qp ? tensor(o[3]) : nullptr, * k, * v, * qw, * kw, * ff, * outp, * kc, * vc, * table, * ids, * slots;
    if (!pos || !optional_tensor(o[1], k) || !optional_tensor(o[2], v) || !optional_tensor(o[4], qw) || !optional_tensor(o[5], kw) || !optional_tensor(o[16], ff) ||
        !optional_tensor(o[17], outp) || !optional_tensor(o[18], kc) || !optional_tensor(o[19], vc) || !optional_tensor(o[20], table) || !optional_tensor(o[21], ids) || !optional_tensor(o[22], slots))
        return nullptr;
    const at::Tensor & q = *qp;
    if (!on_gpu(q)) return nullptr;
    for (const at::Tensor * t : { pos, k, v, qw, kw, ff, outp, kc, vc, table, ids, slots }) SAME_DEVICE(t);
    gqa_norm_rope_args a;
    memset(&a, 0, sizeof a);
    a.eps = (float) PyFloat_AsDouble(o[6]);
    if (PyErr_Occurred() || !int_of(o[7], a.n_dims) || !int_of(o[8], a.mode) || !int_of(o[9], a.n_ctx_orig)) return nullptr;
    a.freq_base = PyFloat_AsDouble(o[10]); a.freq_scale = PyFloat_AsDouble(o[11]); a.ext_factor = PyFloat_AsDouble(o[12]);
    a.attn_factor = PyFloat_AsDouble(o[13]); a.beta_fast = PyFloat_AsDouble(o[14]); a.beta_slow = PyFloat_AsDouble(o[15]);
    if (PyErr_Occurred()) return nullptr;
    REQUIRE(mla_type(q) >= 0 && rows_ok(q, 3, false) && q.size(0) < INTS && q.size(1) < INTS && q.size(2) < INTS);
    const int64_t n_tok = q.size(0);
    a.n_tok = (int32_t) n_tok; a.n_head = (int32_t) q.size(1); a.dk = (int32_t) q.size(2);
    a.src_type = a.w_type = mla_type(q);
    a.q = q.data_ptr(); a.q_nb1 = step(q, 1); a.q_nb2 = step(q, 0);
    REQUIRE(ints(*pos, n_tok));
    a.pos = (const int32_t *) pos->data_ptr();
    a.kv_type = MLA_TYPE_BF16;
    if (qw || kw) {
        a.w_type = mla_type(qw ? *qw : *kw);
        for (const at::Tensor * w : { qw, kw }) REQUIRE(!w || (mla_type(*w) == a.w_type && a.w_type >= 0 && w->dim() == 1 && w->size(0) == a.dk && w->is_contiguous()));
        a.q_weight = qw ? qw->data_ptr() : nullptr; a.k_weight = kw ? kw->data_ptr() : nullptr;
    }
    if (ff) {
        REQUIRE(ff->scalar_type() == at::kFloat && ff->dim() == 1 && ff->size(0) >= a.n_dims / 2 && ff->is_contiguous());
        a.freq_factors = (const float *) ff->data_ptr();
    }
    if (k) {
        REQUIRE(kc && table && ids && (v != nullptr) == (vc != nullptr));
        REQUIRE(k->scalar_type() == q.scalar_type() && rows_ok(*k, 3, false) && k->size(0) == n_tok && k->size(2) == a.dk);
        a.kv_type = mla_type(*kc);
        REQUIRE(a.kv_type > 0 && cache_ok(*kc, a.kv_type) && kc->size(2) == k->size(1) && kc->size(2) < INTS && kc->size(3) == a.dk);
        REQUIRE(table_ok(*table) && table->size(0) < INTS && ints(*ids, n_tok) && (!slots || ints(*slots, n_tok)));
        a.n_head_kv = (int32_t) k->size(1); a.n_seq = (int32_t) table->size(0); a.n_pages = kc->size(0);
        a.k = k->data_ptr(); a.k_nb1 = step(*k, 1); a.k_nb2 = step(*k, 0);
        a.k_cache = pool_of(*kc);
        a.block_table = (const int32_t *) table->data_ptr(); a.bt_stride = table->size(1);
        a.seq_ids = (const int32_t *) ids->data_ptr(); a.slots = slots ? (const int32_t *) slots->data_ptr() : nullptr;
        if (v) {
            REQUIRE(v->scalar_type() == q.scalar_type() && rows_ok(*v, 3, false) && v->size(0) == n_tok && v->size(1) == a.n_head_kv);
            REQUIRE(cache_ok(*vc, a.kv_type) && vc->size(0) == a.n_pages && vc->size(2) == a.n_head_kv && vc->size(3) == v->size(2) && v->size(2) < INTS);
            a.dv = (int32_t) v->size(2);
            a.v = v->data_ptr(); a.v_nb1 = step(*v, 1); a.v_nb2 = step(*v, 0);
            a.v_cache = pool_of(*vc);
        }
    } else REQUIRE(!v && !kc && !vc && !kw);
    const c10::DeviceGuard guard(q.device());
    GqaStream stream;
    if (!stream.take(o[23], q, !outp)) return nullptr;
    at::Tensor made;
    if (!outp) { made = at::empty(q.sizes(), q.options().dtype(kc ? kc->scalar_type() : q.scalar_type())); outp = &made; }
    const at::Tensor & out = *outp;
    a.dst_type = mla_type(out);
    REQUIRE(a.dst_type >= 0 && out.sizes() == q.sizes() && rows_ok(out, 3, true));
    a.q_dst = out.data_ptr(); a.qd_nb1 = step(out, 1); a.qd_nb2 = step(out, 0);
    Apart apart;                                              // (keys and values may lie in the cache, where the caller knows the rows)
    if (!made.defined()) {
        Apart result;
        result.add("q_out", &out);
        for (const auto & [name, t] : { std::pair<const char *, const at::Tensor *>{ "q", &q }, { "k", k }, { "v", v }, { "pos", pos }, { "q_weight", qw }, { "k_weight", kw }, { "freq_factors", ff },
                                        { "k_cache", kc }, { "v_cache", vc }, { "block_table", table }, { "seq_ids", ids }, { "slots", slots } })
            result.add(name, t);
        if (n_tok && !result.check("gqa_norm_rope", 1, &q)) return nullptr;
    }
    apart.add("k_cache", kc); apart.add("v_cache", vc); apart.add("q", &q);
    if (!apart.check("gqa_norm_rope", apart.count() - 1)) return nullptr;
    const int rc = unlocked([&] { return lib.norm_rope(&a, stream.st); });
    if (rc) return failed("gqa_norm_rope_launch", rc);
    return made.defined() ? THPVariable_Wrap(made) : Py_NewRef(o[17]);
}

// gqa_attn(q, k_cache, v_cache, block_table, seq_lens, scale, logit_softcap, window, mask, weights, out, n_workgroups, stream) -> out, or weights without v_cache
PyObject * gqa_attn(PyObject *, PyObject * const * o, Py_ssize_t n) {
    if (!arg_count(n, 13)) return nullptr;
    const at::Tensor * qp = tensor(o[0]), * kc = qp ? tensor(o[1]) : nullptr, * table = kc ? tensor(o[3]) : nullptr, * lens = table ? tensor(o[4]) : nullptr, * vc, * mask, * weights, * outp;
    if (!lens || !optional_tensor(o[2], vc) || !optional_tensor(o[8], mask) || !optional_tensor(o[9], weights) || !optional_tensor(o[10], outp)) return nullptr;
    const at::Tensor & q = *qp;
    if (!on_gpu(q)) return nullptr;
    for (const at::Tensor * t : { kc, table, lens, vc, mask, weights, outp }) SAME_DEVICE(t);
    gqa_attn_args a;
    memset(&a, 0, sizeof a);
    a.scale = (float) PyFloat_AsDouble(o[5]); a.logit_softcap = (float) PyFloat_AsDouble(o[6]);
    const int64_t window = PyLong_AsLongLong(o[7]);
    if (PyErr_Occurred() || !int_of(o[11], a.n_workgroups)) return nullptr;
    REQUIRE(window >= 0 && window < INTS);
    a.window = (int32_t) window;
    REQUIRE(mla_type(q) >= 0 && rows_ok(q, 3, false) && q.size(0) < INTS && q.size(1) < INTS && q.size(2) < INTS);
    const int64_t n_seq = q.size(0), n_head = q.size(1);
    a.n_seq = (int32_t) n_seq; a.n_head = (int32_t) n_head; a.dk = (int32_t) q.size(2);
    a.q_type = mla_type(q); a.q = q.data_ptr(); a.q_nb1 = step(q, 1); a.q_nb2 = step(q, 0);
    a.kv_type = mla_type(*kc);
    REQUIRE(a.kv_type > 0 && cache_ok(*kc, a.kv_type) && kc->size(2) < INTS && kc->size(3) == a.dk);
    a.n_head_kv = (int32_t) kc->size(2); a.n_pages = kc->size(0); a.k = pool_of(*kc);
    if (vc) {
        REQUIRE(cache_ok(*vc, a.kv_type) && vc->size(0) == a.n_pages && vc->size(2) == a.n_head_kv && vc->size(3) < INTS);
        a.dv = (int32_t) vc->size(3); a.v = pool_of(*vc);
    } else REQUIRE(weights && !outp);
    REQUIRE(table_ok(*table) && table->size(0) == n_seq && ints(*lens, n_seq));
    a.block_table = (const int32_t *) table->data_ptr(); a.bt_stride = table->size(1); a.seq_lens = (const int32_t *) lens->data_ptr();
    if (mask) {
        REQUIRE(mask->scalar_type() == at::kHalf && rows_ok(*mask, 2, false) && mask->size(0) == n_seq);
        a.mask = mask->data_ptr(); a.mask_nb1 = mask->stride(0) * 2; a.mask_ne0 = mask->size(1);
        if (!a.mask && n_seq) { PyErr_SetString(PyExc_ValueError, "a mask without columns leaves no row"); return nullptr; }
    }
    if (weights) {
        REQUIRE(weights->scalar_type() == at::kFloat && rows_ok(*weights, 3, true) && weights->size(0) == n_seq && weights->size(1) == a.n_head_kv && weights->size(2) >= a.bt_stride * PAGE);
        a.weights = (float *) weights->data_ptr(); a.w_nb1 = step(*weights, 1); a.w_nb2 = step(*weights, 0);
    }
    const c10::DeviceGuard guard(q.device());
    GqaStream stream;
    if (!stream.take(o[12], q, vc && !outp)) return nullptr;
    at::Tensor made;
    if (vc) {
        if (!outp) { made = at::empty({ n_seq, n_head, (int64_t) a.dv }, q.options()); outp = &made; }
        const at::Tensor & out = *outp;
        a.dst_type = mla_type(out);
        REQUIRE(a.dst_type >= 0 && out.dim() == 3 && out.size(0) == n_seq && out.size(1) == n_head && out.size(2) == a.dv && rows_ok(out, 3, true));
        a.dst = out.data_ptr(); a.d_nb1 = step(out, 1); a.d_nb2 = step(out, 0);
    } else a.dst_type = MLA_TYPE_F32;
    Apart apart;
    if (!made.defined()) apart.add("out", outp);
    apart.add("weights", weights);
    const int written = apart.count();
    apart.add("q", &q); apart.add("k_cache", kc); apart.add("v_cache", vc); apart.add("block_table", table); apart.add("seq_lens", lens); apart.add("mask", mask);
    if (!apart.check("gqa_attn", written)) return nullptr;
    const size_t need = lib.gqa_workspace_size(&a);
    GqaScratch scratch;
    if (!scratch.take(o[0], q, stream, need, a)) return nullptr;
    const int rc = unlocked(a.workspace, [&] { return lib.gqa_attn(&a, stream.st); });
    if (rc) return failed("gqa_attn_launch", rc);
    return made.defined() ? THPVariable_Wrap(made) : Py_NewRef(vc ? o[10] : o[9]);
}

// gqa_evict(weights, block_table, seq_lens, k_cache, v_cache, n_keep, n_sink, n_recent, weights_out, kept, new_lens, stream) -> (kept, new_lens, weights_out)
PyObject * gqa_evict(PyObject *, PyObject * const * o, Py_ssize_t n) {
    if (!arg_count(n, 12)) return nullptr;
    const at::Tensor * qp = tensor(o[0]), * table = qp ? tensor(o[1]) : nullptr, * lens = table ? tensor(o[2]) : nullptr, * kc = lens ? tensor(o[3]) : nullptr, * vc, * wop, * keptp, * newp;
    if (!kc || !optional_tensor(o[4], vc) || !optional_tensor(o[8], wop) || !optional_tensor(o[9], keptp) || !optional_tensor(o[10], newp)) return nullptr;
    const at::Tensor & q = *qp;                               // the weights
    if (!on_gpu(q)) return nullptr;
    for (const at::Tensor * t : { table, lens, kc, vc, wop, keptp, newp }) SAME_DEVICE(t);
    gqa_evict_args a;
    memset(&a, 0, sizeof a);
    if (!int_of(o[5], a.n_keep) || !int_of(o[6], a.n_sink) || !int_of(o[7], a.n_recent)) return nullptr;
    REQUIRE(table_ok(*table));
    const int64_t n_seq = table->size(0), cap = table->size(1) * PAGE;
    REQUIRE(ints(*lens, n_seq));
    a.n_seq = (int32_t) n_seq;
    a.block_table = (const int32_t *) table->data_ptr(); a.bt_stride = table->size(1); a.seq_lens = (const int32_t *) lens->data_ptr();
    REQUIRE(n_seq < INTS && rows_ok(*kc, 4, true) && kc->size(0) >= 1 && kc->size(1) == PAGE && kc->size(2) < INTS && kc->size(3) < INTS / 16);
    a.n_head_kv = (int32_t) kc->size(2); a.n_pages = kc->size(0); a.k = pool_of(*kc);
    a.k_row_bytes = (int32_t) (kc->size(3) * (int64_t) kc->element_size());
    if (vc) {
        REQUIRE(rows_ok(*vc, 4, true) && vc->size(0) == a.n_pages && vc->size(1) == PAGE && vc->size(2) == a.n_head_kv && vc->size(3) < INTS / 16);
        a.v = pool_of(*vc); a.v_row_bytes = (int32_t) (vc->size(3) * (int64_t) vc->element_size());
    }
    REQUIRE(q.scalar_type() == at::kFloat && rows_ok(q, 3, false) && q.size(0) == n_seq && q.size(1) == a.n_head_kv && q.size(2) >= cap);
    a.weights = (const float *) q.data_ptr(); a.w_nb1 = step(q, 1); a.w_nb2 = step(q, 0);
    const c10::DeviceGuard guard(q.device());
    GqaStream stream;
    if (!stream.take(o[11], q, !wop || !keptp || !newp)) return nullptr;
    at::Tensor wo = wop ? *wop : at::empty({ n_seq, (int64_t) a.n_head_kv, cap }, q.options());
    REQUIRE(a.n_keep >= 0);
    at::Tensor kept = keptp ? *keptp : at::empty({ n_seq, (int64_t) a.n_head_kv, (int64_t) a.n_keep }, q.options().dtype(at::kInt));
    at::Tensor fresh = newp ? *newp : at::empty({ n_seq }, q.options().dtype(at::kInt));
    REQUIRE(wo.scalar_type() == at::kFloat && rows_ok(wo, 3, true) && wo.size(0) == n_seq && wo.size(1) == a.n_head_kv && wo.size(2) >= cap);
    REQUIRE(kept.scalar_type() == at::kInt && kept.dim() == 3 && kept.is_contiguous() && kept.size(0) == n_seq && kept.size(1) == a.n_head_kv && kept.size(2) == a.n_keep);
    REQUIRE(ints(fresh, n_seq));
    a.weights_dst = (float *) wo.data_ptr(); a.wd_nb1 = step(wo, 1); a.wd_nb2 = step(wo, 0);
    a.kept = (int32_t *) kept.data_ptr(); a.new_lens = (int32_t *) fresh.data_ptr();
    Apart apart;
    apart.add("weights_out", wop); apart.add("kept", keptp); apart.add("new_lens", newp); apart.add("k_cache", kc); apart.add("v_cache", vc);
    const int written = apart.count();
    apart.add("weights", &q); apart.add("block_table", table); apart.add("seq_lens", lens);
    if (!apart.check("gqa_evict", written, wop ? &q : nullptr)) return nullptr;
    GqaScratch scratch;
    if (!scratch.take(o[0], q, stream, lib.evict_workspace_size(&a), a)) return nullptr;
    const int rc = unlocked(a.workspace, [&] { return lib.evict(&a, stream.st); });
    if (rc) return failed("gqa_evict_launch", rc);
    THPObjectPtr r0(keptp ? Py_NewRef(o[9]) : THPVariable_Wrap(kept)), r1(newp ? Py_NewRef(o[10]) : THPVariable_Wrap(fresh)), r2(wop ? Py_NewRef(o[8]) : THPVariable_Wrap(wo));
    return r0 && r1 && r2 ? PyTuple_Pack(3, r0.get(), r1.get(), r2.get()) : nullptr;
}

// ---- attention of many query rows over the same keys (include/gqa_batch.h)

// Sequences' first tokens, or none and as many tokens each: q_starts int32 [n_seq + 1].
template <typename Args> bool queries(Args & a, const at::Tensor & q, const at::Tensor * starts, int64_t n_seq) {
    if (mla_type(q) <= 0 || !rows_ok(q, 3, false) || q.size(0) >= INTS || q.size(1) >= INTS || q.size(2) >= INTS || n_seq >= INTS) return false;
    a.n_tok = (int32_t) q.size(0); a.n_seq = (int32_t) n_seq; a.n_head = (int32_t) q.size(1); a.dk = (int32_t) q.size(2);
    a.type = mla_type(q); a.q = q.data_ptr(); a.q_nb1 = step(q, 1); a.q_nb2 = step(q, 0);
    if (!starts) return n_seq ? q.size(0) % n_seq == 0 : q.size(0) == 0;
    a.q_starts = (const int32_t *) starts->data_ptr();
    return ints(*starts, n_seq + 1);
}
// mask f16 [n_seq, n]
template <typename Args> bool row_mask(Args & a, const at::Tensor * mask, int64_t n_seq) {
    if (!mask) return true;
    if (mask->scalar_type() != at::kHalf || !rows_ok(*mask, 2, false) || mask->size(0) != n_seq) return false;
    a.mask = mask->data_ptr(); a.mask_nb1 = step(*mask, 0); a.mask_ne0 = mask->size(1);
    return a.mask || !n_seq;
}
// The result: the caller's or a new tensor, [rows of q, heads, dv].
struct Result {
    at::Tensor made;
    const at::Tensor * t;
    template <typename Args> bool take(Args & a, const at::Tensor & q, const at::Tensor * given) {
        t = given;
        if (!t) { made = at::empty({ q.size(0), q.size(1), (int64_t) a.dv }, q.options()); t = &made; }
        if (t->scalar_type() != q.scalar_type() || t->dim() != 3 || t->size(0) != q.size(0) || t->size(1) != q.size(1) || t->size(2) != a.dv || !rows_ok(*t, 3, true)) return false;
        a.dst = t->data_ptr(); a.d_nb1 = step(*t, 1); a.d_nb2 = step(*t, 0);
        return true;
    }
    PyObject * give(PyObject * given) const { return made.defined() ? THPVariable_Wrap(made) : Py_NewRef(given); }
};

// gqa_prompt_attn(q, k_cache, v_cache, block_table, seq_lens, q_starts, scale, logit_softcap, window, causal, mask, out, n_workgroups, stream) -> out
PyObject * gqa_prompt_attn(PyObject *, PyObject * const * o, Py_ssize_t n) {
    if (!arg_count(n, 14)) return nullptr;
    const at::Tensor * qp = tensor(o[0]), * kc = qp ? tensor(o[1]) : nullptr, * vc = kc ? tensor(o[2]) : nullptr, * table = vc ? tensor(o[3]) : nullptr, * lens = table ? tensor(o[4]) : nullptr;
    const at::Tensor * starts, * mask, * outp;
    if (!lens || !optional_tensor(o[5], starts) || !optional_tensor(o[10], mask) || !optional_tensor(o[11], outp)) return nullptr;
    const at::Tensor & q = *qp;
    if (!on_gpu(q)) return nullptr;
    for (const at::Tensor * t : { kc, vc, table, lens, starts, mask, outp }) SAME_DEVICE(t);
    gqa_prompt_attn_args a;
    memset(&a, 0, sizeof a);
    a.scale = (float) PyFloat_AsDouble(o[6]); a.logit_softcap = (float) PyFloat_AsDouble(o[7]);
    const int64_t window = PyLong_AsLongLong(o[8]);
    a.causal = PyObject_IsTrue(o[9]);
    if (PyErr_Occurred() || !int_of(o[12], a.n_workgroups)) return nullptr;
    REQUIRE(window >= 0 && window < INTS);
    a.window = (int32_t) window;
    REQUIRE(table_ok(*table) && ints(*lens, table->size(0)));
    const int64_t n_seq = table->size(0);
    REQUIRE(queries(a, q, starts, n_seq));
    REQUIRE(cache_ok(*kc, a.type) && kc->size(2) < INTS && kc->size(3) == a.dk);
    REQUIRE(cache_ok(*vc, a.type) && vc->size(0) == kc->size(0) && vc->size(2) == kc->size(2) && vc->size(3) < INTS);
    a.n_head_kv = (int32_t) kc->size(2); a.n_pages = kc->size(0); a.dv = (int32_t) vc->size(3);
    a.k = pool_of(*kc); a.v = pool_of(*vc);
    a.block_table = (const int32_t *) table->data_ptr(); a.bt_stride = table->size(1); a.seq_lens = (const int32_t *) lens->data_ptr();
    REQUIRE(row_mask(a, mask, n_seq));
    const c10::DeviceGuard guard(q.device());
    GqaStream stream;
    if (!stream.take(o[13], q, !outp)) return nullptr;
    Result result;
    REQUIRE(result.take(a, q, outp));
    Apart apart;
    if (outp) {
        apart.add("out", outp);
        apart.add("q", &q); apart.add("k_cache", kc); apart.add("v_cache", vc); apart.add("block_table", table); apart.add("seq_lens", lens); apart.add("q_starts", starts); apart.add("mask", mask);
        if (a.n_tok && !apart.check("gqa_prompt_attn", 1)) return nullptr;
    }
    GqaScratch scratch;
    if (!scratch.take(o[0], q, stream, lib.prompt_workspace_size(&a), a)) return nullptr;
    const int rc = unlocked(a.workspace, [&] { return lib.prompt_attn(&a, stream.st); });
    return rc ? failed("gqa_prompt_attn_launch", rc) : result.give(o[11]);
}

// gqa_cross_attn(q, k, v, q_starts, kv_starts, kv_lens, scale, logit_softcap, mask, out, n_workgroups, stream) -> out
PyObject * gqa_cross_attn(PyObject *, PyObject * const * o, Py_ssize_t n) {
    if (!arg_count(n, 12)) return nullptr;
    const at::Tensor * qp = tensor(o[0]), * k = qp ? tensor(o[1]) : nullptr, * v = k ? tensor(o[2]) : nullptr, * starts, * kv_starts, * kv_lens, * mask, * outp;
    if (!v || !optional_tensor(o[3], starts) || !optional_tensor(o[4], kv_starts) || !optional_tensor(o[5], kv_lens) || !optional_tensor(o[8], mask) || !optional_tensor(o[9], outp)) return nullptr;
    const at::Tensor & q = *qp;
    if (!on_gpu(q)) return nullptr;
    for (const at::Tensor * t : { k, v, starts, kv_starts, kv_lens, mask, outp }) SAME_DEVICE(t);
    gqa_cross_attn_args a;
    memset(&a, 0, sizeof a);
    a.scale = (float) PyFloat_AsDouble(o[6]); a.logit_softcap = (float) PyFloat_AsDouble(o[7]);
    if (PyErr_Occurred() || !int_of(o[10], a.n_workgroups)) return nullptr;
    // [n_seq, n, heads, width] padded, or [n, heads, width] with the sequences' first rows
    const bool packed = kv_starts != nullptr;
    const int64_t d = packed ? 3 : 4;
    for (const at::Tensor * t : { k, v }) REQUIRE(mla_type(*t) == mla_type(q) && rows_ok(*t, d, false) && t->size(d - 3) < INTS && t->size(d - 2) < INTS && t->size(d - 1) < INTS);
    const int64_t n_seq = !packed ? k->size(0) : kv_lens ? kv_lens->numel() : kv_starts->numel() - 1;
    REQUIRE(n_seq >= 0 && queries(a, q, starts, n_seq));
    REQUIRE(k->size(d - 1) == a.dk && v->size(d - 2) == k->size(d - 2) && v->size(d - 3) == k->size(d - 3) && (packed || v->size(0) == n_seq));
    if (packed) {
        REQUIRE(ints(*kv_starts, kv_starts->numel()) && kv_starts->numel() >= n_seq);
        a.kv_starts = (const int32_t *) kv_starts->data_ptr();
    }
    if (kv_lens) {
        REQUIRE(ints(*kv_lens, n_seq));
        a.kv_lens = (const int32_t *) kv_lens->data_ptr();
    }
    a.n_head_kv = (int32_t) k->size(d - 2); a.dv = (int32_t) v->size(d - 1); a.n_kv = k->size(d - 3);
    a.k = gqa_pool{ k->data_ptr(), packed ? 0 : step(*k, 0), step(*k, d - 3), step(*k, d - 2) };
    a.v = gqa_pool{ v->data_ptr(), packed ? 0 : step(*v, 0), step(*v, d - 3), step(*v, d - 2) };
    REQUIRE(row_mask(a, mask, n_seq));
    const c10::DeviceGuard guard(q.device());
    GqaStream stream;
    if (!stream.take(o[11], q, !outp)) return nullptr;
    Result result;
    REQUIRE(result.take(a, q, outp));
    Apart apart;
    if (outp) {
        apart.add("out", outp);
        apart.add("q", &q); apart.add("k", k); apart.add("v", v); apart.add("q_starts", starts); apart.add("kv_starts", kv_starts); apart.add("kv_lens", kv_lens); apart.add("mask", mask);
        if (a.n_tok && !apart.check("gqa_cross_attn", 1)) return nullptr;
    }
    GqaScratch scratch;
    if (!scratch.take(o[0], q, stream, lib.cross_workspace_size(&a), a)) return nullptr;
    const int rc = unlocked(a.workspace, [&] { return lib.cross_attn(&a, stream.st); });
    return rc ? failed("gqa_cross_attn_launch", rc) : result.give(o[9]);
}

// gqa_prefix_attn(q, k_cache, v_cache, block_table, seq_lens, prefix_starts, prefix_lens, scale, logit_softcap, mask, out, n_workgroups, stream) -> out
PyObject * gqa_prefix_attn(PyObject *, PyObject * const * o, Py_ssize_t n) {
    if (!arg_count(n, 13)) return nullptr;
    const at::Tensor * in[7];
    for (int i = 0; i < 7; i++) if (!(in[i] = tensor(o[i]))) return nullptr;
    const at::Tensor & q = *in[0], * kc = in[1], * vc = in[2], * table = in[3], * lens = in[4], * starts = in[5], * plens = in[6], * mask, * outp;
    if (!optional_tensor(o[9], mask) || !optional_tensor(o[10], outp)) return nullptr;
    if (!on_gpu(q)) return nullptr;
    for (const at::Tensor * t : { kc, vc, table, lens, starts, plens, mask, outp }) SAME_DEVICE(t);
    gqa_prefix_attn_args a;
    memset(&a, 0, sizeof a);
    a.scale = (float) PyFloat_AsDouble(o[7]); a.logit_softcap = (float) PyFloat_AsDouble(o[8]);
    if (PyErr_Occurred() || !int_of(o[11], a.n_workgroups)) return nullptr;
    REQUIRE(mla_type(q) > 0 && rows_ok(q, 3, false) && q.size(0) < INTS && q.size(1) < INTS && q.size(2) < INTS);
    const int64_t n_seq = q.size(0);
    a.n_seq = (int32_t) n_seq; a.n_head = (int32_t) q.size(1); a.dk = (int32_t) q.size(2); a.type = mla_type(q);
    a.q = q.data_ptr(); a.q_nb1 = step(q, 1); a.q_nb2 = step(q, 0);
    REQUIRE(cache_ok(*kc, a.type) && kc->size(2) < INTS && kc->size(3) == a.dk);
    REQUIRE(cache_ok(*vc, a.type) && vc->size(0) == kc->size(0) && vc->size(2) == kc->size(2) && vc->size(3) < INTS);
    a.n_head_kv = (int32_t) kc->size(2); a.n_pages = kc->size(0); a.dv = (int32_t) vc->size(3);
    a.k = pool_of(*kc); a.v = pool_of(*vc);
    REQUIRE(table_ok(*table) && table->size(0) == n_seq && ints(*lens, n_seq));
    a.block_table = (const int32_t *) table->data_ptr(); a.bt_stride = table->size(1); a.seq_lens = (const int32_t *) lens->data_ptr();
    REQUIRE(plens->numel() < INTS - 1 && ints(*plens, plens->numel()) && ints(*starts, plens->numel() + 1));
    a.n_prefix = (int32_t) plens->numel();
    a.prefix_starts = (const int32_t *) starts->data_ptr(); a.prefix_lens = (const int32_t *) plens->data_ptr();
    REQUIRE(row_mask(a, mask, n_seq));
    const c10::DeviceGuard guard(q.device());
    GqaStream stream;
    if (!stream.take(o[12], q, !outp)) return nullptr;
    Result result;
    REQUIRE(result.take(a, q, outp));
    if (outp) {
        Apart apart;
        apart.add("out", outp);
        apart.add("q", &q); apart.add("k_cache", kc); apart.add("v_cache", vc); apart.add("block_table", table); apart.add("seq_lens", lens); apart.add("prefix_starts", starts);
        apart.add("prefix_lens", plens); apart.add("mask", mask);
        if (n_seq && !apart.check("gqa_prefix_attn", 1)) return nullptr;
    }
    GqaScratch scratch;
    if (!scratch.take(o[0], q, stream, lib.prefix_workspace_size(&a), a)) return nullptr;
    const int rc = unlocked(a.workspace, [&] { return lib.prefix_attn(&a, stream.st); });
    return rc ? failed("gqa_prefix_attn_launch", rc) : result.give(o[10]);
}

// bind(addresses of the entry points in Bound's order, workspace function, workspace table, torch's raw current stream, whether it is capturing, scratch on another stream)
PyObject * bind(PyObject *, PyObject * const * v, Py_ssize_t n) {
    constexpr int N = 19;
    if (!arg_count(n, N + 5)) return nullptr;
    void * p[N];
    for (int i = 0; i < N; i++) p[i] = PyLong_AsVoidPtr(v[i]);
    if (PyErr_Occurred()) return nullptr;
    v += N;
    REQUIRE(PyCallable_Check(v[0]) && PyDict_Check(v[1]) && PyCallable_Check(v[2]) && PyCallable_Check(v[3]) && PyCallable_Check(v[4]));
    lib.workspace_size = (decltype(lib.workspace_size)) p[0]; lib.attn = (decltype(lib.attn)) p[1];
    lib.kv_write = (decltype(lib.kv_write)) p[2]; lib.kv_write_rope = (decltype(lib.kv_write_rope)) p[3];
    lib.rope = (decltype(lib.rope)) p[4]; lib.mul_mat = (decltype(lib.mul_mat)) p[5];
    lib.copy = (decltype(lib.copy)) p[6]; lib.front_batch = (decltype(lib.front_batch)) p[7];
    lib.norm_rope = (decltype(lib.norm_rope)) p[8]; lib.gqa_workspace_size = (decltype(lib.gqa_workspace_size)) p[9];
    lib.gqa_attn = (decltype(lib.gqa_attn)) p[10]; lib.evict_workspace_size = (decltype(lib.evict_workspace_size)) p[11];
    lib.evict = (decltype(lib.evict)) p[12];
    lib.prompt_workspace_size = (decltype(lib.prompt_workspace_size)) p[13]; lib.prompt_attn = (decltype(lib.prompt_attn)) p[14];
    lib.prefix_workspace_size = (decltype(lib.prefix_workspace_size)) p[17]; lib.prefix_attn = (decltype(lib.prefix_attn)) p[18];
    lib.cross_workspace_size = (decltype(lib.cross_workspace_size)) p[15]; lib.cross_attn = (decltype(lib.cross_attn)) p[16];
    lib.workspace = Py_NewRef(v[0]); lib.workspaces = Py_NewRef(v[1]); lib.raw_stream = Py_NewRef(v[2]); lib.capturing = Py_NewRef(v[3]); lib.elsewhere = Py_NewRef(v[4]);
    Py_RETURN_NONE;
}

template <PyObject * (*F)(PyObject *, PyObject * const *, Py_ssize_t)> PyObject * entry(PyObject * self, PyObject * const * v, Py_ssize_t n) {
    try {
        return F(self, v, n);
    } catch (...) {   // (what HANDLE_TH_ERRORS does, without its buffer for torch's warnings: none arise here)
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
}

#define FAST(name) { #name, (PyCFunction) (void (*)(void)) entry<name>, METH_FASTCALL, nullptr }
PyMethodDef methods[] = { FAST(bind), FAST(attn), FAST(rope), FAST(mul_mat), FAST(copy), FAST(kv_write), FAST(front_batch), FAST(gqa_norm_rope), FAST(gqa_attn), FAST(gqa_evict),
                          FAST(gqa_prompt_attn), FAST(gqa_cross_attn), FAST(gqa_prefix_attn), { nullptr, nullptr, 0, nullptr } };
PyModuleDef module = { PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr };

}  // namespace

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&module); }
