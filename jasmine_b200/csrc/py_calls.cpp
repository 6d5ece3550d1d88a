// The frequent calls of the Python plumbing (jasmine_b200/__init__.py) without ctypes: a tensor is described by reading its fields instead of by
// six calls into Python, the structs live on the stack.  What a call of the small operations costs is the host's part: 21 calls of a
// two-layer model of width 128 took 255 us for 91 us of kernels.
//
// Every function returns the call's status, or None for arguments that it leaves to the Python code: anything but plain dense CUDA tensors of the
// types that a jsm_mat knows (subclasses, wrappers of transforms, other types and ranks) and numbers outside the C types.  The
// library is the one that Python has loaded (bind).
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <algorithm>
#include <initializer_list>
#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/python_variable.h>
#include "../../include/jasmine_b200.h"

namespace {

struct Library {
    decltype(&jsm_eval_elementwise) eval_elementwise;
    decltype(&jsm_eval_rows) eval_rows;
    decltype(&jsm_dot_f32) dot_f32;
    decltype(&jsm_embedding) embedding;
    decltype(&jsm_attn_prefill) attn_prefill;
    decltype(&jsm_attn_decode) attn_decode;
    decltype(&jsm_rope_rotate) rope_rotate;
    decltype(&jsm_kv_append_q8) kv_append_q8;
    decltype(&jsm_kv_read) kv_read;
    decltype(&jsm_attn_chunk_scratch_bytes) attn_chunk_scratch_bytes;
    decltype(&jsm_attn_chunk) attn_chunk;
} L = {};

// a plain dense CUDA tensor: nothing between it and its memory
const at::Tensor* plain(PyObject* o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || t.layout() != c10::kStrided || !t.is_cuda()) return nullptr;
    constexpr c10::DispatchKeySet known = c10::DispatchKeySet(c10::DispatchKey::CUDA) | c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView) |
                                          c10::DispatchKeySet(c10::DispatchKey::AutogradCUDA) | c10::DispatchKeySet(c10::DispatchKey::AutocastCUDA);
    return (t.key_set().raw_repr() & ~known.raw_repr()) == 0 ? &t : nullptr;
}

int type_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return JSM_F32;
        case at::kBFloat16: return JSM_BF16;
        case at::kInt: return JSM_I32;
        default: return -1;
    }
}

bool as_mat(PyObject* o, jsm_mat& m) {
    const at::Tensor* t = plain(o);
    if (!t || (t->dim() != 1 && t->dim() != 2)) return false;
    const int type = type_of(*t);
    const int64_t rows = t->dim() == 1 ? 1 : t->size(0), cols = t->size(-1);
    if (type < 0 || rows > INT32_MAX || cols > INT32_MAX) return false;
    m.data = t->mutable_data_ptr();
    m.rows = (int32_t)rows; m.cols = (int32_t)cols;
    m.col_stride = t->stride(-1);
    m.row_stride = t->dim() == 1 ? cols * m.col_stride : t->stride(0);
    m.dtype = type;
    return true;
}
// address of a tensor, or null for None
bool as_pointer(PyObject* o, void*& p) {
    p = nullptr;
    if (o == Py_None) return true;
    const at::Tensor* t = plain(o);
    if (!t) return false;
    p = t->mutable_data_ptr();
    return true;
}
bool as_int(PyObject* o, int& v) {
    if (!PyLong_Check(o)) return false;
    int over = 0;
    const long x = PyLong_AsLongAndOverflow(o, &over);
    v = (int)x;
    return !over && x >= INT32_MIN && x <= INT32_MAX;
}
bool as_float(PyObject* o, float& v) {
    if (PyFloat_Check(o)) v = (float)PyFloat_AS_DOUBLE(o);
    else {
        int i;
        if (!as_int(o, i)) return false;
        v = (float)i;
    }
    return true;
}
// a list or tuple of (op,), (op, index) or (op, number)
bool as_program(PyObject* o, jsm_instr (&p)[JSM_MAX_INSTR], int& n) {
    if (!PyList_Check(o) && !PyTuple_Check(o)) return false;
    const Py_ssize_t len = PySequence_Fast_GET_SIZE(o);
    if (len > JSM_MAX_INSTR) return false;
    n = (int)len;
    for (int k = 0; k < n; ++k) {
        PyObject* e = PySequence_Fast_GET_ITEM(o, k);
        if (!PyTuple_Check(e) || PyTuple_GET_SIZE(e) < 1 || !as_int(PyTuple_GET_ITEM(e, 0), p[k].op)) return false;
        p[k].arg = 0;
        p[k].imm = 0.0f;
        if (PyTuple_GET_SIZE(e) < 2) continue;
        PyObject* a = PyTuple_GET_ITEM(e, 1);
        if (p[k].op == JSM_OP_IMM || p[k].op == JSM_OP_POW ? !as_float(a, p[k].imm) : !as_int(a, p[k].arg)) return false;
    }
    return true;
}
bool as_leaves(PyObject* o, jsm_mat (&m)[JSM_MAX_LEAVES], int& n) {
    if (!PyList_Check(o) && !PyTuple_Check(o)) return false;
    const Py_ssize_t len = PySequence_Fast_GET_SIZE(o);
    if (len > JSM_MAX_LEAVES) return false;
    n = (int)len;
    for (int k = 0; k < n; ++k)
        if (!as_mat(PySequence_Fast_GET_ITEM(o, k), m[k])) return false;
    return true;
}

template <typename Call>
PyObject* status_of(Call call) {
    int s;
    void* stream = c10::cuda::getCurrentCUDAStream().stream();
    Py_BEGIN_ALLOW_THREADS
    s = (int)call(stream);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(s);
}

#define JSM_FAST(name) PyObject* name(PyObject*, PyObject* const* a, Py_ssize_t n_args)
#define JSM_NEED(cond) do { if (!(cond)) Py_RETURN_NONE; } while (0)

JSM_FAST(bind) {  // address of the shared library's handle
    if (n_args != 1) return PyErr_Format(PyExc_TypeError, "bind(handle)");
    void* h = PyLong_AsVoidPtr(a[0]);
    if (PyErr_Occurred()) return nullptr;
    auto find = [&](auto& f, const char* name) { f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(dlsym(h, name)); return f != nullptr; };
    if (!find(L.eval_elementwise, "jsm_eval_elementwise") || !find(L.eval_rows, "jsm_eval_rows") || !find(L.dot_f32, "jsm_dot_f32") ||
        !find(L.embedding, "jsm_embedding") || !find(L.attn_prefill, "jsm_attn_prefill") || !find(L.attn_decode, "jsm_attn_decode") ||
        !find(L.rope_rotate, "jsm_rope_rotate") || !find(L.kv_append_q8, "jsm_kv_append_q8") || !find(L.kv_read, "jsm_kv_read") ||
        !find(L.attn_chunk_scratch_bytes, "jsm_attn_chunk_scratch_bytes") || !find(L.attn_chunk, "jsm_attn_chunk"))
        return PyErr_Format(PyExc_ImportError, "libjasmine_b200: a symbol is missing");
    Py_RETURN_NONE;
}

JSM_FAST(eval_elementwise) {  // instrs, leaves, out
    jsm_instr p[JSM_MAX_INSTR];
    jsm_mat l[JSM_MAX_LEAVES], out;
    int n, nl;
    JSM_NEED(n_args == 3 && as_program(a[0], p, n) && as_leaves(a[1], l, nl) && as_mat(a[2], out));
    return status_of([&](void* st) { return L.eval_elementwise(p, n, l, nl, out, st); });
}

JSM_FAST(eval_rows) {  // kind, axis, instrs, leaves, out, gain, bias, eps
    jsm_instr p[JSM_MAX_INSTR];
    jsm_mat l[JSM_MAX_LEAVES], out;
    int kind, axis, n, nl;
    void *gain, *bias;
    float eps;
    JSM_NEED(n_args == 8 && as_int(a[0], kind) && as_int(a[1], axis) && as_program(a[2], p, n) && as_leaves(a[3], l, nl) && as_mat(a[4], out) &&
             as_pointer(a[5], gain) && as_pointer(a[6], bias) && as_float(a[7], eps));
    return status_of([&](void* st) { return L.eval_rows(kind, axis, p, n, l, nl, (const float*)gain, (const float*)bias, eps, out, st); });
}

JSM_FAST(dot_f32) {  // A, B, out, bias, epilogue, residual
    jsm_mat A, B, out, bias, res;
    int epilogue;
    JSM_NEED(n_args == 6 && as_mat(a[0], A) && as_mat(a[1], B) && as_mat(a[2], out) && (a[3] == Py_None || as_mat(a[3], bias)) && as_int(a[4], epilogue) &&
             (a[5] == Py_None || as_mat(a[5], res)));
    const jsm_mat *pb = a[3] == Py_None ? nullptr : &bias, *pr = a[5] == Py_None ? nullptr : &res;
    return status_of([&](void* st) { return L.dot_f32(A, B, pb, epilogue, pr, out, st); });
}

JSM_FAST(embedding) {  // table, ids, pos_table, positions, out
    void *table, *ids, *pos, *at, *out;
    JSM_NEED(n_args == 5 && as_pointer(a[0], table) && as_pointer(a[1], ids) && as_pointer(a[2], pos) && as_pointer(a[3], at) && as_pointer(a[4], out));
    JSM_NEED(a[0] != Py_None && a[1] != Py_None && a[4] != Py_None);
    const at::Tensor &t = THPVariable_Unpack(a[0]), &i = THPVariable_Unpack(a[1]);
    const int type = type_of(t);
    JSM_NEED(type >= 0 && t.dim() >= 2 && i.dim() >= 1 && t.size(1) <= INT32_MAX && i.size(0) <= INT32_MAX);
    const int T = (int)i.size(0), d = (int)t.size(1);
    return status_of([&](void* st) { return L.embedding(table, pos, (const int32_t*)ids, (const int32_t*)at, out, (jsm_dtype)type, T, d, st); });
}

JSM_FAST(attn_prefill) {  // q, k, v, batch, Hq, Hkv, D, causal, scale, rope, impl, out
    void *q, *k, *v, *rope, *out;
    int batch, hq, hkv, d, causal, impl;
    float scale;
    JSM_NEED(n_args == 12 && as_pointer(a[0], q) && as_pointer(a[1], k) && as_pointer(a[2], v) && as_int(a[3], batch) && as_int(a[4], hq) && as_int(a[5], hkv) &&
             as_int(a[6], d) && as_int(a[7], causal) && as_float(a[8], scale) && as_pointer(a[9], rope) && as_int(a[10], impl) && as_pointer(a[11], out));
    JSM_NEED(a[0] != Py_None && a[1] != Py_None && a[2] != Py_None && a[11] != Py_None && batch > 0);
    const at::Tensor &tq = THPVariable_Unpack(a[0]), &tk = THPVariable_Unpack(a[1]);
    const int type = type_of(tq);
    JSM_NEED(type >= 0 && tq.dim() >= 1 && tk.dim() >= 1 && tq.size(0) <= INT32_MAX && tk.size(0) <= INT32_MAX);
    const int nq = (int)(tq.size(0) / batch), nk = (int)(tk.size(0) / batch);
    return status_of([&](void* st) { return L.attn_prefill(q, k, v, out, (jsm_dtype)type, batch, nq, nk, hq, hkv, d, causal, scale, (const float*)rope, impl, st); });
}

JSM_FAST(attn_decode) {  // q, pool, block_table, context_lens, Hq, Hkv, D, max_context, scale, rope, scratch, out
    void *q, *pool, *table, *lens, *rope, *scratch, *out;
    int hq, hkv, d, most;
    float scale;
    JSM_NEED(n_args == 12 && as_pointer(a[0], q) && as_pointer(a[1], pool) && as_pointer(a[2], table) && as_pointer(a[3], lens) && as_int(a[4], hq) &&
             as_int(a[5], hkv) && as_int(a[6], d) && as_int(a[7], most) && as_float(a[8], scale) && as_pointer(a[9], rope) && as_pointer(a[10], scratch) &&
             as_pointer(a[11], out));
    JSM_NEED(a[0] != Py_None && a[1] != Py_None && a[2] != Py_None && a[3] != Py_None && a[10] != Py_None && a[11] != Py_None);
    const at::Tensor &tq = THPVariable_Unpack(a[0]), &tt = THPVariable_Unpack(a[2]);
    JSM_NEED(tq.dim() >= 1 && tt.dim() >= 2 && tq.size(0) <= INT32_MAX && tt.size(1) <= INT32_MAX);
    const int n = (int)tq.size(0), pages = (int)tt.size(1);
    const int64_t pitch = tq.stride(0);
    return status_of([&](void* st) {
        return L.attn_decode(q, pitch, pool, (const int32_t*)table, pages, (const int32_t*)lens, n, hq, hkv, d, scale, (const float*)rope, most, scratch, out, st);
    });
}

// the same on the current device, where the call runs; the device is asked for once per call, under the interpreter's lock
int call_device = -1;
const at::Tensor* here(PyObject* o) {
    const at::Tensor* t = plain(o);
    return t && t->get_device() == call_device ? t : nullptr;
}
// Rows [T, columns] of adjacent elements; a single row's pitch means nothing.
struct Rows {
    void* data = nullptr;
    int64_t T = 0, pitch = 0;
    int type = -1;
};
bool as_rows(PyObject* o, int64_t columns, Rows& r) {
    const at::Tensor* t = here(o);
    if (!t || t->dim() != 2 || t->size(1) != columns || (columns > 1 && t->stride(1) != 1) || t->size(0) > INT32_MAX) return false;
    r.data = t->mutable_data_ptr();
    r.T = t->size(0);
    r.pitch = r.T > 1 ? t->stride(0) : columns;
    r.type = type_of(*t);
    return true;
}
bool as_ints(PyObject* o, std::initializer_list<int64_t> shape, const int32_t*& p) {
    const at::Tensor* t = here(o);
    if (!t || t->scalar_type() != at::kInt || !t->is_contiguous() || t->dim() != (int64_t)shape.size() || !std::equal(shape.begin(), shape.end(), t->sizes().begin())) return false;
    p = (const int32_t*)t->mutable_data_ptr();
    return true;
}
// a table [positions, rot / 2, 2], or None
bool as_rotation(PyObject* o, int rot, const float*& p, int& n) {
    p = nullptr;
    n = 0;
    if (o == Py_None) return true;
    const at::Tensor* t = here(o);
    if (!t || t->scalar_type() != at::kFloat || !t->is_contiguous() || t->dim() != 3 || t->size(1) != rot / 2 || t->size(2) != 2 || t->size(0) > INT32_MAX) return false;
    p = (const float*)t->mutable_data_ptr();
    n = (int)t->size(0);
    return true;
}
// pool, scales (or None), block table, starts, context lengths
struct Cache {
    void *pool, *scales = nullptr;
    int pages, max_pages, seqs;
    const int32_t *table, *starts, *lens;
};
bool as_cache(PyObject* pool, PyObject* scales, PyObject* table, PyObject* starts, PyObject* lens, int hkv, int d, Cache& c) {
    const at::Tensor *p = here(pool), *b = here(table), *l = here(lens);
    if (!p || !b || !l || p->dim() != 5 || !p->is_contiguous() || p->size(1) != 2 || p->size(2) != hkv || p->size(3) != JSM_PAGE_SIZE || p->size(4) != d || p->size(0) > INT32_MAX)
        return false;
    if (b->dim() != 2 || l->dim() != 1 || b->size(1) > INT32_MAX || l->size(0) > INT32_MAX) return false;
    if (scales != Py_None) {
        const at::Tensor* s = here(scales);
        if (!s || s->scalar_type() != at::kBFloat16 || !s->is_contiguous() || s->dim() != 4 || !std::equal(s->sizes().begin(), s->sizes().end(), p->sizes().begin())) return false;
        c.scales = s->mutable_data_ptr();
    }
    if (p->scalar_type() != (scales != Py_None ? at::kChar : at::kBFloat16)) return false;
    c.pool = p->mutable_data_ptr();
    c.pages = (int)p->size(0);
    c.max_pages = (int)b->size(1);
    c.seqs = (int)l->size(0);
    return as_ints(table, {c.seqs, c.max_pages}, c.table) && as_ints(starts, {c.seqs + 1ll}, c.starts) && as_ints(lens, {c.seqs}, c.lens);
}

JSM_FAST(rope_rotate) {  // q, k, table, Hq, Hkv, D, rot, positions, layout, inverse, q_out, k_out
    call_device = c10::cuda::current_device();
    int hq, hkv, d, rot, layout, n;
    const float* table;
    JSM_NEED(n_args == 12 && as_int(a[3], hq) && as_int(a[4], hkv) && as_int(a[5], d) && as_int(a[6], rot) && as_int(a[8], layout) && a[2] != Py_None &&
             as_rotation(a[2], rot, table, n) && hq >= 0 && hkv >= 0 && d > 0 && (hq > 0 || hkv > 0));
    JSM_NEED((hq > 0) == (a[0] != Py_None) && (hkv > 0) == (a[1] != Py_None));
    Rows q, k, qo, ko;
    JSM_NEED(!hq || (as_rows(a[0], (int64_t)hq * d, q) && as_rows(a[10], (int64_t)hq * d, qo) && q.T == qo.T && q.type == qo.type));
    JSM_NEED(!hkv || (as_rows(a[1], (int64_t)hkv * d, k) && as_rows(a[11], (int64_t)hkv * d, ko) && k.T == ko.T && k.type == ko.type));
    JSM_NEED(!hq || !hkv || (q.T == k.T && q.type == k.type));
    const int T = (int)(hq ? q.T : k.T), type = hq ? q.type : k.type;
    const int32_t* at = nullptr;
    JSM_NEED(type >= 0 && (a[7] == Py_None || as_ints(a[7], {T}, at)) && (a[9] == Py_True || a[9] == Py_False));
    const int inverse = a[9] == Py_True;
    return status_of([&](void* st) {
        return L.rope_rotate(q.data, q.pitch, qo.data, qo.pitch, hq, k.data, k.pitch, ko.data, ko.pitch, hkv, (jsm_dtype)type, d, table, n, rot, layout, inverse, at, T, st);
    });
}

JSM_FAST(kv_append_q8) {  // pool, scales, block_table, k, v, starts, context_lens, Hkv, D, rope, rot, layout
    call_device = c10::cuda::current_device();
    int hkv, d, rot, layout, n;
    const float* table;
    Cache c;
    Rows k, v;
    JSM_NEED(n_args == 12 && as_int(a[7], hkv) && as_int(a[8], d) && as_int(a[10], rot) && as_int(a[11], layout) && as_rotation(a[9], rot, table, n) && hkv > 0 && d > 0 &&
             a[1] != Py_None && as_cache(a[0], a[1], a[2], a[5], a[6], hkv, d, c) && as_rows(a[3], (int64_t)hkv * d, k) && as_rows(a[4], (int64_t)hkv * d, v));
    JSM_NEED(k.type == JSM_BF16 && v.type == JSM_BF16 && k.T == v.T && k.pitch == v.pitch);
    return status_of([&](void* st) {
        return L.kv_append_q8(c.pool, c.scales, c.pages, c.table, c.max_pages, k.data, v.data, k.pitch, c.starts, c.lens, c.seqs, (int)k.T, hkv, d, table, n, rot, layout, st);
    });
}

JSM_FAST(kv_read) {  // pool, scales, block_table, starts, context_lens, T, Hkv, D, k_out, v_out (both or neither), f32; with neither the new outputs come back
    call_device = c10::cuda::current_device();
    int T, hkv, d;
    Cache c;
    Rows k, v;
    JSM_NEED(n_args == 11 && as_int(a[5], T) && as_int(a[6], hkv) && as_int(a[7], d) && T >= 0 && hkv > 0 && d > 0 && as_cache(a[0], a[1], a[2], a[3], a[4], hkv, d, c));
    JSM_NEED((a[8] == Py_None) == (a[9] == Py_None) && (a[10] == Py_True || a[10] == Py_False));
    const bool fresh = a[8] == Py_None;
    PyObject* out = nullptr;
    if (fresh) {
        const auto options = THPVariable_Unpack(a[0]).options().dtype(a[10] == Py_True ? at::kFloat : at::kBFloat16);
        PyObject *ko = THPVariable_Wrap(at::empty({T, (int64_t)hkv * d}, options)), *vo = THPVariable_Wrap(at::empty({T, (int64_t)hkv * d}, options));
        out = PyTuple_Pack(2, ko, vo);
        Py_XDECREF(ko);
        Py_XDECREF(vo);
        if (!out) return nullptr;
    }
    const bool fits = as_rows(fresh ? PyTuple_GET_ITEM(out, 0) : a[8], (int64_t)hkv * d, k) && as_rows(fresh ? PyTuple_GET_ITEM(out, 1) : a[9], (int64_t)hkv * d, v) &&
                      k.type >= 0 && k.type == v.type && k.T == T && v.T == T && k.pitch == v.pitch;
    if (!fits) {
        Py_XDECREF(out);
        Py_RETURN_NONE;
    }
    PyObject* status = status_of([&](void* st) {
        return L.kv_read(c.pool, c.scales, c.pages, c.table, c.max_pages, c.starts, c.lens, c.seqs, T, hkv, d, k.data, v.data, k.pitch, (jsm_dtype)k.type, st);
    });
    if (!fresh || !status || PyLong_AsLong(status) != 0) {
        Py_XDECREF(out);
        return status;
    }
    Py_DECREF(status);
    return out;
}

JSM_FAST(attn_chunk) {  // q, pool, scales, block_table, starts, context_lens, Hq, Hkv, D, max_new, max_context, window, scale, scratch, out
    call_device = c10::cuda::current_device();
    int hq, hkv, d, most_new, most, window;
    float scale;
    Cache c;
    Rows q, out;
    JSM_NEED(n_args == 15 && as_int(a[6], hq) && as_int(a[7], hkv) && as_int(a[8], d) && as_int(a[9], most_new) && as_int(a[10], most) && as_int(a[11], window) &&
             as_float(a[12], scale) && hq > 0 && hkv > 0 && d > 0 && as_cache(a[1], a[2], a[3], a[4], a[5], hkv, d, c) && as_rows(a[0], (int64_t)hq * d, q) &&
             as_rows(a[14], (int64_t)hq * d, out));
    JSM_NEED(q.type == JSM_BF16 && out.type == JSM_BF16 && q.T == out.T);
    void* scratch = nullptr;
    size_t bytes = 0;
    at::Tensor own;
    if (a[13] != Py_None) {
        JSM_NEED(here(a[13]) && as_pointer(a[13], scratch) && THPVariable_Unpack(a[13]).is_contiguous());
        bytes = THPVariable_Unpack(a[13]).nbytes();
    } else if ((bytes = L.attn_chunk_scratch_bytes(c.seqs, (int)q.T, most_new, most, hq, hkv, d, window)) > 0) {
        own = at::empty({(int64_t)bytes}, THPVariable_Unpack(a[0]).options().dtype(at::kByte));
        scratch = own.mutable_data_ptr();
    }
    return status_of([&](void* st) {
        return L.attn_chunk(q.data, q.pitch, c.pool, c.scales, c.pages, c.table, c.max_pages, c.starts, c.lens, c.seqs, (int)q.T, most_new, most, hq, hkv, d, window, scale,
                            scratch, bytes, out.data, out.pitch, st);
    });
}

// torch throws for tensors that keep their memory to themselves (sizes or addresses that are not to be read): the Python code meets the same and raises
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    try {
        return F(self, a, n);
    } catch (...) {
        Py_RETURN_NONE;
    }
}

#define JSM_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<name>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {JSM_METHOD(bind), JSM_METHOD(eval_elementwise), JSM_METHOD(eval_rows), JSM_METHOD(dot_f32), JSM_METHOD(embedding),
                         JSM_METHOD(attn_prefill), JSM_METHOD(attn_decode), JSM_METHOD(rope_rotate), JSM_METHOD(kv_append_q8), JSM_METHOD(kv_read), JSM_METHOD(attn_chunk), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch: the torch whose headers this module has been built with, `<version> <revision>`.  The fields of a tensor are read at their places in that one.
PyMODINIT_FUNC PyInit__native() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch", JSM_TORCH) != 0) Py_CLEAR(m);
    return m;
}
