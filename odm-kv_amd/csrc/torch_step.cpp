// kvquant._native: the decode step's host path over torch tensors (a CPython extension).
//
// A decode step of one layer is 2 kernel launches of together 18 us at 32k tokens, and a model has the host run it once per
// layer and token: what the host adds (argument checks, views, the output tensor, ctypes, bookkeeping) has to stay below
// that.  In Python these were 20 us of a 31 us layer step; here they are about 2.
#include <Python.h>
#include <structmember.h>
#include <stdlib.h>
#include <string.h>
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/odmkv.h"

namespace {

typedef int (*step_fn)(const odmkv_step_t*, const void*, const void*, const void*, int64_t, int64_t, int, void*, float*, void*);

at::ScalarType scalar_of(int code) {
    return code == ODMKV_F16 ? at::kHalf : code == ODMKV_BF16 ? at::kBFloat16 : at::kFloat;
}

struct Step {
    PyObject_HEAD
    odmkv_step_t st;
    step_fn fn;
    PyObject* keep;             // what the block's pointers point into
    long long seq_len;          // tokens the store holds
    long long room;             // exact tokens that can still be appended without touching the host's tables
    long long appended;         // since this object was made
    unsigned long long stream;  // the workspace belongs to it
    int Hkv, device;
    int attends;                // whether an attention call may append its token (the press keeps new tokens exact)
};

PyObject* s_sliding = nullptr; PyObject* s_softcap = nullptr; PyObject* s_aux = nullptr; PyObject* s_scaling = nullptr;

int step_init(PyObject* self_, PyObject* args, PyObject*) {
    Step* self = (Step*)self_;
    unsigned long long fn, store, work, ops, pi_v, cb, cb_host, inv, ws, ws_bytes, stream;
    int B, Hq, Hkv, q_dt, out_dt, device, attends;
    double scaling;
    long long seq_len, room;
    PyObject* keep;
    if (!PyArg_ParseTuple(args, "KKKKKKKKKKKiiiiiidpLLO", &fn, &store, &work, &ops, &pi_v, &cb, &cb_host, &inv, &ws, &ws_bytes, &stream,
                          &B, &Hq, &Hkv, &q_dt, &out_dt, &device, &scaling, &attends, &seq_len, &room, &keep))
        return -1;
    if (!fn || !store || !work || B <= 0 || Hkv <= 0 || Hq % Hkv || q_dt < 0 || q_dt > 2 || out_dt < 0 || out_dt > 2) {
        PyErr_SetString(PyExc_ValueError, "Step: bad arguments");
        return -1;
    }
    self->fn = (step_fn)(uintptr_t)fn;
    odmkv_step_t& s = self->st;
    s.store = (const odmkv_packed_t*)(uintptr_t)store;
    s.work = (const odmkv_worklist_t*)(uintptr_t)work;
    s.pi_k_ops = (const uint16_t*)(uintptr_t)ops;
    s.pi_v = (const float*)(uintptr_t)pi_v;
    s.codebooks = (const float*)(uintptr_t)cb;
    s.codebooks_host = (const float*)(uintptr_t)cb_host;
    s.inv_scales = (const float*)(uintptr_t)inv;
    s.workspace = (void*)(uintptr_t)ws;
    s.workspace_bytes = (size_t)ws_bytes;
    s.B = B; s.Hq = Hq; s.q_dtype = q_dt; s.out_dtype = out_dt; s.scaling = (float)scaling;
    self->stream = stream; self->Hkv = Hkv; self->device = device; self->attends = attends;
    self->seq_len = seq_len; self->room = room; self->appended = 0;
    Py_INCREF(keep);
    Py_XSETREF(self->keep, keep);
    return 0;
}

void step_dealloc(PyObject* self) {
    Py_XDECREF(((Step*)self)->keep);
    Py_TYPE(self)->tp_free(self);
}

bool query_fits(const Step* s, const at::Tensor& q) {
    const odmkv_step_t& st = s->st;
    return q.is_cuda() && q.get_device() == s->device && q.scalar_type() == scalar_of(st.q_dtype) && q.is_contiguous()
           && q.numel() == (int64_t)st.B * st.Hq * ODMKV_HEAD_DIM && q.dim() >= 3 && q.size(0) == st.B && q.size(1) == st.Hq;
}

// Append the last token of keys / values [B, Hkv, n, 128] and attend with query; nullptr and no Python error: this call is
// not what the block was made for, nothing was done.
PyObject* run(Step* s, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, double scaling, unsigned long long stream) {
    const odmkv_step_t& st = s->st;
    if (s->room <= 0 || (float)scaling != st.scaling || stream != s->stream) return nullptr;
    if (!query_fits(s, q)) return nullptr;
    const at::ScalarType exact = scalar_of(st.store->exact_dtype);
    if (k.dim() != 4 || v.dim() != 4 || k.scalar_type() != exact || v.scalar_type() != exact || !k.is_cuda() || !v.is_cuda()
        || k.get_device() != s->device || v.get_device() != s->device)
        return nullptr;
    const auto ks = k.sizes(), kt = k.strides(), vt = v.strides();
    if (ks != v.sizes() || ks[0] != st.B || ks[1] != s->Hkv || ks[2] < 1 || ks[3] != ODMKV_HEAD_DIM) return nullptr;
    if (kt[3] != 1 || vt[3] != 1 || kt[0] != vt[0] || kt[1] != vt[1]) return nullptr;
    const char* kp = (const char*)k.data_ptr() + (ks[2] - 1) * kt[2] * 2;
    const char* vp = (const char*)v.data_ptr() + (ks[2] - 1) * vt[2] * 2;
    at::Tensor out = at::empty({st.B, 1, st.Hq, ODMKV_HEAD_DIM}, q.options().dtype(scalar_of(st.out_dtype)));
    const int rc = s->fn(&st, q.data_ptr(), kp, vp, kt[0], kt[1], (int)s->seq_len, out.data_ptr(), nullptr, (void*)(uintptr_t)stream);
    if (rc) return PyErr_Format(rc == ODMKV_EHIP ? PyExc_RuntimeError : PyExc_ValueError, "odmkv: decode step failed (code %d)", rc);
    s->seq_len += 1; s->room -= 1; s->appended += 1;
    return THPVariable_Wrap(std::move(out));
}

#define GUARDED(...)                                                   \
    try { __VA_ARGS__ } catch (const std::exception& e) {                     \
        PyErr_SetString(PyExc_RuntimeError, e.what());                 \
        return nullptr;                                                \
    }

// step(query, keys, values, scaling, stream): one new token; [B, 1, Hq, 128], or None if the block does not fit the call
PyObject* step_step(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    if (n != 5 || !THPVariable_Check(a[0]) || !THPVariable_Check(a[1]) || !THPVariable_Check(a[2])) {
        PyErr_SetString(PyExc_TypeError, "step(query, keys, values, scaling, stream)");
        return nullptr;
    }
    const double scaling = PyFloat_AsDouble(a[3]);
    const unsigned long long stream = PyLong_AsUnsignedLongLong(a[4]);
    if (PyErr_Occurred()) return nullptr;
    GUARDED(
        const at::Tensor& k = THPVariable_Unpack(a[1]);
        PyObject* out = k.dim() == 4 && k.size(2) == 1 ? run((Step*)self, THPVariable_Unpack(a[0]), k, THPVariable_Unpack(a[2]), scaling, stream) : nullptr;
        if (!out && !PyErr_Occurred()) Py_RETURN_NONE;
        return out;
    )
}

// attend(query, keys, values, kwargs, stream): an attention call of a model over the store; None: not a call for the block
PyObject* step_attend(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    if (n != 5 || !THPVariable_Check(a[0]) || !THPVariable_Check(a[1]) || !THPVariable_Check(a[2]) || !PyDict_Check(a[3])) {
        PyErr_SetString(PyExc_TypeError, "attend(query, keys, values, kwargs, stream)");
        return nullptr;
    }
    Step* s = (Step*)self;
    if (!s->attends) Py_RETURN_NONE;
    for (PyObject* name : {s_sliding, s_softcap, s_aux}) {
        PyObject* x = PyDict_GetItem(a[3], name);
        if (x && x != Py_None) Py_RETURN_NONE;
    }
    double scaling = 0.08838834764831845;                     // 128 ** -0.5
    PyObject* sc = PyDict_GetItem(a[3], s_scaling);
    if (sc && sc != Py_None) scaling = PyFloat_AsDouble(sc);
    const unsigned long long stream = PyLong_AsUnsignedLongLong(a[4]);
    if (PyErr_Occurred()) return nullptr;
    const char* off = getenv("ODMKV_FUSED_DECODE");
    if (off && strcmp(off, "0") == 0) Py_RETURN_NONE;
    GUARDED(
        const at::Tensor& q = THPVariable_Unpack(a[0]);
        const at::Tensor& k = THPVariable_Unpack(a[1]);
        // one query token, and the dense length (or that of its aliased views) one ahead of the store's
        if (q.dim() != 4 || q.size(2) != 1 || k.dim() != 4 || k.size(2) != s->seq_len + 1 || s->st.q_dtype != s->st.out_dtype) Py_RETURN_NONE;
        PyObject* out = run(s, q, k, THPVariable_Unpack(a[2]), scaling, stream);
        if (!out && !PyErr_Occurred()) Py_RETURN_NONE;
        return out;
    )
}

// look(query, scaling, stream): attention alone, nothing appended; [B, Hq, 128], or None if the block does not fit the call
PyObject* step_look(PyObject* self, PyObject* const* a, Py_ssize_t n) {
    if (n != 3 || !THPVariable_Check(a[0])) {
        PyErr_SetString(PyExc_TypeError, "look(query, scaling, stream)");
        return nullptr;
    }
    const double scaling = PyFloat_AsDouble(a[1]);
    const unsigned long long stream = PyLong_AsUnsignedLongLong(a[2]);
    if (PyErr_Occurred()) return nullptr;
    GUARDED(
        Step* s = (Step*)self;
        const odmkv_step_t& st = s->st;
        const at::Tensor& q = THPVariable_Unpack(a[0]);
        if (!query_fits(s, q) || (float)scaling != st.scaling || stream != s->stream) Py_RETURN_NONE;
        at::Tensor out = at::empty({st.B, st.Hq, ODMKV_HEAD_DIM}, q.options().dtype(scalar_of(st.out_dtype)));
        const int rc = s->fn(&st, q.data_ptr(), nullptr, nullptr, 0, 0, 0, out.data_ptr(), nullptr, (void*)(uintptr_t)stream);
        if (rc) return PyErr_Format(rc == ODMKV_EHIP ? PyExc_RuntimeError : PyExc_ValueError, "odmkv: decode attention failed (code %d)", rc);
        return THPVariable_Wrap(std::move(out));
    )
}

PyMethodDef step_methods[] = {
    {"step", (PyCFunction)(void*)step_step, METH_FASTCALL, nullptr},
    {"look", (PyCFunction)(void*)step_look, METH_FASTCALL, nullptr},
    {"attend", (PyCFunction)(void*)step_attend, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyMemberDef step_members[] = {
    {"seq_len", T_LONGLONG, offsetof(Step, seq_len), READONLY, nullptr},
    {"room", T_LONGLONG, offsetof(Step, room), READONLY, nullptr},
    {"appended", T_LONGLONG, offsetof(Step, appended), READONLY, nullptr},
    {nullptr, 0, 0, 0, nullptr}};

PyTypeObject StepType = {PyVarObject_HEAD_INIT(nullptr, 0)};

PyObject* alias_both(const at::Tensor& keys, const at::Tensor& values, long long length) {
    const at::Tensor* both[2] = {&keys, &values};
    for (const at::Tensor* t : both)
        if (t->dim() != 4 || t->size(2) < 1) return PyErr_Format(PyExc_ValueError, "alias: [B, H, n, D] tensors with a token at least");
    at::Tensor view[2];
    for (int i = 0; i < 2; ++i) {
        const auto z = both[i]->sizes(); const auto r = both[i]->strides();
        view[i] = both[i]->as_strided({z[0], z[1], length, z[3]}, {r[0], r[1], 0, r[3]}, both[i]->storage_offset() + (z[2] - 1) * r[2]);
    }
    PyObject* out = PyTuple_New(2);
    if (out)
        for (int i = 0; i < 2; ++i) PyTuple_SET_ITEM(out, i, THPVariable_Wrap(std::move(view[i])));
    return out;
}

// alias(keys, values, length): [B, H, n, D] each -> stride-0 views [B, H, length, D] of the last token
PyObject* native_alias(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 3 || !THPVariable_Check(a[0]) || !THPVariable_Check(a[1])) {
        PyErr_SetString(PyExc_TypeError, "alias(keys, values, length)");
        return nullptr;
    }
    const long long length = PyLong_AsLongLong(a[2]);
    if (PyErr_Occurred()) return nullptr;
    GUARDED(
        return alias_both(THPVariable_Unpack(a[0]), THPVariable_Unpack(a[1]), length);
    )
}

// ---- the paged cache's calls of every layer and step: None where a call does not fit as it is, and Python checks, copies or refuses
typedef int (*write_fn)(const odmkv_pages_t*, int, const void*, int64_t, int64_t, int64_t, const void*, int64_t, int64_t, int64_t, int, void*);
typedef int (*attend_fn)(const odmkv_attend_t*, void*);
typedef size_t (*attend_bytes_fn)(const odmkv_pages_t*, int, int, int);

// rows of 128 of the cache's type on its device that start on 16 bytes
bool rows_fit(const odmkv_pages_t* p, const at::Tensor& t, int device) {
    if (t.dim() != 4 || !t.is_cuda() || t.get_device() != device || t.scalar_type() != scalar_of(p->dtype)) return false;
    const auto z = t.sizes(); const auto r = t.strides();
    return z[0] == p->rows && z[3] == ODMKV_HEAD_DIM && r[3] == 1 && ((r[0] | r[1] | r[2]) & 7) == 0 && ((uintptr_t)t.data_ptr() & 15) == 0;
}

PyObject* raise_odmkv(int rc, const char* what) {
    return PyErr_Format(rc == ODMKV_EHIP ? PyExc_RuntimeError : PyExc_ValueError, "odmkv: %s failed (code %d)", what, rc);
}

// paged_write(entry, pages, device, layer, keys, values, stream): True, or None
PyObject* native_paged_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 7 || !THPVariable_Check(a[4]) || !THPVariable_Check(a[5])) {
        PyErr_SetString(PyExc_TypeError, "paged_write(entry, pages, device, layer, keys, values, stream)");
        return nullptr;
    }
    const write_fn fn = (write_fn)(uintptr_t)PyLong_AsUnsignedLongLong(a[0]);
    const odmkv_pages_t* p = (const odmkv_pages_t*)(uintptr_t)PyLong_AsUnsignedLongLong(a[1]);
    const int device = (int)PyLong_AsLong(a[2]);
    const long layer = PyLong_AsLong(a[3]);
    const unsigned long long stream = PyLong_AsUnsignedLongLong(a[6]);
    if (PyErr_Occurred()) return nullptr;
    GUARDED(
        const at::Tensor& k = THPVariable_Unpack(a[4]);
        const at::Tensor& v = THPVariable_Unpack(a[5]);
        if (layer < 0 || layer >= p->layers || !rows_fit(p, k, device) || !rows_fit(p, v, device) || k.sizes() != v.sizes() || k.size(1) != p->Hkv
            || k.size(2) > INT32_MAX) Py_RETURN_NONE;
        const int rc = fn(p, (int)layer, k.data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.data_ptr(), v.stride(0), v.stride(1), v.stride(2),
                          (int)k.size(2), (void*)(uintptr_t)stream);
        if (rc) return raise_odmkv(rc, "storing tokens");
        Py_RETURN_TRUE;
    )
}

// paged_attend(attend entry, workspace entry, pages, device, layer, query, scaling, cap, window, max_length, want_lse, counts, slopes, prefix, starts,
// stream, plan): out, or (out, lse), or None.  counts, slopes, prefix, starts: None, or tensors of the right type and shape, contiguous.
PyObject* native_paged_attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 17 || !THPVariable_Check(a[5])) {
        PyErr_SetString(PyExc_TypeError, "paged_attend(attend, bytes, pages, device, layer, query, scaling, cap, window, max_length, want_lse, counts, "
                                         "slopes, prefix, starts, stream, plan)");
        return nullptr;
    }
    const attend_fn fn = (attend_fn)(uintptr_t)PyLong_AsUnsignedLongLong(a[0]);
    const attend_bytes_fn bytes_of = (attend_bytes_fn)(uintptr_t)PyLong_AsUnsignedLongLong(a[1]);
    const odmkv_pages_t* p = (const odmkv_pages_t*)(uintptr_t)PyLong_AsUnsignedLongLong(a[2]);
    const int device = (int)PyLong_AsLong(a[3]);
    const long layer = PyLong_AsLong(a[4]);
    const double scaling = PyFloat_AsDouble(a[6]);
    const double cap = PyFloat_AsDouble(a[7]);
    const long long window = PyLong_AsLongLong(a[8]);
    const long long longest = PyLong_AsLongLong(a[9]);
    const int want_lse = PyObject_IsTrue(a[10]);
    const unsigned long long stream = PyLong_AsUnsignedLongLong(a[15]);
    const unsigned long long plan = PyLong_AsUnsignedLongLong(a[16]);
    if (PyErr_Occurred()) return nullptr;
    GUARDED(
        const at::Tensor& q = THPVariable_Unpack(a[5]);
        if (layer < 0 || layer >= p->layers || !rows_fit(p, q, device)) Py_RETURN_NONE;
        const int64_t Hq = q.size(1);
        const int64_t L = q.size(2);
        if (Hq <= 0 || Hq % p->Hkv || Hq / p->Hkv > ODMKV_MAX_GROUP || L < 1 || L > (1 << 26)) Py_RETURN_NONE;
        const void* small[4];
        for (int i = 0; i < 4; ++i) {
            small[i] = nullptr;
            if (a[11 + i] == Py_None) continue;
            if (!THPVariable_Check(a[11 + i])) Py_RETURN_NONE;
            const at::Tensor& t = THPVariable_Unpack(a[11 + i]);
            const int64_t want = i == 1 ? Hq : p->rows;
            if (!t.is_cuda() || t.get_device() != device || t.scalar_type() != (i == 1 ? at::kFloat : at::kInt) || !t.is_contiguous() || t.dim() < 1
                || t.size(0) != want || (i < 3 ? t.dim() != 1 : t.dim() > 2 || (t.dim() == 2 && t.size(1) != L))) Py_RETURN_NONE;
            small[i] = t.data_ptr();
        }
        const bool some = a[11] != Py_None;                   // (rows behind a count come back as 0)
        const int64_t shape[4] = {p->rows, L, Hq, ODMKV_HEAD_DIM};
        const int64_t lse_shape[3] = {p->rows, Hq, L};
        const auto make = [&](at::IntArrayRef z, at::ScalarType type) { return some ? at::zeros(z, q.options().dtype(type)) : at::empty(z, q.options().dtype(type)); };
        at::Tensor out = make(at::IntArrayRef(shape, 4), q.scalar_type());
        at::Tensor lse;
        if (want_lse) lse = make(at::IntArrayRef(lse_shape, 3), at::kFloat);
        const size_t bytes = bytes_of(p, (int)Hq, (int)L, (int)longest);
        at::Tensor ws;
        if (bytes) ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));      // (of its own for every call: a graph's is the graph's)
        odmkv_attend_t d;
        memset(&d, 0, sizeof d);
        d.pages = p; d.q = q.data_ptr(); d.q_stride_b = q.stride(0); d.q_stride_h = q.stride(1); d.q_stride_l = q.stride(2);
        d.out = out.data_ptr();
        d.lse = want_lse ? (float*)lse.data_ptr() : nullptr;
        d.counts = (const int32_t*)small[0]; d.slopes = (const float*)small[1]; d.prefix = (const int32_t*)small[2]; d.starts = (const int32_t*)small[3];
        if (small[3]) {
            const at::Tensor& t = THPVariable_Unpack(a[14]);
            d.start_stride_b = t.stride(0);
            d.start_stride_l = t.dim() == 2 ? t.stride(1) : 0;
        }
        d.workspace = bytes ? ws.data_ptr() : nullptr; d.workspace_bytes = bytes;
        d.layer = (int)layer; d.L = (int)L; d.Hq = (int)Hq; d.window = (int)window; d.max_length = (int)longest;
        d.scaling = (float)scaling; d.cap = (float)cap; d.plan = (const int32_t*)(uintptr_t)plan;
        const int rc = fn(&d, (void*)(uintptr_t)stream);
        if (rc) return raise_odmkv(rc, "attention over the paged cache");
        if (!want_lse) return THPVariable_Wrap(std::move(out));
        PyObject* both = PyTuple_New(2);
        if (both) {
            PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(out)));
            PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(lse)));
        }
        return both;
    )
}

typedef int (*rotate_fn)(const odmkv_rotate_t*, void*);
typedef int (*prompt_fn)(const odmkv_prompt_attend_t*, void*);
typedef size_t (*prompt_bytes_fn)(int, int, int, int, int, int, int, int, float);

// gradients that a call would have to record, or a tangent that it would have to carry on
bool recorded(const at::Tensor& t) { return (t.requires_grad() && at::GradMode::is_enabled()) || t._fw_grad(0).defined(); }
// [B, heads, T, 128] in 16 bits with rows that start on 16 bytes, and nothing to record
bool heads_fit(const at::Tensor& t, at::ScalarType type, int device) {
    if (t.dim() != 4 || !t.is_cuda() || t.get_device() != device || t.scalar_type() != type || recorded(t)) return false;
    const auto r = t.strides();
    return t.size(3) == ODMKV_HEAD_DIM && r[3] == 1 && ((r[0] | r[1] | r[2]) & 7) == 0 && ((uintptr_t)t.data_ptr() & 15) == 0 && t.size(2) <= (1 << 26);
}
// None, or int32 [n] on the device; false: something else
bool ints_fit(PyObject* o, int64_t n, int device, const int32_t*& at) {
    at = nullptr;
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) return false;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.get_device() != device || t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n || !t.is_contiguous()) return false;
    at = (const int32_t*)t.data_ptr();
    return true;
}
PyObject* pair_of(at::Tensor a, at::Tensor b) {
    PyObject* both = PyTuple_New(2);
    if (both) {
        PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(a)));
        PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(b)));
    }
    return both;
}

// paged_write_rotated(entry, pages, device, layer, query, keys, values, cosine, sine, offsets, starts, interleaved, return_keys, grown, stream): query turned, or (query, keys), or
// None
PyObject* native_paged_write_rotated(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 15) {
        PyErr_SetString(PyExc_TypeError, "paged_write_rotated(entry, pages, device, layer, query, keys, values, cosine, sine, offsets, starts, interleaved, return_keys, grown, stream)");
        return nullptr;
    }
    for (int i = 4; i < 9; ++i)
        if (!THPVariable_Check(a[i])) Py_RETURN_NONE;
    const rotate_fn fn = (rotate_fn)(uintptr_t)PyLong_AsUnsignedLongLong(a[0]);
    const odmkv_pages_t* p = (const odmkv_pages_t*)(uintptr_t)PyLong_AsUnsignedLongLong(a[1]);
    const int device = (int)PyLong_AsLong(a[2]);
    const long layer = PyLong_AsLong(a[3]);
    const int interleaved = PyObject_IsTrue(a[11]);
    const int want_keys = PyObject_IsTrue(a[12]);
    const long long grown = PyLong_AsLongLong(a[13]);
    const unsigned long long stream = PyLong_AsUnsignedLongLong(a[14]);
    if (PyErr_Occurred()) return nullptr;
    GUARDED(
        const at::Tensor& q = THPVariable_Unpack(a[4]);
        const at::Tensor& k = THPVariable_Unpack(a[5]);
        const at::Tensor& v = THPVariable_Unpack(a[6]);
        const at::Tensor& c = THPVariable_Unpack(a[7]);
        const at::Tensor& s = THPVariable_Unpack(a[8]);
        const at::ScalarType type = scalar_of(p->dtype);
        const bool packed = a[9] != Py_None;
        const int64_t B = packed ? 1 : p->rows;
        if (layer < 0 || layer >= p->layers || !heads_fit(q, type, device) || !heads_fit(k, type, device) || !heads_fit(v, type, device)) Py_RETURN_NONE;
        const int64_t T = k.size(2);
        const int64_t Hq = q.size(1);
        if (q.size(0) != B || k.size(0) != B || v.sizes() != k.sizes() || k.size(1) != p->Hkv || q.size(2) != T || Hq < 1 || Hq > 65535 || T < 1 || T < grown) Py_RETURN_NONE;
        for (const at::Tensor* t : {&c, &s})
            if (t->dim() != 2 || !t->is_cuda() || t->get_device() != device || t->scalar_type() != at::kFloat || !t->is_contiguous() || t->sizes() != c.sizes() || ((uintptr_t)t->data_ptr() & 15) || recorded(*t)) Py_RETURN_NONE;
        const int64_t half = c.size(1);
        if (half < 8 || half > ODMKV_HEAD_DIM / 2 || half % 8 || c.size(0) < 1 || c.size(0) > INT32_MAX) Py_RETURN_NONE;
        odmkv_rotate_t d;
        memset(&d, 0, sizeof d);
        if (!ints_fit(a[9], (int64_t)p->rows + 1, device, d.offsets) || !ints_fit(a[10], p->rows, device, d.starts)) Py_RETURN_NONE;
        // (token by token, looked at head by head)
        const auto by_token = [&](int64_t heads) {
            return at::empty_strided({B, heads, T, ODMKV_HEAD_DIM}, {T * heads * ODMKV_HEAD_DIM, ODMKV_HEAD_DIM, heads * ODMKV_HEAD_DIM, 1}, q.options());
        };
        at::Tensor turned = by_token(Hq);
        at::Tensor keys;
        if (want_keys) keys = by_token(p->Hkv);
        d.pages = p;
        d.q = q.data_ptr(); d.q_stride_b = q.stride(0); d.q_stride_h = q.stride(1); d.q_stride_t = q.stride(2);
        d.k = k.data_ptr(); d.k_stride_b = k.stride(0); d.k_stride_h = k.stride(1); d.k_stride_t = k.stride(2);
        d.v = v.data_ptr(); d.v_stride_b = v.stride(0); d.v_stride_h = v.stride(1); d.v_stride_t = v.stride(2);
        d.q_out = turned.data_ptr(); d.k_out = want_keys ? keys.data_ptr() : nullptr;
        d.cosine = (const float*)c.data_ptr(); d.sine = (const float*)s.data_ptr();
        d.layer = (int)layer; d.T = (int)(packed ? (grown > 1 ? grown : 1) : T); d.tokens = (int)T; d.Hq = (int)Hq;
        d.turned = (int)(2 * half); d.interleaved = interleaved; d.table = (int)c.size(0);
        const int rc = fn(&d, (void*)(uintptr_t)stream);
        if (rc) return raise_odmkv(rc, "storing turned tokens");
        if (!want_keys) return THPVariable_Wrap(std::move(turned));
        return pair_of(std::move(turned), std::move(keys));
    )
}

// prompt_attend(entry, workspace entry, device, query, keys, values, offsets, key_offsets, starts, causal, window, scaling, cap, want_lse, stream): out, or (out, lse), or None
PyObject* native_prompt_attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 15) {
        PyErr_SetString(PyExc_TypeError, "prompt_attend(entry, bytes, device, query, keys, values, offsets, key_offsets, starts, causal, window, scaling, cap, want_lse, stream)");
        return nullptr;
    }
    for (int i = 3; i < 6; ++i)
        if (!THPVariable_Check(a[i])) Py_RETURN_NONE;
    const prompt_fn fn = (prompt_fn)(uintptr_t)PyLong_AsUnsignedLongLong(a[0]);
    const prompt_bytes_fn bytes_of = (prompt_bytes_fn)(uintptr_t)PyLong_AsUnsignedLongLong(a[1]);
    const int device = (int)PyLong_AsLong(a[2]);
    const int causal = PyObject_IsTrue(a[9]);
    const long long window = PyLong_AsLongLong(a[10]);
    const double scaling = PyFloat_AsDouble(a[11]);
    const double cap = PyFloat_AsDouble(a[12]);
    const int want_lse = PyObject_IsTrue(a[13]);
    const unsigned long long stream = PyLong_AsUnsignedLongLong(a[14]);
    if (PyErr_Occurred()) return nullptr;
    GUARDED(
        const at::Tensor& q = THPVariable_Unpack(a[3]);
        const at::Tensor& k = THPVariable_Unpack(a[4]);
        const at::Tensor& v = THPVariable_Unpack(a[5]);
        const at::ScalarType type = q.scalar_type();
        if ((type != at::kHalf && type != at::kBFloat16) || !heads_fit(q, type, device) || !heads_fit(k, type, device) || !heads_fit(v, type, device)) Py_RETURN_NONE;
        const int64_t B = q.size(0);
        const int64_t Hq = q.size(1);
        const int64_t L = q.size(2);
        const int64_t Hkv = k.size(1);
        const int64_t T = k.size(2);
        const bool packed = a[6] != Py_None;
        if (k.sizes() != v.sizes() || k.size(0) != B || B < 1 || Hkv < 1 || Hq < 1 || Hq % Hkv || Hq > 65535 || L < 1 || k.stride(2) >= (1 << 24) || v.stride(2) >= (1 << 24)) Py_RETURN_NONE;
        int64_t rows = B;
        if (packed) {
            if (B != 1 || !THPVariable_Check(a[6]) || (a[7] == Py_None && L != T)) Py_RETURN_NONE;
            const at::Tensor& t = THPVariable_Unpack(a[6]);
            if (t.dim() != 1 || t.size(0) < 2) Py_RETURN_NONE;
            rows = t.size(0) - 1;
        } else if (a[7] != Py_None) Py_RETURN_NONE;
        if (rows > (1 << 20)) Py_RETURN_NONE;
        odmkv_prompt_attend_t d;
        memset(&d, 0, sizeof d);
        if (!ints_fit(a[6], rows + 1, device, d.offsets) || !ints_fit(a[7], rows + 1, device, d.key_offsets) || !ints_fit(a[8], rows, device, d.starts)) Py_RETURN_NONE;
        at::Tensor out = at::empty({B, L, Hq, ODMKV_HEAD_DIM}, q.options());
        at::Tensor lse;
        if (want_lse) lse = at::empty({B, Hq, L}, q.options().dtype(at::kFloat));
        const size_t bytes = bytes_of(packed, (int)rows, (int)Hq, (int)Hkv, (int)L, (int)T, causal, (int)window, (float)cap);
        at::Tensor ws;
        if (bytes) ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));      // (of its own for every call: a graph's is the graph's)
        d.q = q.data_ptr(); d.q_stride_b = q.stride(0); d.q_stride_h = q.stride(1); d.q_stride_t = q.stride(2);
        d.k = k.data_ptr(); d.k_stride_b = k.stride(0); d.k_stride_h = k.stride(1); d.k_stride_t = k.stride(2);
        d.v = v.data_ptr(); d.v_stride_b = v.stride(0); d.v_stride_h = v.stride(1); d.v_stride_t = v.stride(2);
        d.out = out.data_ptr(); d.lse = want_lse ? (float*)lse.data_ptr() : nullptr;
        d.workspace = bytes ? ws.data_ptr() : nullptr; d.workspace_bytes = bytes;
        d.dtype = type == at::kHalf ? ODMKV_F16 : ODMKV_BF16;
        d.rows = (int)rows; d.L = (int)L; d.T = (int)T; d.Hq = (int)Hq; d.Hkv = (int)Hkv; d.causal = causal; d.window = (int)window;
        d.scaling = (float)scaling; d.cap = (float)cap;
        const int rc = fn(&d, (void*)(uintptr_t)stream);
        if (rc) return raise_odmkv(rc, "attention of a prompt");
        if (!want_lse) return THPVariable_Wrap(std::move(out));
        return pair_of(std::move(out), std::move(lse));
    )
}

PyMethodDef module_methods[] = {
    {"paged_write_rotated", (PyCFunction)(void*)native_paged_write_rotated, METH_FASTCALL, nullptr},
    {"prompt_attend", (PyCFunction)(void*)native_prompt_attend, METH_FASTCALL, nullptr},
    {"paged_write", (PyCFunction)(void*)native_paged_write, METH_FASTCALL, nullptr},
    {"paged_attend", (PyCFunction)(void*)native_paged_attend, METH_FASTCALL, nullptr},
    {"alias", (PyCFunction)(void*)native_alias, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, module_methods};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) {
    s_sliding = PyUnicode_InternFromString("sliding_window"); s_softcap = PyUnicode_InternFromString("softcap");
    s_aux = PyUnicode_InternFromString("s_aux"); s_scaling = PyUnicode_InternFromString("scaling");
    StepType.tp_name = "kvquant._native.Step";
    StepType.tp_basicsize = sizeof(Step);
    StepType.tp_flags = Py_TPFLAGS_DEFAULT;
    StepType.tp_new = PyType_GenericNew;
    StepType.tp_init = step_init;
    StepType.tp_dealloc = step_dealloc;
    StepType.tp_methods = step_methods;
    StepType.tp_members = step_members;
    if (PyType_Ready(&StepType) < 0) return nullptr;
    PyObject* m = PyModule_Create(&module_def);
    if (!m) return nullptr;
    Py_INCREF(&StepType);
    if (PyModule_AddObject(m, "Step", (PyObject*)&StepType) < 0) { Py_DECREF(&StepType); Py_DECREF(m); return nullptr; }
    return m;
}
