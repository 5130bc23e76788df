// ztcp_torch.cpp -- torch tensors to the C ABI of the operators on hot pages
// (include/ztcp.h) for vlx-tee_amd/attention.py.
//
// A decoding step calls these operators once a layer and its kernels last a few
// microseconds, so the checks, the outputs' allocation and the call are made
// here: in Python they took 18 to 26 us of host time a call, more than the
// kernels of one sequence.  Functions take positional arguments only; names,
// defaults and documentation are attention.py's.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <stdexcept>
#include <string>

#include "../../include/ztcp.h"

namespace {

struct Refused : std::runtime_error {   // becomes a ValueError
    using std::runtime_error::runtime_error;
};

void need(bool ok, const char* why) {
    if (!ok) throw Refused(why);
}
void need(bool ok, const char* name, const char* why) {
    if (!ok) throw Refused(std::string(name) + why);
}

void done(int rc, const char* what) {
    if (rc == ZTCP_OK) return;
    if (rc == ZTCP_EINVAL || rc == ZTCP_EOVERLAP) throw Refused(std::string(what) + ": " + ztcp_last_error());
    throw std::runtime_error(std::string(what) + ": " + ztcp_strerror(rc) + " (code " + std::to_string(rc) + ")");
}

const at::Tensor* tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) throw Refused(std::string(name) + " must be a tensor");
    const at::Tensor* t = &THPVariable_Unpack(o);
    if (at::GradMode::is_enabled() && t->requires_grad())
        throw Refused(std::string(name) + " requires a gradient, which this operator does not have (torch.no_grad())");
    if (t->_fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
        throw Refused(std::string(name) + " carries a tangent, which this operator would drop");
    return t;
}
const at::Tensor* tensor_or_none(PyObject* o, const char* name) { return o == Py_None ? nullptr : tensor(o, name); }

int64_t whole(PyObject* o, const char* name) {
    const long long x = PyLong_AsLongLong(o);
    if (x == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        throw Refused(std::string(name) + " must be a whole number of 64 bits");
    }
    return x;
}
double number(PyObject* o, const char* name) {
    const double x = PyFloat_AsDouble(o);
    if (x == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        throw Refused(std::string(name) + " must be a number");
    }
    return x;
}

bool truth(PyObject* o, const char* name) {
    const int x = PyObject_IsTrue(o);
    if (x < 0) {
        PyErr_Clear();
        throw Refused(std::string(name) + " must be true or false");
    }
    return x != 0;
}

// A tensor that the caller holds has been written: what torch saved of it for a gradient is no longer what it was.
// (Tensors of inference mode have no versions.)
void written(const at::Tensor* t) {
    if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

void* stream_of(const at::Device& d) { return (void*)c10::hip::getCurrentHIPStream(d.index()).stream(); }

at::Tensor make(at::IntArrayRef shape, at::ScalarType type, const at::Device& d) {
    return at::empty(shape, at::TensorOptions().dtype(type).device(d));
}

// A pool of pages [n_pages, page_tokens, kv_heads, head_dim], each page contiguous.
struct Pool {
    const at::Tensor* k;
    ztcp_page_pool pool;
    ztcp_geometry g;
    Pool(const at::Tensor* k_pages, const at::Tensor* v_pages, int64_t rope_dim) : k(k_pages) {
        page_check(*k_pages, "k_pages");
        if (v_pages) {
            page_check(*v_pages, "v_pages");
            need(v_pages->sizes() == k->sizes() && v_pages->scalar_type() == k->scalar_type() && v_pages->device() == k->device(),
                 "v_pages must match k_pages in shape, dtype and device");
        }
        pool = ztcp_page_pool{k->data_ptr(), v_pages ? v_pages->data_ptr() : nullptr, k->size(0), step(*k), step(v_pages ? *v_pages : *k)};
        g = ztcp_geometry{k->size(1), k->size(2), k->size(3), rope_dim,
                          k->scalar_type() == at::kBFloat16 ? ZTCP_HOT_BF16 : ZTCP_HOT_FP16, v_pages ? 0 : 1};
    }
    static void page_check(const at::Tensor& t, const char* name) {
        need(t.dim() == 4, name, " must have shape [n_pages, page_tokens, kv_heads, head_dim]");
        need(t.is_cuda() && (t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16), name,
             " must be a HIP float16 or bfloat16 tensor");
        const int64_t h = t.size(2), d = t.size(3);
        need(t.numel() > 0 && (d == 1 || t.stride(3) == 1) && (h == 1 || t.stride(2) == d) &&
                 (t.size(1) == 1 || t.stride(1) == h * d),
             name, " must hold pages, each of them contiguous");
    }
    static int64_t step(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2) * t.size(3); }
    at::Device device() const { return k->device(); }

    // Elements between the tokens of [tokens, heads, head_dim] rows.
    int64_t tokens(const at::Tensor& t, const char* name, bool kv_heads = false) const {
        need(t.dim() == 3, name, " must have shape [tokens, heads, head_dim]");
        need(t.scalar_type() == k->scalar_type() && t.device() == device(), name, " must match the pages' dtype and device");
        need(t.size(2) == k->size(3), name, "'s head_dim must be the pages'");
        need(!kv_heads || t.size(1) == k->size(2), name, " must have the pages' heads");
        need(t.numel() == 0 || ((t.size(2) == 1 || t.stride(2) == 1) && (t.size(1) <= 1 || t.stride(1) == t.size(2))), name,
             ": a token's heads must be contiguous");
        return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2);
    }
    const void* array(const at::Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef shape) const {
        return plain(t, name, type, shape, device());
    }
    static void* plain(const at::Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef shape, const at::Device& d) {
        if (!(t.scalar_type() == type && t.device() == d && t.sizes() == shape && t.is_contiguous())) {
            std::string s = std::string(name) + " must be a contiguous " + c10::toString(type) + " tensor of shape [";
            for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
            throw Refused(s + "] on the pages' device");
        }
        return t.data_ptr();
    }
    // Entries between the rows of a page table.
    static int64_t table(const at::Tensor& t, const at::Device& d) {
        need(t.dim() == 2 && t.scalar_type() == at::kInt && t.device() == d && t.size(1) > 0 &&
                 (t.size(1) == 1 || t.stride(1) == 1),
             "page_table must be an int32 tensor [sequences, pages] on the pages' device, its rows contiguous");
        return t.size(0) > 1 ? t.stride(0) : t.size(1);
    }
    ztcp_paged_batch batch(const at::Tensor& page_table, const at::Tensor& kv_lens, const at::Tensor& q_starts, int64_t rows,
                           PyObject* max_q_len) const {
        const int64_t stride = table(page_table, device()), s = page_table.size(0);
        const int64_t most = max_q_len == Py_None ? 0 : whole(max_q_len, "max_q_len");
        need(most >= 0, "max_q_len must not be negative");
        return ztcp_paged_batch{(const int32_t*)page_table.data_ptr(), stride, page_table.size(1),
                                (const int32_t*)array(kv_lens, "kv_lens", at::kInt, {s}),
                                (const int32_t*)array(q_starts, "q_starts", at::kInt, {s + 1}), s, rows, most};
    }
};

PyObject* append_tokens(PyObject* const* a) {
    const at::Tensor *q = tensor(a[0], "q"), *k = tensor(a[1], "k"), *v = tensor_or_none(a[2], "v");
    const at::Tensor *k_pages = tensor(a[3], "k_pages"), *v_pages = tensor_or_none(a[4], "v_pages");
    const at::Tensor *slots = tensor(a[5], "slots"), *positions = tensor(a[6], "positions"), *rope = tensor(a[7], "rope");
    const at::Tensor* weight[2] = {tensor_or_none(a[8], "q_weight"), tensor_or_none(a[9], "k_weight")};
    const at::Tensor* given = tensor_or_none(a[12], "q_out");
    need((v == nullptr) == (v_pages == nullptr), "v and v_pages must both be given or both be None");
    need(rope->dim() == 2, "rope must have shape [max_position, rope_dim]");
    const Pool p(k_pages, v_pages, rope->size(1));
    const at::Device d = p.device();
    const int64_t qs = p.tokens(*q, "q"), ks = p.tokens(*k, "k", true), vs = v ? p.tokens(*v, "v", true) : 0, n = q->size(0);
    need(k->size(0) == n && (!v || v->size(0) == n), "q, k and v must have the same number of tokens");
    const void* rope_ptr = p.array(*rope, "rope", at::kFloat, {rope->size(0), rope->size(1)});
    const void* w[2];
    int64_t wl[2];
    for (int i = 0; i < 2; ++i) {
        const char* name = i ? "k_weight" : "q_weight";
        need(!weight[i] || weight[i]->numel() > 0, name, " must not be empty");
        w[i] = weight[i] ? p.array(*weight[i], name, k_pages->scalar_type(), {weight[i]->numel()}) : nullptr;
        wl[i] = weight[i] ? weight[i]->numel() : 0;
    }
    need(!given || given->sizes() == q->sizes(), "q_out must have q's shape");
    const at::Tensor out = given ? *given : make(q->sizes(), q->scalar_type(), d);
    const int64_t os = p.tokens(out, "q_out");
    const void* slot_ptr = p.array(*slots, "slots", at::kLong, {n});
    const void* pos_ptr = p.array(*positions, "positions", at::kInt, {n});
    const float eps = (float)number(a[10], "eps");
    const c10::DeviceGuard guard(d);
    done(ztcp_append_tokens(q->data_ptr(), qs, out.data_ptr(), os, k->data_ptr(), ks, v ? v->data_ptr() : nullptr, vs, n,
                            q->size(1), &p.pool, &p.g, (const int64_t*)slot_ptr, (const int32_t*)pos_ptr,
                            (const float*)rope_ptr, rope->size(0), w[0], wl[0], w[1], wl[1], eps, truth(a[11], "interleaved"),
                            stream_of(d)),
         "append_tokens");
    for (const at::Tensor* t : {given, k_pages, v_pages}) written(t);
    return THPVariable_Wrap(out);
}

float scale_of(PyObject* o, int64_t head_dim) {
    return o == Py_None ? (float)(1.0 / std::sqrt((double)head_dim)) : (float)number(o, "scale");
}

PyObject* paged_attention(PyObject* const* a) {
    need(a[2] != Py_None, "paged_attention needs K and V pages (single-buffer pages have none)");
    const at::Tensor *q = tensor(a[0], "q"), *k_pages = tensor(a[1], "k_pages"), *v_pages = tensor(a[2], "v_pages");
    const at::Tensor *table = tensor(a[3], "page_table"), *lens = tensor(a[4], "kv_lens"), *starts = tensor(a[5], "q_starts");
    const bool want_lse = truth(a[8], "return_lse");
    const at::Tensor* given = tensor_or_none(a[9], "out");
    const Pool p(k_pages, v_pages, 0);
    const at::Device d = p.device();
    const int64_t qs = p.tokens(*q, "q"), n = q->size(0), heads = q->size(1);
    const ztcp_paged_batch batch = p.batch(*table, *lens, *starts, n, a[7]);
    const at::Tensor out = given ? *given : make(q->sizes(), q->scalar_type(), d);
    if (given) p.array(out, "out", q->scalar_type(), q->sizes());
    const at::Tensor lse = want_lse ? make({n, heads}, at::kFloat, d) : at::Tensor();
    const float scale = scale_of(a[6], k_pages->size(3));
    const c10::DeviceGuard guard(d);
    const size_t bytes = ztcp_paged_attention_workspace(&batch, &p.pool, &p.g, heads);
    if (bytes == (size_t)-1) done(*ztcp_last_error() ? ZTCP_EINVAL : ZTCP_EHIP, "paged_attention");
    // the caching allocator gives it to later work of this stream only
    const at::Tensor work = bytes ? make({(int64_t)bytes}, at::kByte, d) : at::Tensor();
    done(ztcp_paged_attention(q->data_ptr(), qs, out.data_ptr(), want_lse ? (float*)lse.data_ptr() : nullptr, heads, &p.pool,
                              &batch, &p.g, scale, bytes ? work.data_ptr() : nullptr, bytes, stream_of(d)),
         "paged_attention");
    written(given);
    PyObject* o = THPVariable_Wrap(out);
    if (!want_lse || !o) return o;
    PyObject* l = THPVariable_Wrap(lse);
    PyObject* both = l ? PyTuple_Pack(2, o, l) : nullptr;
    Py_DECREF(o);
    Py_XDECREF(l);
    return both;
}

PyObject* attention_mass(PyObject* const* a) {
    const at::Tensor *q = tensor(a[0], "q"), *lse = tensor(a[1], "lse"), *k_pages = tensor(a[2], "k_pages");
    const at::Tensor *table = tensor(a[3], "page_table"), *lens = tensor(a[4], "kv_lens"), *starts = tensor(a[5], "q_starts");
    const at::Tensor* mass = tensor(a[6], "mass");
    const at::Tensor* given = tensor_or_none(a[10], "out");
    const Pool p(k_pages, nullptr, 0);
    const at::Device d = p.device();
    const int64_t qs = p.tokens(*q, "q"), n = q->size(0), heads = q->size(1);
    const ztcp_paged_batch batch = p.batch(*table, *lens, *starts, n, a[9]);
    const int64_t shape[3] = {table->size(0), k_pages->size(2), table->size(1)};
    const at::Tensor out = given ? *given : make(shape, at::kFloat, d);
    if (given) p.array(out, "out", at::kFloat, shape);
    const void* lse_ptr = p.array(*lse, "lse", at::kFloat, {n, heads});
    const void* mass_ptr = p.array(*mass, "mass", at::kFloat, shape);
    const float scale = scale_of(a[7], k_pages->size(3)), decay = (float)number(a[8], "decay");
    const c10::DeviceGuard guard(d);
    done(ztcp_attention_mass(q->data_ptr(), qs, (const float*)lse_ptr, heads, &p.pool, &batch, &p.g, scale,
                             (const float*)mass_ptr, decay, (float*)out.data_ptr(), stream_of(d)),
         "attention_mass");
    written(given);
    return THPVariable_Wrap(out);
}

PyObject* evict_pages(PyObject* const* a) {
    const at::Tensor *mass = tensor(a[0], "mass"), *table = tensor(a[1], "page_table"), *lens = tensor(a[2], "kv_lens");
    need(mass->is_cuda() && mass->dim() == 3, "mass must be a HIP tensor [sequences, kv_heads, pages]");
    const at::Device d = mass->device();
    const int64_t stride = Pool::table(*table, d), s = table->size(0), mp = table->size(1), heads = mass->size(1);
    const void* mass_ptr = Pool::plain(*mass, "mass", at::kFloat, {s, heads, mp}, d);
    const void* lens_ptr = Pool::plain(*lens, "kv_lens", at::kInt, {s}, d);
    const bool in_place = truth(a[7], "in_place");
    at::Tensor out[5];
    out[0] = in_place ? *table : make({s, mp}, at::kInt, d);
    out[1] = in_place ? *mass : make({s, heads, mp}, at::kFloat, d);
    out[2] = in_place ? *lens : make({s}, at::kInt, d);
    out[3] = make({s, mp}, at::kInt, d);
    out[4] = make({s}, at::kInt, d);
    const int64_t tokens = whole(a[3], "page_tokens"), budget = whole(a[4], "budget"), sink = whole(a[5], "sink"),
                  recent = whole(a[6], "recent");
    const c10::DeviceGuard guard(d);
    done(ztcp_evict_pages((const float*)mass_ptr, (const int32_t*)table->data_ptr(), stride, (const int32_t*)lens_ptr, s, heads,
                          mp, tokens, budget, sink, recent, (int32_t*)out[0].data_ptr(), in_place ? stride : mp,
                          (float*)out[1].data_ptr(), (int32_t*)out[2].data_ptr(), (int32_t*)out[3].data_ptr(),
                          (int32_t*)out[4].data_ptr(), stream_of(d)),
         "evict_pages");
    for (const at::Tensor* t : {table, mass, lens}) written(in_place ? t : nullptr);
    PyObject* all = PyTuple_New(5);
    for (int i = 0; all && i < 5; ++i) {
        PyObject* o = THPVariable_Wrap(out[i]);
        if (!o) {
            Py_DECREF(all);
            return nullptr;
        }
        PyTuple_SET_ITEM(all, i, o);
    }
    return all;
}

// No C++ exception leaves a C entry.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "%d positional arguments wanted, %zd given", N, n);
        return nullptr;
    }
    try {
        return F(args);
    } catch (const Refused& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const c10::OutOfMemoryError& e) {
        PyObject* torch = PyImport_ImportModule("torch");
        PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
        PyErr_Clear();
        PyErr_SetString(type ? type : PyExc_MemoryError, e.what_without_backtrace());
        Py_XDECREF(type);
        Py_XDECREF(torch);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

#define ZT_FUNCTION(name, n) {#name, (PyCFunction)(void*)entry<name, n>, METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {ZT_FUNCTION(append_tokens, 13), ZT_FUNCTION(paged_attention, 10), ZT_FUNCTION(attention_mass, 11),
                          ZT_FUNCTION(evict_pages, 8), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_ztcp_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ztcp_torch(void) { return PyModule_Create(&kModule); }
